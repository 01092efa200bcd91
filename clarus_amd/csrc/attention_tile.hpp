// Device code shared by the kernels that hold a tile of keys and values in LDS and 32 rows of queries per wave
// (cross_attention.hip says how): layout of the tiles, their copies, a tile's step of the softmax, the finished rows and
// the join of keys split over workgroups.
#pragma once

#include "common.hpp"

namespace clarus {

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr int XA_T = 256;    // threads of a join or bits workgroup
constexpr float XA_FLOOR = -3e38f;  // running maximum before any key: exp2(-inf - XA_FLOOR) = 0, no inf - inf
constexpr float XA_MOST = 3.402823466e38f;  // the largest finite fp32
constexpr float XA_SLACK = 8.f;     // a running maximum may lag the scores' by this (log2)
constexpr float XA_FAR = 8388608.f;  // 2^23: up to this size a running maximum is within a quarter of the product it rounds

enum : int { MASK_NONE = 0, MASK_KEYS = 1, MASK_PAIRS = 2, MASK_ROWS = 3 };

struct CrossP {
  const void *q, *k, *v;
  void* out;
  const unsigned char* mask;
  const uint64_t* bits;      // MASK_PAIRS: [n][lq][nw] words of 64 keys, image stride bbs (words)
  int64_t nw, bbs;
  float* part;               // [split][nk][rows][D] O, then [split][nk][rows] (m, l)
  int64_t qbs, ldq, kbs, ldk, vbs, ldv, mbs, mqs;
  int64_t rows;              // lq * rep
  int64_t lk, split_len, nk; // nk = n * kv_heads
  int64_t nblk;              // row blocks (resident: workgroups) of an (image, kv head)
  int lq, rep, kv_heads, d, splits, o_dt;
  float c;                   // scale log2(e)
};

// a and b of lanes l and l ^ 32: the low half keeps a's low and gets a's high lanes in b, the high half gets b's low
// lanes in a and keeps b's high
__device__ __forceinline__ void swap32(unsigned& a, unsigned& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

// max / sum with lane ^ 32
__device__ __forceinline__ float max32(float v) {
  unsigned a = __float_as_uint(v), b = a;
  swap32(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float sum32(float v) {
  unsigned a = __float_as_uint(v), b = a;
  swap32(a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

template <int DT, int D>
struct XaTile {
  static constexpr int ES = DT == DT_BF16 ? 2 : 4;
  static constexpr int KT = DT == DT_BF16 ? 64 : 32;  // keys per tile
  static constexpr int ROWB = D * ES;                 // bytes of a row in LDS
  static constexpr int CPR = ROWB / 16;               // 16-byte chunks per row
  static constexpr int BYTES = KT * ROWB;
  static constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xffffffffull;
  // chunk c of row r sits at position c ^ swz(r). K: 16 lanes read one chunk of 16 consecutive rows; V: bf16
  // 8 rows x 4 chunks (transposing), fp32 two rows 4 apart x 8 chunks: each over all banks (fp32 V of 32 and
  // 96 columns excepted, whose rows r and r + 4 meet)
  static __device__ __forceinline__ int swz_k(int r) {
    return ROWB == 64 ? (r >> 2) & 3 : ROWB == 128 || ROWB == 384 ? (r >> 1) & 7 : ROWB == 192 ? (r >> 2) & 3 : r & 15;
  }
  static __device__ __forceinline__ int swz_v(int r) {
    if constexpr (DT == DT_BF16) return D == 64 ? ((r >> 1) & 1) * 4 : D == 128 ? (r & 3) * 4 : 0;
    return D == 64 || D == 128 ? ((r >> 2) & 1) * 8 : 0;
  }
  static __device__ __forceinline__ int at_k(int r, int c) { return r * ROWB + (c ^ swz_k(r)) * 16; }
  static __device__ __forceinline__ int at_v(int r, int c) { return r * ROWB + (c ^ swz_v(r)) * 16; }
};

// 16-byte chunks of a row of Q per lane. C: the head's columns in sixteens, what a score sums over
template <int DT, int C> constexpr int xa_qn = DT == DT_BF16 ? C / 16 : C / 8;

// what a masked, padding or absent piece of K or V is copied from
__device__ const u32x4 xa_zeros[1] = {u32x4{0, 0, 0, 0}};

// keep ? v : -inf, keep = bit `bit` of w (v may be NaN)
__device__ __forceinline__ float keep_bit(float v, unsigned w, int bit) {
  const unsigned k = (unsigned)__builtin_amdgcn_sbfe((int)w, bit, 1);
  return __uint_as_float((__float_as_uint(v) & k) | (0xff800000u & ~k));
}

// one row of a wave: its query and head
struct XaRow {
  int64_t qi;
  int head;
};

__device__ __forceinline__ XaRow xa_row(const CrossP& p, int kvh, int64_t row) {
  // 32-bit division: rows < 2^31
  const int qi = p.rep == 1 ? (int)row : (int)((unsigned)row / (unsigned)p.rep);
  return XaRow{qi, kvh * p.rep + (int)row - qi * p.rep};
}

// Q^T fragments of a row
template <int DT, int C>
__device__ __forceinline__ void xa_load_q(const CrossP& p, int64_t n, const XaRow& r, int hl, u32x4 (&qf)[xa_qn<DT, C>]) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4, E = 16 / ES, QN = xa_qn<DT, C>;
  const unsigned char* qp = (const unsigned char*)p.q + (n * p.qbs + r.qi * p.ldq + (int64_t)r.head * p.d) * ES;
#pragma unroll
  for (int s = 0; s < QN; ++s) {
    const int at = (2 * s + hl) * E;
    qf[s] = *reinterpret_cast<const u32x4*>(qp + (at < p.d ? at : 0) * ES);
  }
  if (p.d < C) {
#pragma unroll
    for (int s = 0; s < QN; ++s)
      if ((2 * s + hl) * E >= p.d) qf[s] = u32x4{0, 0, 0, 0};
  }
}

// 16 mask bytes (0 masked, any other value kept) at p, the first `left` of them there, as 16 bits
__device__ __forceinline__ unsigned xa_bits16(const unsigned char* p, int64_t left) {
  struct __attribute__((packed, aligned(1))) Bytes { u32x4 v; };
  u32x4 w = {0, 0, 0, 0};
  if (left >= 16) {
    w = reinterpret_cast<const Bytes*>(p)->v;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) w[i >> 2] |= (unsigned)p[i] << (8 * (i & 3));
  }
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned any = (((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) >> 7 & 0x01010101u;  // byte != 0
    r |= (any * 0x10204080u >> 28) << (4 * i);                                             // bytes 0 .. 3 -> bits 28 .. 31
  }
  return r;
}

// One tile of NB x 32 keys for a wave's 32 rows: S^T = K Q^T, the softmax's step, O^T += V^T P^T. bits: the keys that
// count, of a lane's row under MASK_PAIRS; whole: all of them; fresh: o is still 0; far: the maximum of
// a row of the wave has been past XA_FAR; MASK_ROWS: the rows that are not live keep nothing of the tile, the others `bits`
template <int DT, int D, int C, int MASK, int NB, bool ANEW>
__device__ __forceinline__ void xa_tile(const unsigned char* ks, const unsigned char* vs, const u32x4 (&qf)[xa_qn<DT, C>],
                                        f32x16 (&o)[D / 32], float& m, float& l, bool& far, float c, uint64_t bits, bool whole, bool fresh,
                                        bool live = true) {
  using T = XaTile<DT, D>;
  constexpr int DB = D / 32, QN = xa_qn<DT, C>;
  // ANEW: the lane's LDS offsets are worked out for each tile instead of kept over the loop, where they spill
  int lane = threadIdx.x & 63;
  if constexpr (ANEW) asm volatile("" : "+v"(lane));
  const int col = lane & 31, hl = lane >> 5;
  f32x16 s[NB];
  // Waves of one SIMD that reach the products together share the matrix core and then wait for each other's arithmetic:
  // the wave that is further in its tile goes first (14400 x 3600, 8 heads of 64: 147 us without, 141; 57600 x 3600, 4
  // heads of 128: 477 and 466)
  __builtin_amdgcn_s_setprio(0);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(ks + T::at_k(32 * b + col, 2 * i + hl));
      if constexpr (DT == DT_BF16) {
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, qf[i]), s[b], 0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(qf[i][e]), s[b], 0, 0, 0);
      }
    }
  }
  __builtin_amdgcn_s_setprio(1);
  // masked and padding keys weigh nothing, whatever their scores
  if (!(MASK == MASK_PAIRS ? __all(whole) : whole)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const unsigned w = (unsigned)(bits >> (32 * b)) >> (4 * hl);
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] = keep_bit(s[b][j], w, 8 * (j >> 2) + (j & 3));
    }
  }
  // the running maximum moves only when a score passes it by XA_SLACK (weights then stay below 2^XA_SLACK,
  // and fp32 sums keep their digits): the accumulators are rescaled in few tiles instead of all
  float mx = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) mx = MASK == MASK_ROWS ? __builtin_elementwise_maximum(mx, s[b][j]) : fmaxf(mx, s[b][j]);
  // of a row that is not live -inf as maximum makes every finite score a weight of 0; one that is not finite (the maximum
  // of MASK_ROWS passes NaN on) is put to 0 first. 14400 queries that choose each for themselves: 385 us with this, 386
  // without, 403 with a test of the weights behind the exponentials, which the products then wait for
  const float limit = MASK == MASK_ROWS && !live ? XA_MOST : m + XA_SLACK;
  if (MASK == MASK_ROWS ? __any(!(mx * c <= limit)) : __any(mx * c > m + XA_SLACK)) {
    if (MASK == MASK_ROWS && !live) {
      if (!(mx * c <= limit)) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
      }
      mx = -INFINITY;
    }
    mx = max32(mx);
    const float mn = fmaxf(m, mx * c);
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
    far |= __any(fabsf(m) > XA_FAR && fabsf(m) < -XA_FLOOR) != 0;
    if (!fresh) {
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[b][j] *= alpha;
    }
  }
  // The product in fmaf(s, c, -m) is exact and m is rounded: past XA_FAR half a step of m would, as an exponent, overflow or
  // leave nothing of the weights, so there the products are rounded as m was. One bit of the wave, which moves with m alone:
  // times within 1% (heads of 40 and 80 3%) of those without
  if (far) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] *= c;
    c = 1.f;
  }
  const float mw = MASK == MASK_ROWS && !live ? INFINITY : m;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[b][j] = __builtin_amdgcn_exp2f(fmaf(s[b][j], c, -mw));
      l += s[b][j];
    }
  __builtin_amdgcn_s_setprio(2);
  if constexpr (DT == DT_BF16) {
    const int i = lane & 15;
    const int vr = 4 * hl + (i >> 2), vc = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
    for (int ks2 = 0; ks2 < 2 * NB; ++ks2) {
      f32x8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) pv.v[e] = s[ks2 >> 1][8 * (ks2 & 1) + e];
      const bf16x8 pb = pack_bf16(pv);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        typedef __attribute__((ext_vector_type(8))) short s16x8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(vs + T::at_v(16 * ks2 + vr, 4 * b + vc) + (i & 1) * 8));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(vs + T::at_v(16 * ks2 + vr + 8, 4 * b + vc) + (i & 1) * 8));
        const s16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), pb, o[b], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int r = 32 * kb + 8 * (j >> 2) + 4 * hl + (j & 3);
          const float a = *reinterpret_cast<const float*>(vs + T::at_v(r, 8 * b + (col >> 2)) + (col & 3) * 4);
          o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[kb][j], o[b], 0, 0, 0);
        }
  }
}

// a finished row: O / l (every lane takes part; live: the row is there)
template <int D>
__device__ __forceinline__ void xa_store(const CrossP& p, int64_t n, const XaRow& r, const f32x16 (&o)[D / 32], float l, bool live) {
  const int hl = (threadIdx.x >> 5) & 1;
  const float inv = l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l);
  const int64_t at = ((n * p.lq + r.qi) * (int64_t)(p.kv_heads * p.rep) + r.head) * p.d;
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int j = 0; j < 16; j += 8) {
      f32x4 y[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i >> 2][i & 3] = o[b][j + i] * inv;
      if (p.o_dt == DT_BF16) {
        // columns 8 (j / 4) + 4 hl .. + 3 of two j / 4: exchanged so that each lane stores 8 columns
        u32x4 w = {pack2_bf16(y[0][0], y[0][1]), pack2_bf16(y[0][2], y[0][3]), pack2_bf16(y[1][0], y[1][1]), pack2_bf16(y[1][2], y[1][3])};
        unsigned a0 = w[0], a1 = w[1], b0 = w[2], b1 = w[3];
        swap32(a0, b0);
        swap32(a1, b1);
        const int dd = 32 * b + 2 * j + 8 * hl;
        if (dd < p.d && live) *reinterpret_cast<u32x4*>((unsigned short*)p.out + at + dd) = u32x4{a0, a1, b0, b1};
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int dd = 32 * b + 2 * j + 8 * i + 4 * hl;
          if (dd < p.d && live) *reinterpret_cast<f32x4*>((float*)p.out + at + dd) = y[i];
        }
      }
    }
}

// The copies of a tile's K and V to LDS: this lane's piece of each of a wave's 1 KiB copies (W waves share a tile)
template <int DT, int D, int W>
struct XaCopy {
  using T = XaTile<DT, D>;
  static constexpr int NI = (T::BYTES / 1024 + W - 1) / W;  // copies per wave and operand
  static constexpr bool EVEN = T::BYTES / 1024 % W == 0;
  uint32_t koff[NI], voff[NI];  // from the tile's first row
  int row[NI];
  bool have_k[NI], have_v[NI];  // the chunk lies within the head
  int wave;

  __device__ __forceinline__ XaCopy(const CrossP& p, int wave_, int lane) : wave(wave_) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int at = (wave + W * j) * 1024 + lane * 16;
      const int r = at / T::ROWB, cpos = (at % T::ROWB) / 16;
      const int ck = cpos ^ T::swz_k(r), cv = cpos ^ T::swz_v(r);
      row[j] = r;
      koff[j] = (uint32_t)(r * p.ldk * T::ES) + ck * 16;
      voff[j] = (uint32_t)(r * p.ldv * T::ES) + cv * 16;
      have_k[j] = ck * 16 < p.d * T::ES;
      have_v[j] = cv * 16 < p.d * T::ES;
    }
  }
  __device__ __forceinline__ void operator()(const CrossP& p, const unsigned char* kt, const unsigned char* vt, unsigned char* tile,
                                             uint64_t bits) const {
    unsigned char* dst = tile + wave * 1024;
#define XA_COPY(src, to)                                                                                   \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src),                  \
                                   (__attribute__((address_space(3))) void*)(to), 16, 0, 0)
    if (bits == T::ALL && p.d == D) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= T::BYTES / 1024) break;
        XA_COPY(kt + koff[j], dst + j * W * 1024);
        XA_COPY(vt + voff[j], dst + T::BYTES + j * W * 1024);
      }
    } else {
      const unsigned char* zero = (const unsigned char*)xa_zeros;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= T::BYTES / 1024) break;
        const bool in = (bits >> row[j]) & 1;
        XA_COPY(in && have_k[j] ? kt + koff[j] : zero, dst + j * W * 1024);
        XA_COPY(in && have_v[j] ? vt + voff[j] : zero, dst + T::BYTES + j * W * 1024);
      }
    }
#undef XA_COPY
  }
};

// this lane's key of a tile counts (MASK_KEYS: the mask's byte)
template <int KT, int MASK>
__device__ __forceinline__ int xa_key_byte(const unsigned char* mkey, int64_t base, int64_t k1, int lane) {
  const int64_t key = base + lane;
  const bool in = lane < KT && key < k1;
  if constexpr (MASK == MASK_KEYS) return in ? mkey[key] : 0;
  return in;
}

// any of the KT mask bytes at p (past `left` of them unknown: counted, and sorted out where they are used)
template <int KT>
__device__ __forceinline__ bool xa_any(const unsigned char* p, int64_t left) {
  struct __attribute__((packed, aligned(1))) Bytes { u32x4 v; };
  u32x4 any = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < KT; i += 16)
    if (i + 16 <= left) any |= reinterpret_cast<const Bytes*>(p + i)->v;
  return left < KT || (any[0] | any[1] | any[2] | any[3]);
}

// The splits' (O, m, l) joined. TPR threads hold a row's columns (4 each), gs groups of them its splits: group i takes
// splits i, i + gs, .., XJ_BATCH of them in flight, and the groups are joined through LDS, in a fixed order
constexpr int XJ_BATCH = 8;

template <int D>
__global__ void __launch_bounds__(XA_T) xa_join_kernel(const CrossP p, int gs) {
  constexpr int TPR = D <= 32 ? 8 : D <= 64 ? 16 : 32;
  __shared__ f32x4 so[XA_T];
  __shared__ float2 sml[XA_T];
  const int tid = threadIdx.x, col = (tid % TPR) * 4, part = tid / TPR % gs, rpb = XA_T / (TPR * gs);
  const int64_t total = p.nk * p.rows, at_row = (int64_t)blockIdx.x * rpb + tid / (TPR * gs);
  const int64_t first = at_row < total ? at_row : total - 1;  // (image, kv head) x rows + row; past the end: the last one
  const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.splits * total * D) + first;
  const float* po = p.part + first * D + (col < D ? col : 0);
  float m = XA_FLOOR, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < p.splits; s0 += XJ_BATCH * gs) {
    float2 t[XJ_BATCH];
    f32x4 x[XJ_BATCH];
#pragma unroll
    for (int i = 0; i < XJ_BATCH; ++i) {
      const int64_t at = (int64_t)(s0 + i * gs < p.splits ? s0 + i * gs : s0) * total;
      t[i] = ml[at];
      x[i] = *reinterpret_cast<const f32x4*>(po + at * D);
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < XJ_BATCH; ++i) mn = fmaxf(mn, t[i].x);
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
    o *= alpha;
#pragma unroll
    for (int i = 0; i < XJ_BATCH; ++i) {
      if (s0 + i * gs >= p.splits) break;
      const float w = __builtin_amdgcn_exp2f(t[i].x - m);
      l = fmaf(t[i].y, w, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[i][e], w, o[e]);
    }
  }
  if (gs > 1) {
    so[tid] = o;
    sml[tid] = float2{m, l};
    __syncthreads();
    if (part) return;
    for (int i = 1; i < gs; ++i) {
      const float2 t = sml[tid + i * TPR];
      const f32x4 x = so[tid + i * TPR];
      const float mn = fmaxf(m, t.x), alpha = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(t.x - mn);
      m = mn;
      l = fmaf(t.y, w, l * alpha);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], w, o[e] * alpha);
    }
  }
  if (at_row >= total || col >= p.d) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t nk = first / p.rows, n = nk / p.kv_heads;
  const XaRow r = xa_row(p, (int)(nk - n * p.kv_heads), first - nk * p.rows);
  const int64_t at = ((n * p.lq + r.qi) * (int64_t)(p.kv_heads * p.rep) + r.head) * p.d + col;
  if (p.o_dt == DT_BF16)
    *reinterpret_cast<u32x2*>((unsigned short*)p.out + at) = u32x2{pack2_bf16(o[0] * inv, o[1] * inv), pack2_bf16(o[2] * inv, o[3] * inv)};
  else
    *reinterpret_cast<f32x4*>((float*)p.out + at) = f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
}

}  // namespace

}  // namespace clarus
