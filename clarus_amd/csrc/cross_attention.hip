// Attention of one sequence of positions (pixels, or a few tokens) over the states of an encoder of
// another length, on gfx950:
//   o[q] = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  over the keys the mask keeps; 0 where it keeps none.
//
// One pass over the keys with the running maximum m and sum l of the softmax: a workgroup holds 128
// rows (4 waves x 32), takes K and V a tile at a time through LDS (double buffered, the next tile's
// loads in flight during the current one's products) and never writes a score to memory. A row is a
// query and one of the heads that share a kv head, so shared heads fill the tile of a single query.
//   S^T = K Q^T       a lane of a 32 x 32 MFMA holds one row's scores of 16 keys: maxima and sums
//                     need one exchange, with lane ^ 32
//   O^T = V^T P^T     P^T is the B operand as it is: lane l holds keys 8 (i / 4) + 4 (l / 32) + i % 4
//                     of each 16, and V^T is read in that order (bf16: transposing LDS reads; fp32: one
//                     float per lane), so P moves through no LDS
// m, l and O are fp32. bf16: products of bf16 q, k, v are exact in fp32; P is rounded once to bf16 for
// the product with V (half a step, 2^-9 relative per weight, of independent signs: the result's own
// rounding to bf16 is as large). fp32: every product runs on fp32 MFMAs.
// A masked or padding key's score is taken as -inf whatever its K holds, and its V row as 0.
// Few rows: the keys are split over workgroups, whose (O, m, l) xa_join_kernel joins.
#include "capi.hpp"
#include "common.hpp"

namespace clarus {

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr int XA_T = 256;    // threads
constexpr int XA_ROWS = 128; // rows of a workgroup
constexpr float XA_FLOOR = -3e38f;  // running maximum before any key: exp2(-inf - XA_FLOOR) = 0, no inf - inf

constexpr float XA_SLACK = 8.f;

enum : int { MASK_NONE = 0, MASK_KEYS = 1, MASK_PAIRS = 2 };

struct CrossP {
  const void *q, *k, *v;
  void* out;
  const unsigned char* mask;
  float* part;               // [split][nk][rows][D] O, then [split][nk][rows] m, then l
  int64_t qbs, ldq, kbs, ldk, vbs, ldv, mbs, mqs;
  int64_t rows;              // lq * rep
  int64_t lk, split_len, nk; // nk = n * kv_heads
  int64_t nblk;              // row blocks
  int lq, rep, kv_heads, d, splits, o_dt;
  float c;                   // scale log2(e)
};

// max / sum with lane ^ 32
__device__ __forceinline__ float xor32(float v) {
  return __shfl_xor(v, 32, 64);
}

template <int DT, int D>
struct XaTile {
  static constexpr int ES = DT == DT_BF16 ? 2 : 4;
  static constexpr int KT = DT == DT_BF16 ? 64 : 32;  // keys per tile
  static constexpr int ROWB = D * ES;                 // bytes of a row in LDS
  static constexpr int CPR = ROWB / 16;               // 16-byte chunks per row
  static constexpr int BYTES = KT * ROWB;
  static constexpr int NI = BYTES / 1024 / (XA_T / 64);  // 1 KiB copies per wave and operand
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

// what a masked, padding or absent piece of K or V is copied from
__device__ const u32x4 xa_zeros[1] = {u32x4{0, 0, 0, 0}};

// keep ? v : -inf, keep = bit `bit` of w (v may be NaN)
__device__ __forceinline__ float keep_bit(float v, unsigned w, int bit) {
  const unsigned k = (unsigned)__builtin_amdgcn_sbfe((int)w, bit, 1);
  return __uint_as_float((__float_as_uint(v) & k) | (0xff800000u & ~k));
}

template <int DT, int D, int MASK>
__global__ void __launch_bounds__(XA_T, D <= 64 ? 4 : 2) xa_kernel(const CrossP p) {
  using T = XaTile<DT, D>;
  constexpr int KT = T::KT, KB = KT / 32, DB = D / 32, ES = T::ES, NI = T::NI;
  constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xffffffffull;
  __shared__ __align__(16) unsigned char tiles[2][2 * T::BYTES];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hl = lane >> 5;
  // row blocks of one (image, kv head) run on one XCD, whose L2 then holds that head's K and V
  const int64_t total = p.nblk * p.nk * p.splits, span = (total + 7) >> 3;
  const int64_t id = (int64_t)(blockIdx.x & 7) * span + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= span || id >= total) return;
  const int64_t rb = id % p.nblk, hs = id / p.nblk;
  const int split = (int)(hs % p.splits);
  const int64_t nk = hs / p.splits;
  const int64_t n = nk / p.kv_heads;
  const int kvh = (int)(nk - n * p.kv_heads);

  const int64_t wrow = rb * XA_ROWS + wave * 32;  // the wave's first row
  const bool busy = wrow < p.rows;
  const int64_t row = wrow + col < p.rows ? wrow + col : p.rows - 1;  // rows past the end repeat the last one
  const int64_t qi = row / p.rep;
  const int head = kvh * p.rep + (int)(row - qi * p.rep);

  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)kvh * p.d) * ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)kvh * p.d) * ES;
  const unsigned char* mrow = MASK == MASK_PAIRS ? p.mask + n * p.mbs + qi * p.mqs : nullptr;
  const unsigned char* mkey = MASK == MASK_KEYS ? p.mask + n * p.mbs : nullptr;

  const int64_t k0 = (int64_t)split * p.split_len, k1 = k0 + p.split_len < p.lk ? k0 + p.split_len : p.lk;
  const int ntile = (int)((k1 - k0 + KT - 1) / KT);

  // this lane's piece of each copy: row and chunk of the tile, and its offset from the tile's first row
  uint32_t koff[NI], voff[NI];
  int rowc[NI];      // row
  bool have_k[NI], have_v[NI];  // the chunk lies within the head
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int at = (wave + (XA_T / 64) * j) * 1024 + lane * 16;
    const int r = at / T::ROWB, cpos = (at % T::ROWB) / 16;
    const int ck = cpos ^ T::swz_k(r), cv = cpos ^ T::swz_v(r);
    rowc[j] = r;
    koff[j] = (uint32_t)(r * p.ldk * ES) + ck * 16;
    voff[j] = (uint32_t)(r * p.ldv * ES) + cv * 16;
    have_k[j] = ck * 16 < p.d * ES;
    have_v[j] = cv * 16 < p.d * ES;
  }
  // the kept keys of a tile, one bit each. MASK_KEYS: the byte is loaded a tile ahead of its use
  auto key_byte = [&](int t) __attribute__((always_inline)) -> int {
    const int64_t key = k0 + (int64_t)t * KT + lane;
    const bool in = lane < KT && key < k1;
    if constexpr (MASK == MASK_KEYS) return in ? mkey[key] : 0;
    return in;
  };
  auto copy = [&](int t, uint64_t bits) __attribute__((always_inline)) {
    const int64_t base = k0 + (int64_t)t * KT;
    const unsigned char* kt = kp + base * p.ldk * ES;
    const unsigned char* vt = vp + base * p.ldv * ES;
    unsigned char* dst = tiles[t & 1] + wave * 1024;
#define XA_COPY(src, to)                                                                                   \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src),                  \
                                   (__attribute__((address_space(3))) void*)(to), 16, 0, 0)
    if (bits == ALL && p.d == D) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        XA_COPY(kt + koff[j], dst + j * (XA_T / 64) * 1024);
        XA_COPY(vt + voff[j], dst + T::BYTES + j * (XA_T / 64) * 1024);
      }
    } else {
      const unsigned char* zero = (const unsigned char*)xa_zeros;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const bool in = (bits >> rowc[j]) & 1;
        XA_COPY(in && have_k[j] ? kt + koff[j] : zero, dst + j * (XA_T / 64) * 1024);
        XA_COPY(in && have_v[j] ? vt + voff[j] : zero, dst + T::BYTES + j * (XA_T / 64) * 1024);
      }
    }
#undef XA_COPY
  };

  // Q^T fragments
  constexpr int QN = DT == DT_BF16 ? D / 16 : D / 8;  // 16-byte chunks per lane
  u32x4 qf[QN];
  {
    const unsigned char* qp = (const unsigned char*)p.q + (n * p.qbs + qi * p.ldq + (int64_t)head * p.d) * ES;
    constexpr int E = 16 / ES;
#pragma unroll
    for (int s = 0; s < QN; ++s) {
      const int at = (2 * s + hl) * E;
      qf[s] = at < p.d ? *reinterpret_cast<const u32x4*>(qp + at * ES) : u32x4{0, 0, 0, 0};
    }
  }

  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[b][j] = 0.f;
  float m = XA_FLOOR, l = 0.f;

  uint64_t bits = 0;
  int byte = 0;
  if (ntile > 0) {
    bits = __ballot(key_byte(0));
    if (ntile > 1) byte = key_byte(1);
    if (bits) copy(0, bits);
  }
  for (int t = 0; t < ntile; ++t) {
    const uint64_t now = bits;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies of tile t have landed
    barrier_keep_vm();                   // everybody's have, and tile t - 1 has been read
    if (t + 1 < ntile) {
      bits = __ballot(byte);
      if (t + 2 < ntile) byte = key_byte(t + 2);
      if (bits) copy(t + 1, bits);
    }
    if (!busy || !now) continue;
    const unsigned char* ks = tiles[t & 1];
    const unsigned char* vs = tiles[t & 1] + T::BYTES;
    unsigned pair[KB][4];
    if constexpr (MASK == MASK_PAIRS) {
      const int64_t base = k0 + (int64_t)t * KT;
      unsigned any = 0;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {
          const int64_t key = base + 32 * b + 8 * j4 + 4 * hl;
          unsigned w = 0;
          if (now == ALL) {
            __builtin_memcpy(&w, mrow + key, 4);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w |= (key + j < k1 ? (unsigned)mrow[key + j] : 0u) << (8 * j);
          }
          pair[b][j4] = w;
          any |= w;
        }
      if (!__any(any)) continue;
    }
    f32x16 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
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
    // masked and padding keys weigh nothing, whatever their scores
    if constexpr (MASK == MASK_PAIRS) {
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[b][j] = keep_bit(s[b][j], pair[b][j >> 2], 8 * (j & 3));
    } else if (now != ALL) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const unsigned w = (unsigned)(now >> (32 * b)) >> (4 * hl);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[b][j] = keep_bit(s[b][j], w, 8 * (j >> 2) + (j & 3));
      }
    }
    // the running maximum moves only when a score passes it by XA_SLACK (weights then stay below 2^XA_SLACK,
    // and fp32 sums keep their digits): the accumulators are rescaled in few tiles instead of all
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[b][j]);
    if (__any(mx * p.c > m + XA_SLACK)) {
      mx = fmaxf(mx, xor32(mx));
      const float mn = fmaxf(m, mx * p.c);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[b][j] *= alpha;
    }
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        s[b][j] = __builtin_amdgcn_exp2f(fmaf(s[b][j], p.c, -m));
        l += s[b][j];
      }
    if constexpr (DT == DT_BF16) {
      const int i = lane & 15;
      const int vr = 4 * hl + (i >> 2), vc = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
      for (int ks2 = 0; ks2 < KT / 16; ++ks2) {
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
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int r = 32 * kb + 8 * (j >> 2) + 4 * hl + (j & 3);
            const float a = *reinterpret_cast<const float*>(vs + T::at_v(r, 8 * b + (col >> 2)) + (col & 3) * 4);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[kb][j], o[b], 0, 0, 0);
          }
    }
  }
  if (!busy || wrow + col >= p.rows) return;
  l += xor32(l);
  if (p.splits > 1) {
    const int64_t at = ((int64_t)split * p.nk + nk) * p.rows + row, all = (int64_t)p.splits * p.nk * p.rows;
    float* po = p.part + at * D;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int j4 = 0; j4 < 4; ++j4)
        *reinterpret_cast<f32x4*>(po + 32 * b + 8 * j4 + 4 * hl) = f32x4{o[b][4 * j4], o[b][4 * j4 + 1], o[b][4 * j4 + 2], o[b][4 * j4 + 3]};
    if (hl == 0) {
      p.part[all * D + at] = m;
      p.part[all * (D + 1) + at] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = ((n * p.lq + qi) * (int64_t)(p.kv_heads * p.rep) + head) * p.d;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j4 = 0; j4 < 4; ++j4) {
      const int dd = 32 * b + 8 * j4 + 4 * hl;
      if (dd >= p.d) continue;
      const f32x4 y = f32x4{o[b][4 * j4] * inv, o[b][4 * j4 + 1] * inv, o[b][4 * j4 + 2] * inv, o[b][4 * j4 + 3] * inv};
      if (p.o_dt == DT_BF16)
        *reinterpret_cast<u32x2*>((unsigned short*)p.out + at + dd) = u32x2{pack2_bf16(y[0], y[1]), pack2_bf16(y[2], y[3])};
      else
        *reinterpret_cast<f32x4*>((float*)p.out + at + dd) = y;
    }
}

// one wave per row: the splits' (O, m, l) joined in split order
template <int D>
__global__ void __launch_bounds__(64) xa_join_kernel(const CrossP p) {
  const int64_t row = blockIdx.x, nk = blockIdx.y, all = (int64_t)p.splits * p.nk * p.rows;
  const int64_t step = p.nk * p.rows, first = nk * p.rows + row;
  const float *pm = p.part + all * D + first, *pl = p.part + all * (D + 1) + first;
  float m = XA_FLOOR;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, pm[s * step]);
  float l = 0.f;
  for (int s = 0; s < p.splits; ++s) l = fmaf(pl[s * step], __builtin_amdgcn_exp2f(pm[s * step] - m), l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t n = nk / p.kv_heads, qi = row / p.rep;
  const int head = (int)(nk - n * p.kv_heads) * p.rep + (int)(row - qi * p.rep);
  const int64_t at = ((n * p.lq + qi) * (int64_t)(p.kv_heads * p.rep) + head) * p.d;
  for (int dd = threadIdx.x; dd < p.d; dd += 64) {
    float o = 0.f;
    for (int s = 0; s < p.splits; ++s) o = fmaf(p.part[(first + s * step) * D + dd], __builtin_amdgcn_exp2f(pm[s * step] - m), o);
    store1(p.out, p.o_dt, at + dd, o * inv);
  }
}

int xa_pad(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

struct XaPlan {
  int64_t nblk, split_len;
  int splits;
};

XaPlan xa_plan(int32_t dt, int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads) {
  XaPlan g;
  const int kt = dt == DT_BF16 ? 64 : 32;
  g.nblk = cdiv(lq * (heads / kv_heads), XA_ROWS);
  const int64_t blocks = g.nblk * n * kv_heads;
  // split the keys while the row blocks leave CUs idle: two workgroups per CU, four tiles or more each
  int64_t want = 2LL * device_cus() / blocks;
  const int64_t most = cdiv(lk, 4 * kt);
  if (want > most) want = most;
  if (want < 1) want = 1;
  g.split_len = cdiv(cdiv(lk, want), kt) * kt;
  if (g.split_len < kt) g.split_len = kt;
  g.splits = (int)(lk > 0 ? cdiv(lk, g.split_len) : 1);
  return g;
}

template <int DT, int D>
void xa_launch(const CrossP& k, int mask, hipStream_t st) {
  const dim3 grid((unsigned)(8 * ((k.nblk * k.nk * k.splits + 7) / 8)));
  if (mask == MASK_NONE) hipLaunchKernelGGL((xa_kernel<DT, D, MASK_NONE>), grid, dim3(XA_T), 0, st, k);
  else if (mask == MASK_KEYS) hipLaunchKernelGGL((xa_kernel<DT, D, MASK_KEYS>), grid, dim3(XA_T), 0, st, k);
  else hipLaunchKernelGGL((xa_kernel<DT, D, MASK_PAIRS>), grid, dim3(XA_T), 0, st, k);
  if (k.splits > 1) hipLaunchKernelGGL((xa_join_kernel<D>), dim3((unsigned)k.rows, (unsigned)k.nk), dim3(64), 0, st, k);
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" size_t clarus_hip_cross_attention_workspace(int32_t dtype, int64_t n, int64_t lq, int64_t lk, int64_t heads,
                                                       int64_t kv_heads, int64_t d) {
  if (n <= 0 || lq <= 0 || lk < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || d <= 0 || d > 128) return 0;
  const XaPlan g = xa_plan(dtype, n, lq, lk, heads, kv_heads);
  return g.splits > 1 ? (size_t)g.splits * n * heads * lq * (xa_pad(d) + 2) * sizeof(float) : 0;
}

extern "C" int clarus_hip_cross_attention(const ClarusCrossArgs* a, void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  CLARUS_REQUIRE(a, "cross_attention: null arguments");
  CLARUS_REQUIRE(a->q && a->k && a->v && a->out, "cross_attention: null operand");
  CLARUS_REQUIRE(a->n > 0 && a->lq > 0 && a->lk > 0 && a->heads > 0 && a->kv_heads > 0, "cross_attention: empty problem");
  CLARUS_REQUIRE(a->heads % a->kv_heads == 0, "cross_attention: heads a multiple of kv_heads");
  CLARUS_REQUIRE(a->d >= 8 && a->d <= 128 && a->d % 8 == 0, "cross_attention: head width a multiple of 8, at most 128");
  CLARUS_REQUIRE((a->dtype == DT_BF16 || a->dtype == DT_F32) && (a->o_dtype == DT_BF16 || a->o_dtype == DT_F32),
                 "cross_attention: bf16 or fp32");
  CLARUS_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "cross_attention: scale positive and finite");
  const int64_t es = a->dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && a->ldq * es % 16 == 0 &&
                     a->ldk * es % 16 == 0 && a->ldv * es % 16 == 0 && a->q_bstride * es % 16 == 0 &&
                     a->k_bstride * es % 16 == 0 && a->v_bstride * es % 16 == 0,
                 "cross_attention: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldk < (1 << 24) && a->ldv < (1 << 24), "cross_attention: rows of k and v less than 2^24 elements apart");
  CLARUS_REQUIRE(a->ldq >= 0 && a->ldk >= 0 && a->ldv >= 0 && a->q_bstride >= 0 && a->k_bstride >= 0 && a->v_bstride >= 0,
                 "cross_attention: strides");
  CLARUS_REQUIRE(a->mask_mode >= MASK_NONE && a->mask_mode <= MASK_PAIRS && (a->mask_mode == MASK_NONE || a->mask),
                 "cross_attention: mask");
  CLARUS_REQUIRE(a->lq < ((int64_t)1 << 31) && a->lk < ((int64_t)1 << 31) && a->n * a->kv_heads < 65536 &&
                     a->lq * (a->heads / a->kv_heads) < ((int64_t)1 << 31),
                 "cross_attention: too large");
  const XaPlan g = xa_plan(a->dtype, a->n, a->lq, a->lk, a->heads, a->kv_heads);
  CLARUS_REQUIRE(8 * ((g.nblk * a->n * a->kv_heads * g.splits + 7) / 8) < ((int64_t)1 << 31), "cross_attention: too large");
  const size_t need = clarus_hip_cross_attention_workspace(a->dtype, a->n, a->lq, a->lk, a->heads, a->kv_heads, a->d);
  CLARUS_REQUIRE(need == 0 || (scratch && aligned(scratch, 16) && scratch_bytes >= need),
                 "cross_attention: scratch %zu < %zu bytes", scratch_bytes, need);
  CrossP k{};
  k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out; k.mask = (const unsigned char*)a->mask; k.part = (float*)scratch;
  k.qbs = a->q_bstride; k.ldq = a->ldq; k.kbs = a->k_bstride; k.ldk = a->ldk; k.vbs = a->v_bstride; k.ldv = a->ldv;
  k.mbs = a->mask_bstride; k.mqs = a->mask_qstride;
  k.rep = (int)(a->heads / a->kv_heads); k.kv_heads = (int)a->kv_heads; k.d = (int)a->d; k.lq = (int)a->lq;
  k.rows = a->lq * k.rep; k.lk = a->lk; k.nk = a->n * a->kv_heads;
  k.nblk = g.nblk; k.split_len = g.split_len; k.splits = g.splits;
  k.o_dt = a->o_dtype;
  k.c = a->scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const int D = xa_pad(a->d);
  note_kernel("xa_kernel d=%d splits=%d", D, g.splits);
#define CLARUS_XA(DT)                                        \
  do {                                                       \
    if (D == 32) xa_launch<DT, 32>(k, a->mask_mode, st);     \
    else if (D == 64) xa_launch<DT, 64>(k, a->mask_mode, st); \
    else if (D == 96) xa_launch<DT, 96>(k, a->mask_mode, st); \
    else xa_launch<DT, 128>(k, a->mask_mode, st);            \
  } while (0)
  if (a->dtype == DT_BF16) CLARUS_XA(DT_BF16);
  else CLARUS_XA(DT_F32);
#undef CLARUS_XA
  return check_launch("cross_attention");
}
