// Causal linear attention with a decay for each head, from a state and to one, on gfx950; per image and kv head
//   S_t = e^g S_{t-1} + k_t v_t^T,   o_t[h] = scale q_t[h]^T S_t   for the heads h that share the kv head.
//
//   la_step_kernel   a few tokens: the state in registers, read and written once, token after token
//   la_chunk_kernel  longer sequences, in segments of whole chunks of 64 (fp32: 32) tokens. Within a chunk
//                      o_i = e^{g (i + 1)} q_i^T S + sum_{j <= i} e^{g (i - j)} (q_i . k_j) v_j,
//                      S <- e^{g c} S + sum_j e^{g (c - 1 - j)} k_j v_j^T
//                    as matrix products; once without outputs for what a segment adds to the state, once from the
//                    state that it starts with
//   la_carry_kernel  the segments' start states, and the state after the last
// A sequence that is no whole number of chunks is padded in front (k, v = 0), so that every factor is a power of e^g with
// an exponent that is not negative. States, sums and factors are fp32 (a segment's factor is kept as two fp32 numbers from
// 64 bits, and the factors of its chunks make up for each other's rounding: a state held over many calls, segments and chunks
// does not drift by it).
//
// A wave holds 32 columns of values: S as MFMA accumulators, rows dk. As an A operand (rows = values) the accumulators
// stand as they are for S^T, in the order of dk in which q's fragments are put by exchanging halves with lane ^ 32; P^T
// goes from the accumulators of K Q^T into the product with V^T likewise, and V^T is both that product's operand and,
// weighted, the state's. bf16: products of bf16 q, k, v are exact in fp32; the weighted values go in three bf16 parts
// (2^-24 of them left out) where a segment's sum for the state is made, in two (2^-16) where only outputs follow, S in two
// as an operand, and the weights q . k within a chunk are rounded once to bf16 (2^-8 of each, of independent
// signs: about as much as the output's own rounding). fp32: every product on fp32 MFMAs.
//
// What bounds it: a token, memory (64 states of 16 heads of 128 x 128: 28.7 us, 4.7 TB/s). Chunks: K and V read twice, and a
// wave's chain from chunk to chunk; 57600 tokens, 8 heads of 64 x 64, bf16: 34.6 us for the segments' sums, 9.1 for the chain
// of segments, 66 for the outputs (236 MB in all: 46 us at a large copy's rate); 2 x 5003 of 48 x 96, 8 heads on 4, fp32: 14.6,
// 6.7 and 51.3, of which the fp32 MFMAs alone are some 31 where two of the 1272 waves share a SIMD. Keys of
// 128 in bf16: 28800 tokens, 8 heads of 128 x 128: 44, 16 and 156, where the output pass spills 112 to 121 of its
// VGPRs (fp32 keys of 96: 53 to 55; other forms 11 at most).
#include <algorithm>
#include <math.h>

#include "attention_tile.hpp"
#include "capi.hpp"

namespace clarus {

namespace {

constexpr int LA_T = 256;  // threads of a step or carry workgroup
constexpr float LA_LEAST = -1000.f;  // log2 of a decay: 2^-1000 is 0 in fp32, and 0 times it no NaN

struct LinP {
  const void *q, *k, *v;
  void* out;
  const float *s_in, *decay;
  float *s_out, *part;
  int* careful;          // segments with values that are not finite, for each wave's columns
  int64_t qbs, ldq, kbs, ldk, vbs, ldv;
  int64_t l;             // tokens
  int64_t nk, nseg, seg; // (image, kv head) pairs, segments, tokens of one
  int64_t pad;           // in front of the first token
  int rep, kv_heads, dk, dv, o_dt;
  int slices;            // of the values' columns (step)
  float scale;
};

// log2 of a head's decay
__device__ __forceinline__ float la_log2(const LinP& p, int h) {
  const float g = p.decay[h] * 1.4426950408889634f;
  return g < LA_LEAST ? LA_LEAST : g;
}

// e^{g n} as two floats
struct Factor { float hi, lo; };
__device__ __forceinline__ Factor la_factor(const LinP& p, int h, int64_t n) {
  double e = (double)p.decay[h] * (double)n * 1.4426950408889634074;
  e = n == 0 ? 0.0 : e < (double)LA_LEAST ? (double)LA_LEAST : e;
  const double f = exp2(e);
  Factor r;
  r.hi = (float)f;
  r.lo = r.hi < 3e38f ? (float)(f - (double)r.hi) : 0.f;
  return r;
}
__device__ __forceinline__ float la_scaled(float s, const Factor& f, float add) { return fmaf(s, f.hi, fmaf(s, f.lo, add)); }

// ---------------------------------------------------------------- a few tokens
// A workgroup holds DVS columns of a state, a thread four of them in NP rows RG apart
template <int DT, int DVS, int NP>
__global__ void __launch_bounds__(LA_T) la_step_kernel(const LinP p) {
  constexpr int TPR = DVS / 4, RG = LA_T / TPR, ES = DT == DT_BF16 ? 2 : 4;
  __shared__ float ks[RG * NP], qs[RG * NP];
  __shared__ f32x4 po[LA_T];
  const int tid = threadIdx.x, rg = tid / TPR, c4 = tid - rg * TPR;
  const int64_t nk = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - nk * p.slices);
  const int64_t n = nk / p.kv_heads;
  const int h = (int)(nk - n * p.kv_heads), col = slice * DVS + c4 * 4;
  const bool mine = col < p.dv;
  const Factor f = la_factor(p, h, 1);
  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)h * p.dk) * ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)h * p.dv) * ES;
  f32x4 s[NP];
  const int64_t at = nk * p.dk * p.dv + col;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = rg + RG * i;
    s[i] = p.s_in && mine && r < p.dk ? *reinterpret_cast<const f32x4*>(p.s_in + at + (int64_t)r * p.dv) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int64_t t = 0; t < p.l; ++t) {
    __syncthreads();
    for (int i = tid; i < RG * NP; i += LA_T) ks[i] = i < p.dk ? load1(kp, DT, t * p.ldk + i) : 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (mine)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = load1(vp, DT, t * p.ldv + col + e);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float k = ks[rg + RG * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = la_scaled(s[i][e], f, k * v[e]);
    }
    for (int r = 0; r < p.rep; ++r) {
      const int head = h * p.rep + r;
      const unsigned char* qp = (const unsigned char*)p.q + (n * p.qbs + t * p.ldq + (int64_t)head * p.dk) * ES;
      if (r) __syncthreads();
      for (int i = tid; i < RG * NP; i += LA_T) qs[i] = i < p.dk ? load1(qp, DT, i) : 0.f;
      __syncthreads();
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float q = qs[rg + RG * i];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(q, s[i][e], o[e]);
      }
      po[tid] = o;
      __syncthreads();
      if (rg == 0 && mine) {
        for (int i = 1; i < RG; ++i) o += po[tid + i * TPR];
        const int64_t to = ((n * p.l + t) * (int64_t)(p.kv_heads * p.rep) + head) * p.dv + col;
        if (p.o_dt == DT_BF16)
          *reinterpret_cast<u32x2*>((unsigned short*)p.out + to) =
              u32x2{pack2_bf16(o[0] * p.scale, o[1] * p.scale), pack2_bf16(o[2] * p.scale, o[3] * p.scale)};
        else
          *reinterpret_cast<f32x4*>((float*)p.out + to) = o * p.scale;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = rg + RG * i;
    if (mine && r < p.dk) *reinterpret_cast<f32x4*>(p.s_out + at + (int64_t)r * p.dv) = s[i];
  }
}

// ---------------------------------------------------------------- chunks
// Tokens of a chunk: 64 in bf16, 32 in fp32 and with wide keys in bf16, whose state and queries fill the registers
template <int DT, int DK> constexpr int la_kt = DT == DT_BF16 && DK <= 32 ? 64 : 32;

// The copies of one tile (KT tokens, D columns of LDS) by W waves, 1 KiB each
template <int DT, int D, int KT, int W>
struct LaCopy {
  using T = XaTile<DT, D>;
  static constexpr int BYTES = KT * T::ROWB, NI = (BYTES / 1024 + W - 1) / W;
  static constexpr bool EVEN = BYTES / 1024 % W == 0;
  uint32_t off[NI];  // from the tile's first row

  __device__ __forceinline__ LaCopy(int64_t ld, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int at = (wave + W * j) * 1024 + lane * 16, r = at / T::ROWB, c = ((at % T::ROWB) / 16) ^ T::swz_k(r);
      off[j] = (uint32_t)(r * ld * T::ES) + c * 16;
    }
  }
  // rows before `pad` and columns from d on as zeros
  __device__ __forceinline__ void operator()(const unsigned char* src, int d, int pad, unsigned char* dst, int wave, int lane) const {
#define LA_COPY(from)                                                                          \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from),     \
                                   (__attribute__((address_space(3))) void*)(dst + (wave + W * j) * 1024), 16, 0, 0)
    if (pad == 0 && d == D) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= BYTES / 1024) break;
        LA_COPY(src + off[j]);
      }
    } else {
      const unsigned char* zero = (const unsigned char*)xa_zeros;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= BYTES / 1024) break;
        const int at = (wave + W * j) * 1024 + lane * 16, r = at / T::ROWB, c = ((at % T::ROWB) / 16) ^ T::swz_k(r);
        LA_COPY(r >= pad && c * 16 < d * T::ES ? src + off[j] : zero);
      }
    }
#undef LA_COPY
  }
};

// 32 x 16 fragment of a tile's transpose (rows = columns 32 b .. of the tile, 16 tokens 16 ks ..), tokens in the order of
// the accumulators
template <int D>
__device__ __forceinline__ bf16x8 la_turned(const unsigned char* tile, int ks, int b, int lane) {
  using T = XaTile<DT_BF16, D>;
  typedef __attribute__((ext_vector_type(8))) short s16x8;
  const int i = lane & 15, vr = 16 * ks + 4 * (lane >> 5) + (i >> 2), vc = 4 * b + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(tile + T::at_k(vr, vc) + (i & 1) * 8));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(tile + T::at_k(vr + 8, vc) + (i & 1) * 8));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ f32x16 la_mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// chunks in LDS: the one at work and the next (fp32), or the next two on their way (bf16); K, V and Q of the first head
template <int DT, int DK, int W, bool OUT>
struct LaChunk {
  static constexpr int KT = la_kt<DT, DK>, BUFS = DT == DT_BF16 ? 3 : 2, KBYTES = KT * XaTile<DT, DK>::ROWB,
                       VBYTES = KT * XaTile<DT, 32 * W>::ROWB, QBYTES = OUT ? KBYTES : 0, BYTES = KBYTES + VBYTES + QBYTES;
};

// W waves, 32 columns of values each. OUT: outputs, from the segment's start state; else what the segment adds.
// CAREFUL: for a segment with values that are not finite. The weight 0 that such a value has for the queries before it would
// make them NaN, so the product gets a 0 in its place, and the outputs from its token on are NaN.
template <int DT, int DK, int W, bool OUT, bool CAREFUL>
__device__ __forceinline__ void la_chunks(const LinP& p, const unsigned n, const unsigned h, const unsigned seg,
                                          unsigned char (*tiles)[LaChunk<DT, DK, W, OUT>::BYTES]) {
  using TK = XaTile<DT, DK>;
  using TV = XaTile<DT, 32 * W>;
  using L = LaChunk<DT, DK, W, OUT>;
  constexpr int KT = L::KT, QT = KT / 32, DB = DK / 32, QN = xa_qn<DT, DK>, ES = TK::ES;
  constexpr int KBYTES = L::KBYTES, VBYTES = L::VBYTES, QBYTES = L::QBYTES, BUFS = L::BUFS, AHEAD = BUFS - 1;
  const int tid = threadIdx.x, lane0 = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane0 & 31, hl = lane0 >> 5;
  const int64_t nk = (int64_t)n * p.kv_heads + h;
  // padded places: token = place - pad
  const int64_t t0 = seg * p.seg, t1 = t0 + p.seg < p.l + p.pad ? t0 + p.seg : p.l + p.pad;
  const int nchunk = (int)((t1 - t0) / KT);

  const float g = la_log2(p, h);
  f32x16 s[DB];
  float* part = p.part + ((nk * p.nseg + seg) * W + wave) * (DB * 16 * 64) + lane0;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) s[b][j] = OUT ? part[(b * 16 + j) * 64] : 0.f;
  // e^{g (c - 1 - r)} of row r = 16 ks + 8 (i / 4) + 4 hl + i % 4 of a chunk (fp32: 16 values of i)
  float fi[DT == DT_BF16 ? 8 : 16], fk[KT / 16];
  constexpr int LAST = DT == DT_BF16 ? 15 : KT - 1;
#pragma unroll
  for (int i = 0; i < (DT == DT_BF16 ? 8 : 16); ++i) fi[i] = __builtin_amdgcn_exp2f(g * (float)(LAST - (8 * (i >> 2) + 4 * hl + (i & 3))));
#pragma unroll
  for (int i = 0; i < KT / 16; ++i) fk[i] = __builtin_amdgcn_exp2f(g * (float)(KT - 16 - 16 * i));
  // e^{g (i - j)} of query i = col of a tile of 32 and key j of the same tile (0 behind the query), and of the one before
  float same[OUT ? 16 : 1], before[OUT && QT == 2 ? 16 : 1];
  if constexpr (OUT) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int gap = col - (8 * (j >> 2) + 4 * hl + (j & 3));
      same[j] = gap >= 0 ? __builtin_amdgcn_exp2f(g * (float)gap) : 0.f;
      if constexpr (QT == 2) before[j] = __builtin_amdgcn_exp2f(g * (float)(gap + 32));
    }
  }
  const float whole = __builtin_amdgcn_exp2f(g * (float)KT);
  // `whole` is off by up to 2^-24 of itself, chunk after chunk to the same side, by `lack` (e^x - 1 by its series; past x = -1/2 a
  // state does not last for it to show). What the chunks so far lack is added to the next one's factor, which rounds to a neighbour of
  // `whole` when it is half a step: factors of a long segment are as exact together as one. Of a state 625 chunks old: up to
  // 140 x 2^-24 off without, its roundings' 15 x 2^-24 with it
  const float x = p.decay[h] * (float)KT;
  const float e = 1.f + x * (1.f / 2 + x * (1.f / 6 + x * (1.f / 24 + x * (1.f / 120 + x * (1.f / 720 + x * (1.f / 5040 + x / 40320))))));
  const float lack = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fabsf(x) < 0.5f ? x * e - (whole - 1.f) : 0.f)));
  float lacking = 0.f;

  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)h * p.dk) * ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)h * p.dv) * ES;
  const LaCopy<DT, DK, KT, W> copy_k(p.ldk, wave, lane0), copy_q(p.ldq, wave, lane0);
  const LaCopy<DT, 32 * W, KT, W> copy_v(p.ldv, wave, lane0);
  const unsigned char* qp0 = (const unsigned char*)p.q + (n * p.qbs + (int64_t)h * p.rep * p.dk) * ES;
  auto fill = [&](int c) __attribute__((always_inline)) {
    const int64_t at = t0 + (int64_t)c * KT - p.pad;  // token of the chunk's first place, negative in the padding
    const int pad = at < 0 ? (int)-at : 0;
    unsigned char* to = tiles[c % BUFS];
    copy_k(kp + at * p.ldk * ES, p.dk, pad, to, wave, lane0);
    copy_v(vp + at * p.ldv * ES, p.dv, pad, to + KBYTES, wave, lane0);
    if constexpr (OUT) copy_q(qp0 + at * p.ldq * ES, p.dk, pad, to + KBYTES + VBYTES, wave, lane0);
  };
  // what a wave issues at least for a chunk: with as many operations in flight, the chunk before has landed
  constexpr int COPIES = KBYTES / 1024 / W + VBYTES / 1024 / W + QBYTES / 1024 / W;
#pragma unroll
  for (int c = 0; c < AHEAD; ++c)
    if (c < nchunk) fill(c);
#pragma unroll 1
  for (int c = 0; c < nchunk; ++c) {
    // LDS and output offsets are worked out for each chunk instead of kept over the loop, where they spill
    int lane = lane0;
    asm volatile("" : "+v"(lane));
    const int col = lane & 31, hl = lane >> 5;
    const int64_t first = t0 + (int64_t)c * KT - p.pad;
    const int pad = first < 0 ? (int)-first : 0;
    // this wave's copies of the chunk have landed, the next one's may be on their way
    if (AHEAD == 2 && c + 1 < nchunk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COPIES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    barrier_keep_vm();  // everybody's have, and the chunk before has been read
    const unsigned char *kt = tiles[c % BUFS], *vt = kt + KBYTES, *qt = vt + VBYTES;
    if (BUFS == 2 && c + 1 < nchunk) fill(c + 1);
    bf16x8 vf[DT == DT_BF16 ? KT / 16 : 1];
    float vx[DT == DT_BF16 ? 1 : 16];
    if constexpr (DT == DT_BF16) {
#pragma unroll
      for (int ks = 0; ks < KT / 16; ++ks) vf[ks] = la_turned<32 * W>(vt, ks, wave, lane);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        vx[j] = *reinterpret_cast<const float*>(vt + TV::at_k(8 * (j >> 2) + 4 * hl + (j & 3), 8 * wave + (col >> 2)) + (col & 3) * 4);
    }
    int bad = KT;  // the first token whose value in this lane's column is not finite
    if constexpr (CAREFUL) {
      if constexpr (DT == DT_BF16) {
#pragma unroll
        for (int ks = KT / 16 - 1; ks >= 0; --ks)
#pragma unroll
          for (int e = 7; e >= 0; --e)
            if (!(fabsf((float)vf[ks][e]) < INFINITY)) {
              bad = 16 * ks + 8 * (e >> 2) + 4 * hl + (e & 3);
              vf[ks][e] = (bf16_t)0.f;
            }
      } else {
#pragma unroll
        for (int j = 15; j >= 0; --j)
          if (!(fabsf(vx[j]) < INFINITY)) {
            bad = 8 * (j >> 2) + 4 * hl + (j & 3);
            vx[j] = 0.f;
          }
      }
      const int other = __shfl_xor(bad, 32);
      bad = other < bad ? other : bad;
    }
    if constexpr (OUT) {
#pragma unroll 1
      for (int r = 0; r < p.rep; ++r) {
        u32x4 qf[QT][QN];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int64_t token = first + 32 * t + col;
          const unsigned char* qp = qp0 + ((token < 0 ? 0 : token) * p.ldq + (int64_t)r * p.dk) * ES;
#pragma unroll
          for (int i = 0; i < QN; ++i) {
            if (r == 0) {
              qf[t][i] = *reinterpret_cast<const u32x4*>(qt + TK::at_k(32 * t + col, 2 * i + hl));
            } else {
              const int at = (2 * i + hl) * (16 / ES);
              qf[t][i] = *reinterpret_cast<const u32x4*>(qp + (at < p.dk ? at : 0) * ES);
              if (p.dk < DK && at >= p.dk) qf[t][i] = u32x4{0, 0, 0, 0};
            }
          }
        }
        f32x16 o[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[t][j] = 0.f;
        // S^T Q^T
        if constexpr (DT == DT_BF16) {
#pragma unroll
          for (int i = 0; i < QN; ++i) {
            f32x8 x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[e] = s[i >> 1][8 * (i & 1) + e];
            bf16x8 hi, lo;
            split_bf16(x, hi, lo);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              unsigned x0 = qf[t][i][0], x1 = qf[t][i][1], y0 = qf[t][i][2], y1 = qf[t][i][3];
              swap32(x0, y0);
              swap32(x1, y1);
              const bf16x8 q = __builtin_bit_cast(bf16x8, u32x4{x0, x1, y0, y1});
              o[t] = la_mfma(hi, q, o[t]);
              o[t] = la_mfma(lo, q, o[t]);
            }
          }
        } else {
#pragma unroll
          for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              o[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(s[b][j], __uint_as_float(qf[0][4 * b + (j >> 2)][j & 3]), o[0], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int since = 32 * t + col + 1 - pad;
          const float f = __builtin_amdgcn_exp2f(g * (float)(since > 0 ? since : 0));
#pragma unroll
          for (int j = 0; j < 16; ++j) o[t][j] *= f;
        }
        __builtin_amdgcn_sched_barrier(0);
        // P^T = (K Q^T) weighted, O^T += V^T P^T
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int b = 0; b <= t; ++b) {
            f32x16 w;
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = 0.f;
#pragma unroll
            for (int i = 0; i < QN; ++i) {
              const u32x4 a = *reinterpret_cast<const u32x4*>(kt + TK::at_k(32 * b + col, 2 * i + hl));
              if constexpr (DT == DT_BF16) {
                w = la_mfma(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, qf[t][i]), w);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(qf[t][i][e]), w, 0, 0, 0);
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (b != t) w[j] *= before[QT == 2 ? j : 0];
              else w[j] = col >= 8 * (j >> 2) + 4 * hl + (j & 3) ? w[j] * same[j] : 0.f;  // whatever a later key holds
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (DT == DT_BF16) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                f32x8 x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x.v[e] = w[8 * half + e];
                o[t] = la_mfma(vf[2 * b + half], pack_bf16(x), o[t]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(vx[j], w[j], o[t], 0, 0, 0);
            }
          }
        if constexpr (CAREFUL) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int from = __shfl(bad, 8 * (j >> 2) + 4 * hl + (j & 3));
#pragma unroll
            for (int t = 0; t < QT; ++t)
              if (32 * t + col >= from) o[t][j] = NAN;
          }
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const bool live = 32 * t + col >= pad;
          const int64_t at = ((n * p.l + first + 32 * t + col) * (int64_t)(p.kv_heads * p.rep) + h * p.rep + r) * p.dv + 32 * wave;
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            f32x4 y[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i >> 2][i & 3] = o[t][j + i] * p.scale;
            if (p.o_dt == DT_BF16) {
              unsigned a0 = pack2_bf16(y[0][0], y[0][1]), a1 = pack2_bf16(y[0][2], y[0][3]), b0 = pack2_bf16(y[1][0], y[1][1]),
                       b1 = pack2_bf16(y[1][2], y[1][3]);
              swap32(a0, b0);
              swap32(a1, b1);
              const int c8 = 2 * j + 8 * hl;
              if (live && 32 * wave + c8 < p.dv) *reinterpret_cast<u32x4*>((unsigned short*)p.out + at + c8) = u32x4{a0, a1, b0, b1};
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int c4 = 2 * j + 8 * i + 4 * hl;
                if (live && 32 * wave + c4 < p.dv) *reinterpret_cast<f32x4*>((float*)p.out + at + c4) = y[i];
              }
            }
          }
        }
      }
      if (c + 1 == nchunk) break;  // no output needs the state behind the last chunk
    }
    __builtin_amdgcn_sched_barrier(0);
    // the state behind this chunk
    float keep = whole + (lacking + lack);
    if (pad) keep = __builtin_amdgcn_exp2f(g * (float)(KT - pad));
    else lacking = lacking + lack - (keep - whole);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] *= keep;
    if constexpr (DT == DT_BF16) {
#pragma unroll
      for (int ks = 0; ks < KT / 16; ++ks) {
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = (float)vf[ks][e] * (fi[e] * fk[ks]);
        bf16x8 part3[3];
        split_bf16(x, part3[0], part3[1]);
        if constexpr (!OUT) {
#pragma unroll
          for (int e = 0; e < 8; ++e) part3[2][e] = (bf16_t)(x.v[e] - (float)part3[0][e] - (float)part3[1][e]);
        }
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          const bf16x8 a = la_turned<DK>(kt, ks, b, lane);
#pragma unroll
          for (int i = 0; i < (OUT ? 2 : 3); ++i) s[b] = la_mfma(a, part3[i], s[b]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = vx[j] * fi[j];
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          const float a = *reinterpret_cast<const float*>(kt + TK::at_k(8 * (j >> 2) + 4 * hl + (j & 3), 8 * b + (col >> 2)) + (col & 3) * 4);
          s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x, s[b], 0, 0, 0);
        }
      }
    }
    if (CAREFUL && bad < KT) {
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[b][j] = NAN;
    }
    // behind the outputs' stores, which the wait above would else wait for too
    if (AHEAD == 2 && c + 2 < nchunk) fill(c + 2);
  }
  if constexpr (!OUT) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(b * 16 + j) * 64] = s[b][j];
    // a value that is not finite leaves no row of its column finite
    const bool careful = __any(!(fabsf(s[0][0]) < INFINITY));
    if (lane0 == 0) p.careful[(nk * p.nseg + seg) * W + wave] = careful;
  }
}

template <int DT, int DK, int W, bool OUT>
__global__ void __launch_bounds__(64 * W, 2) la_chunk_kernel(const LinP p) {
  using L = LaChunk<DT, DK, W, OUT>;
  __shared__ __align__(16) unsigned char tiles[L::BUFS][L::BYTES];
  // neighbouring heads of a segment, which share lines of rows, on one XCD
  const unsigned total = (unsigned)(p.nk * p.nseg), span = (total + 7) >> 3, id = (blockIdx.x & 7) * span + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= span || id >= total) return;
  const unsigned rest = id / (unsigned)p.kv_heads, h = id - rest * (unsigned)p.kv_heads;
  const unsigned n = rest / (unsigned)p.nseg, seg = rest - n * (unsigned)p.nseg;
  if constexpr (OUT) {
    int careful = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) careful |= p.careful[(((int64_t)n * p.kv_heads + h) * p.nseg + seg) * W + w];
    if (__builtin_amdgcn_readfirstlane(careful)) {
      la_chunks<DT, DK, W, true, true>(p, n, h, seg, tiles);
      return;
    }
  }
  la_chunks<DT, DK, W, OUT, false>(p, n, h, seg, tiles);
}

// In place of what each segment adds the state that it starts with; the state behind the last. A workgroup takes LA_T / G elements
// (in the accumulators' order) and G x N segments at a time: a thread has N of them of one element in registers,
// and the G groups are chained through LDS (57600 tokens in 120 segments, 8 heads of 64 x 64: 9.1 us with G = 8, 15.0 with a
// thread per element and chain, the next 8 segments in flight). As few as there are segments for (1024 states of
// 128 x 128, one segment: 88 us with G = N = 1, 235 with N = 16, 1542 with G = 8 too)
constexpr int LA_GROUP = 16, LA_MOST = 8;

template <int G, int N>
__global__ void __launch_bounds__(LA_T) la_carry_kernel(const LinP p, int waves, int db) {
  constexpr int E = LA_T / G;
  __shared__ float sums[G][E];
  __shared__ Factor facts[G + 3];  // of the groups; of the first segment, one between, the last
  const unsigned per = waves * db * 16 * 64;  // elements of a state, padded
  const int tid = threadIdx.x, grp = tid / E;
  const unsigned nk = blockIdx.x / (per / E), e = (blockIdx.x - nk * (per / E)) * E + tid % E, h = nk % (unsigned)p.kv_heads;
  const int lane = e & 63, reg = (e >> 6) % (unsigned)(db * 16), wave = e / (unsigned)(db * 16 * 64), j = reg & 15;
  const int r = 32 * (reg >> 4) + 8 * (j >> 2) + 4 * (lane >> 5) + (j & 3), c = 32 * wave + (lane & 31);
  const bool in = r < p.dk && c < p.dv;
  const int64_t at = (int64_t)nk * p.dk * p.dv + (int64_t)r * p.dv + c;
  auto token = [&](int64_t s) __attribute__((always_inline)) {  // before segment s
    const int64_t t = (s < p.nseg ? s : p.nseg) * p.seg - p.pad;
    return t < 0 ? 0 : t < p.l ? t : p.l;
  };
  float* part = p.part + (int64_t)nk * p.nseg * per + e;
  float s = p.s_in && in ? p.s_in[at] : 0.f;
#pragma unroll 1
  for (int64_t r0 = 0; r0 < p.nseg; r0 += N * G) {
    const int64_t s0 = r0 + grp * N;
    const int mine = (int)(p.nseg - s0 < 0 ? 0 : p.nseg - s0 < N ? p.nseg - s0 : N);
    float add[N];
#pragma unroll
    for (int k = 0; k < N; ++k) add[k] = part[(s0 + k < p.nseg ? s0 + k : p.nseg - 1) * per];
    __syncthreads();  // the groups before have been read
    if (tid < G + 3) {
      const int64_t a = tid < G ? r0 + tid * N : tid == G ? 0 : tid == G + 1 ? 1 : p.nseg - 1;
      const int64_t b = tid < G ? a + N : a + 1;
      facts[tid] = la_factor(p, h, tid == G + 1 ? p.seg : token(b) - token(a));
    }
    __syncthreads();
    // the first and the last segment's may differ from the others'
    const float fh = facts[G + 1].hi, fl = facts[G + 1].lo;
    const float h0 = s0 == 0 ? facts[G].hi : fh, l0 = s0 == 0 ? facts[G].lo : fl;
    const int end = p.nseg - 1 - s0 < N && p.nseg - 1 > 0 ? (int)(p.nseg - 1 - s0) : -1;
    const float h1 = facts[G + 2].hi, l1 = facts[G + 2].lo;
    auto step = [&](float v, int k) __attribute__((always_inline)) {
      const float hi = k == end ? h1 : k == 0 ? h0 : fh, lo = k == end ? l1 : k == 0 ? l0 : fl;
      return fmaf(v, hi, fmaf(v, lo, add[k]));
    };
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) v = k < mine ? step(v, k) : v;
    sums[grp][tid % E] = v;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g == grp) v = s;  // what this group starts with
      s = fmaf(s, facts[g].hi, fmaf(s, facts[g].lo, sums[g][tid % E]));
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < mine) {
        part[(s0 + k) * per] = v;
        v = step(v, k);
      }
  }
  if (grp == 0 && in) p.s_out[at] = s;
}

struct LaPlan {
  bool chunks;
  int64_t seg, nseg, pad;
  int waves, slice;  // of values: waves of 32 columns; columns of a step workgroup
  size_t part, flags;  // bytes of scratch
};

// Token by token a step of the state and one of each head's output, in chunks three launches, whatever the length up to a
// chunk. us token by token / in chunks, bf16: 8 states of 64 x 64 8.7 / 15 (4 tokens), 14 / 15 (8), 25 / 15 (16); 32 with 4
// heads each 20 / 19 (4), 38 / 19 (8), 256 39 / 24 (8); 32 in fp32 14 / 20 (8), 24 / 19 (16). Where moving the states is
// most of the time: 1024 of 128 x 128 60 / 138 (8), 96 / 141 (16), 170 / 143 (32). States that are too many for a grid of
// pieces stay with the first.
bool la_by_token(int64_t nk, int64_t l, int64_t rep, int64_t dk, int64_t dv) {
  if (nk * cdiv(dv, 32) * cdiv(dk, 32) >= 1 << 18) return true;
  return l * (1 + rep) <= (nk * dk * dv >= 1 << 22 ? 40 : 20);
}

LaPlan la_plan(int32_t dt, int64_t n, int64_t l, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv) {
  LaPlan g{};
  const int64_t nk = n * kv_heads;
  if (la_by_token(nk, l, heads / kv_heads, dk, dv)) {
    g.slice = dv <= 32 ? 32 : dv <= 64 ? 64 : 128;
    while (g.slice > 32 && nk * cdiv(dv, g.slice) < 2 * device_cus()) g.slice /= 2;
    return g;
  }
  const int64_t kt = dt == DT_BF16 && dk <= 32 ? 64 : 32, chunks = cdiv(l, kt);
  g.chunks = true;
  g.waves = (int)cdiv(dv, 32);
  g.pad = chunks * kt - l;
  // as many segments as run at once, two waves per SIMD: the slowest of two rounds would be the time
  const int64_t want = device_cus() * (8 / g.waves) / nk;
  g.seg = cdiv(chunks, std::max<int64_t>(std::min(want, cdiv(chunks, 2)), 1)) * kt;
  g.nseg = cdiv(chunks * kt, g.seg);
  g.part = (size_t)(nk * g.nseg) * g.waves * cdiv(dk, 32) * 4096;
  g.flags = (size_t)(nk * g.nseg) * g.waves * 4;
  return g;
}

bool la_fits(int64_t n, int64_t l, int64_t heads, int64_t kv_heads) {
  return n < (1 << 20) && kv_heads < (1 << 20) && n * kv_heads < (1 << 20) && heads < (1 << 20) && l < ((int64_t)1 << 31);
}

template <int DT, int DK, int W>
void la_launch(const LinP& k, hipStream_t st) {
  const dim3 grid((unsigned)(8 * cdiv(k.nk * k.nseg, 8)));
  constexpr int DB = DK / 32;
  hipLaunchKernelGGL((la_chunk_kernel<DT, DK, W, false>), grid, dim3(64 * W), 0, st, k);
  const unsigned states = (unsigned)(k.nk * W * DB * 4);  // in pieces of LA_T elements
#define CLARUS_CARRY(G, N) hipLaunchKernelGGL((la_carry_kernel<G, N>), dim3(G * states), dim3(LA_T), 0, st, k, W, DB)
  if (k.nseg == 1) CLARUS_CARRY(1, 1);
  else if (k.nseg <= 4) CLARUS_CARRY(1, 4);
  else if (k.nseg <= LA_GROUP) CLARUS_CARRY(1, LA_GROUP);
  else if (k.nseg <= 2 * LA_GROUP) CLARUS_CARRY(2, LA_GROUP);
  else if (k.nseg <= 4 * LA_GROUP) CLARUS_CARRY(4, LA_GROUP);
  else CLARUS_CARRY(LA_MOST, LA_GROUP);
#undef CLARUS_CARRY
  hipLaunchKernelGGL((la_chunk_kernel<DT, DK, W, true>), grid, dim3(64 * W), 0, st, k);
}

template <int DT, int DK>
void la_launch_dk(const LinP& k, int waves, hipStream_t st) {
  if (waves == 1) la_launch<DT, DK, 1>(k, st);
  else if (waves == 2) la_launch<DT, DK, 2>(k, st);
  else if (waves == 3) la_launch<DT, DK, 3>(k, st);
  else la_launch<DT, DK, 4>(k, st);
}

template <int DT>
void la_launch_dt(const LinP& k, const LaPlan& g, hipStream_t st) {
  if (g.chunks) {
    if (k.dk <= 32) la_launch_dk<DT, 32>(k, g.waves, st);
    else if (k.dk <= 64) la_launch_dk<DT, 64>(k, g.waves, st);
    else if (k.dk <= 96) la_launch_dk<DT, 96>(k, g.waves, st);
    else la_launch_dk<DT, 128>(k, g.waves, st);
    return;
  }
  const dim3 grid((unsigned)(k.nk * k.slices));
#define CLARUS_LA(DVS)                                                                                                   \
  do {                                                                                                                   \
    if (k.dk <= 32) hipLaunchKernelGGL((la_step_kernel<DT, DVS, 32 * DVS / 1024>), grid, dim3(LA_T), 0, st, k);          \
    else if (k.dk <= 64) hipLaunchKernelGGL((la_step_kernel<DT, DVS, 64 * DVS / 1024>), grid, dim3(LA_T), 0, st, k);     \
    else hipLaunchKernelGGL((la_step_kernel<DT, DVS, 128 * DVS / 1024>), grid, dim3(LA_T), 0, st, k);                    \
  } while (0)
  if (g.slice == 32) CLARUS_LA(32);
  else if (g.slice == 64) CLARUS_LA(64);
  else CLARUS_LA(128);
#undef CLARUS_LA
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" size_t clarus_hip_linear_attention_workspace(int32_t dtype, int64_t n, int64_t l, int64_t heads, int64_t kv_heads,
                                                        int64_t dk, int64_t dv) {
  if (n <= 0 || l <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dk <= 0 || dk > 128 || dv <= 0 || dv > 128 ||
      !la_fits(n, l, heads, kv_heads))
    return 0;
  const LaPlan g = la_plan(dtype, n, l, heads, kv_heads, dk, dv);
  return g.part + g.flags;
}

extern "C" int clarus_hip_linear_attention(const ClarusLinearArgs* a, void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  CLARUS_REQUIRE(a, "linear_attention: null arguments");
  CLARUS_REQUIRE(a->q && a->k && a->v && a->out && a->log_decay && a->state_out, "linear_attention: null operand");
  CLARUS_REQUIRE(a->n > 0 && a->l > 0 && a->heads > 0 && a->kv_heads > 0, "linear_attention: empty problem");
  CLARUS_REQUIRE(a->heads % a->kv_heads == 0, "linear_attention: heads a multiple of kv_heads");
  CLARUS_REQUIRE(a->dk >= 8 && a->dk <= 128 && a->dk % 8 == 0 && a->dv >= 8 && a->dv <= 128 && a->dv % 8 == 0,
                 "linear_attention: head widths multiples of 8, at most 128");
  CLARUS_REQUIRE((a->dtype == DT_BF16 || a->dtype == DT_F32) && (a->o_dtype == DT_BF16 || a->o_dtype == DT_F32),
                 "linear_attention: bf16 or fp32");
  CLARUS_REQUIRE(a->scale == a->scale && fabsf(a->scale) < INFINITY, "linear_attention: scale");
  const int64_t es = a->dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && a->ldq * es % 16 == 0 &&
                     a->ldk * es % 16 == 0 && a->ldv * es % 16 == 0 && a->q_bstride * es % 16 == 0 &&
                     a->k_bstride * es % 16 == 0 && a->v_bstride * es % 16 == 0,
                 "linear_attention: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldq >= 0 && a->ldk >= 0 && a->ldv >= 0 && a->q_bstride >= 0 && a->k_bstride >= 0 && a->v_bstride >= 0,
                 "linear_attention: strides");
  CLARUS_REQUIRE(a->ldq < (1 << 24) && a->ldk < (1 << 24) && a->ldv < (1 << 24), "linear_attention: rows less than 2^24 elements apart");
  CLARUS_REQUIRE(aligned(a->state_in, 16) && aligned(a->state_out, 16) && aligned(a->log_decay, 4), "linear_attention: aligned states");
  CLARUS_REQUIRE(la_fits(a->n, a->l, a->heads, a->kv_heads), "linear_attention: too large");
  const LaPlan g = la_plan(a->dtype, a->n, a->l, a->heads, a->kv_heads, a->dk, a->dv);
  CLARUS_REQUIRE(g.part == 0 || (scratch && aligned(scratch, 16) && scratch_bytes >= g.part + g.flags),
                 "linear_attention: scratch %zu < %zu bytes", scratch_bytes, g.part + g.flags);
  LinP k{};
  k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out;
  k.s_in = a->state_in; k.s_out = a->state_out; k.decay = a->log_decay; k.part = (float*)scratch;
  k.careful = g.part ? (int*)((char*)scratch + g.part) : nullptr;
  k.qbs = a->q_bstride; k.ldq = a->ldq; k.kbs = a->k_bstride; k.ldk = a->ldk; k.vbs = a->v_bstride; k.ldv = a->ldv;
  k.l = a->l; k.nk = a->n * a->kv_heads; k.nseg = g.nseg; k.seg = g.seg; k.pad = g.pad;
  k.rep = (int)(a->heads / a->kv_heads); k.kv_heads = (int)a->kv_heads; k.dk = (int)a->dk; k.dv = (int)a->dv;
  k.o_dt = a->o_dtype; k.scale = a->scale;
  k.slices = g.chunks ? 1 : (int)cdiv(a->dv, g.slice);
  note_kernel(g.chunks ? "la_chunk_kernel segments=%lld waves=%d" : "la_step_kernel slices=%lld of %d",
              (long long)(g.chunks ? g.nseg : k.slices), g.chunks ? g.waves : g.slice);
  if (a->dtype == DT_BF16) la_launch_dt<DT_BF16>(k, g, (hipStream_t)stream);
  else la_launch_dt<DT_F32>(k, g, (hipStream_t)stream);
  return check_launch("linear_attention");
}
