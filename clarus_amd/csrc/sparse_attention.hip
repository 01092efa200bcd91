// Attention over the blocks of keys that a cheap score selects, on gfx950. Per image and head:
//   m_b = mean of the kept keys of block b,  a_g = mean of the queries of group g  (64 bits, rounded to fp32)
//   the `top` blocks of the largest a_g . m_b (64 bits; equal ones: the lowest index; a block without a kept key: never)
//   o_i = softmax_j(scale q_i . k_j) v_j  over the kept keys j of the blocks chosen by i's group; 0 where there are none.
//
//   sp_means_kernel   the means of blocks of keys, or of groups of queries
//   sp_pick_kernel    up to 1024 blocks: scores and choice, as bits, 64 blocks a word
//   sp_score_kernel   more blocks: scores of a slab of rows, 64 bits
//   sp_choose_kernel  a row's choice from them
//   sp_kernel         the attention: 32 rows per wave as in cross_attention.hip (a row is a query and one of the heads that
//                     share a kv head); a workgroup takes the blocks that any of its rows has chosen, one after another
//                     through LDS, and a wave those of its own rows; a row that has not chosen a block weighs it by 0
//   xa_join_kernel    joins the parts of blocks split over workgroups, where rows are few
//
// What bounds it: 14400 queries of 8 heads of 64, each with 16 of 225 blocks, 370 us: in sp_kernel, where a wave's 32 rows
// have chosen 72 blocks between them and walk them all (under rocprof 292), and in sp_pick_kernel, the steps of the search beside fp32
// MFMAs (109). 57600, 64 choosing together: 290, of which sp_kernel's softmax steps 242 (500 TFLOP/s). A token of 8
// images over 30001 keys: 79, the latency of three launches and of the chain of blocks in each workgroup.
#include <algorithm>

#include "attention_tile.hpp"
#include "capi.hpp"

namespace clarus {

namespace {

constexpr int SP_T = 256;
constexpr int SP_WORDS = 16;   // words of 64 blocks that a workgroup of sp_kernel lists at a time
constexpr int SP_TILE = 64;    // rows and blocks of a score workgroup
constexpr int64_t SP_SLAB = 128 << 20;  // bytes of scores at a time, about

struct SparseP {
  CrossP x;
  uint64_t* chosen;       // [n][heads][groups][nw]
  const float* means;     // [n][nb][kv_heads * d]
  const void* asks;       // rows of queries, or of their groups' means (fp32)
  int64_t abs, lda;
  double* score;          // of a slab, [row][nb]
  int64_t nw, nb, groups, first;  // first: the slab's first tile of rows
  int64_t tiles;          // tiles of an image and kv head
  int tile;               // rows of one
  int block, group, top, heads, ask_dt;
};

// ---------------------------------------------------------------- means
// A workgroup: one block of rows (of `size`; the last may be shorter) and up to 8 x SP_T / rg columns, rg rows at a time
template <int DT>
__global__ void __launch_bounds__(SP_T) sp_means_kernel(const unsigned char* x, int64_t xbs, int64_t ldx, const unsigned char* mask, int64_t mbs,
                                                        float* out, int64_t rows, int64_t c, int64_t size, unsigned nb, int rg) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4;
  __shared__ double part[SP_T][8];
  __shared__ int count[SP_T];
  const int tid = threadIdx.x, per = SP_T / rg, r0 = tid / per;
  const unsigned n = blockIdx.x / nb, b = blockIdx.x - n * nb;
  const int64_t col = ((int64_t)blockIdx.y * per + tid - r0 * per) * 8;
  const bool in = col < c;
  const int64_t first = (int64_t)b * size, last = first + size < rows ? first + size : rows;
  double s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.0;
  int kept = 0;
  const unsigned char* xp = x + (n * xbs + (in ? col : 0)) * ES;
  for (int64_t r = first + r0; r < last; r += rg) {
    if (mask && !mask[n * mbs + r]) continue;
    ++kept;
    const f32x8 v = load8<DT>(xp + r * ldx * ES);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += (double)v.v[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[tid][e] = s[e];
  count[tid] = kept;
  __syncthreads();
  if (r0 || !in) return;
  for (int i = 1; i < rg; ++i) {
    kept += count[tid + i * per];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += part[tid + i * per][e];
  }
  float* to = out + ((int64_t)n * nb + b) * c + col;
#pragma unroll
  for (int e = 0; e < 8; ++e) to[e] = (float)(s[e] / (double)kept);  // 0 / 0 where nothing is kept
}

// ---------------------------------------------------------------- scores
// The rows (group, head) of an image and kv head share its means. They are taken in tiles of at most SP_TILE, and rows of
// a tile times 64 blocks are a workgroup's; waves without a row leave the products to the others. (8 images' token of 16 heads
// and 4 kv heads of 128 against 2049 blocks: 1400 us with tiles of the heads in order, each with means of its own, 41-56 now)
__global__ void __launch_bounds__(SP_T) sp_score_kernel(const SparseP p) {
  constexpr int KC = 32;  // columns at a time
  __shared__ float sa[SP_TILE][KC + 1], sm[SP_TILE][KC + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, d = p.x.d;
  const int64_t tile = p.first + blockIdx.x, nk = tile / p.tiles, row0 = (tile - nk * p.tiles) * p.tile, b0 = (int64_t)blockIdx.y * SP_TILE;
  const int64_t n = nk / p.x.kv_heads, kvh = nk - n * p.x.kv_heads, rows = p.groups * p.x.rep;
  const int all = (int)(rows - row0 < p.tile ? rows - row0 : p.tile);
  double acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0;
  const float* mp = p.means + (n * p.nb * p.x.kv_heads + kvh) * d;
  for (int c0 = 0; c0 < d; c0 += KC) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SP_TILE * KC / SP_T; ++j) {
      const int r = (tid + j * SP_T) / KC, c = tid % KC;
      if (r < all) {
        const unsigned g = (unsigned)(row0 + r) / (unsigned)p.x.rep;  // rows < 2^31
        const int64_t h = kvh * p.x.rep + row0 + r - (int64_t)g * p.x.rep;
        sa[r][c] = c0 + c < d ? load1(p.asks, p.ask_dt, n * p.abs + g * p.lda + h * d + c0 + c) : 0.f;
      }
      sm[r][c] = b0 + r < p.nb && c0 + c < d ? mp[(b0 + r) * p.x.kv_heads * d + c0 + c] : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < KC; ++c) {
      double a[4], m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = sa[ty + 16 * i][c], m[i] = sm[tx + 16 * i][c];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ty + 16 * i < all)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fma(a[i], m[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (ty + 16 * i < all && b0 + tx + 16 * j < p.nb)
        p.score[((int64_t)blockIdx.x * p.tile + ty + 16 * i) * p.nb + b0 + tx + 16 * j] = acc[i][j];
}

// order of scores as whole numbers; 0: none (NaN, -inf)
__device__ __forceinline__ uint64_t sp_key(double v) {
  if (!(v > -INFINITY)) return 0;
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// A workgroup per row. The largest threshold that leaves `top` scores is halved towards by counts, and found as soon as one
// leaves just `top`. K: scores that a thread holds in registers (0: more, read again for each count). 8192 rows of 2048 blocks:
// 55 us; byte by byte from the highest with counters in LDS 417, and a token's 16 rows of 4097 blocks 106 instead of 15
template <int K>
__global__ void __launch_bounds__(SP_T) sp_choose_kernel(const SparseP p) {
  constexpr int W = SP_T / 64;
  __shared__ int part[2][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t tile = p.first + blockIdx.x / p.tile, nk = tile / p.tiles;
  const int64_t row = (tile - nk * p.tiles) * p.tile + blockIdx.x % p.tile;
  if (row >= p.groups * p.x.rep) return;
  const int64_t n = nk / p.x.kv_heads, g = row / p.x.rep, h = (nk - n * p.x.kv_heads) * p.x.rep + row - g * p.x.rep;
  const double* s = p.score + (int64_t)blockIdx.x * p.nb;
  uint64_t* to = p.chosen + ((n * p.heads + h) * p.groups + g) * p.nw;
  uint64_t key[K ? K : 1];
  if constexpr (K != 0) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int64_t b = i * SP_T + tid;
      key[i] = sp_key(s[b < p.nb ? b : p.nb - 1]);
      if (b >= p.nb) key[i] = 0;
    }
  }
  int turn = 0;
  auto total = [&](int mine) __attribute__((always_inline)) {  // of the waves
    if (lane == 0) part[turn][wave] = mine;
    __syncthreads();
    int c = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) c += part[turn][w];
    turn ^= 1;  // written again only behind the next barrier but one
    return c;
  };
  auto count = [&](uint64_t t) __attribute__((always_inline)) {  // keys from t on
    int c = 0;
    if constexpr (K != 0) {
#pragma unroll
      for (int i = 0; i < K; ++i) c += __popcll(__ballot(key[i] >= t));
    } else {
      for (int64_t b = tid; b < p.nw * 64; b += SP_T) c += __popcll(__ballot(b < p.nb && sp_key(s[b < p.nb ? b : 0]) >= t));
    }
    return total(c);
  };
  // count(lo) >= top > count(hi), unless fewer have a score
  uint64_t lo = 1, hi = 0xffffffffffffffffull;
  int above = 0;  // count(hi)
  bool just = count(lo) <= p.top;
  while (!just && hi - lo > 1) {
    const uint64_t mid = lo + (hi - lo) / 2;
    const int c = count(mid);
    if (c >= p.top) lo = mid;
    else hi = mid, above = c;
    just = c == p.top;
  }
  // the keys from lo on; or those above, and of the ones equal to lo the first
  int left = p.top - above;
  auto word = [&](uint64_t k, int64_t at) __attribute__((always_inline)) {
    uint64_t w;
    if (just) {
      w = __ballot(k >= lo);
    } else {
      const uint64_t same = __ballot(k == lo);
      int before = 0, sum = 0;
      if (lane == 0) part[turn][wave] = __popcll(same);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (i < wave) before += part[turn][i];
        sum += part[turn][i];
      }
      turn ^= 1;
      w = __ballot(k > lo || (k == lo && before + (int)__popcll(same & ((1ull << lane) - 1)) < left));
      left -= sum;
    }
    if (lane == 0 && at < p.nw) to[at] = w;
  };
  if constexpr (K != 0) {
#pragma unroll
    for (int i = 0; i < K; ++i) word(key[i], i * W + wave);
  } else {
    for (int64_t b0 = 0; b0 < p.nb; b0 += SP_T) word(b0 + tid < p.nb ? sp_key(s[b0 + tid]) : 0, b0 / 64 + wave);
  }
}

// ---------------------------------------------------------------- scores and choice in one
// A workgroup: W waves, 32 rows (groups and the heads that share a kv head) of one (image, kv head). A wave holds the scores of
// NT tiles of 32 blocks in registers, from fp32 MFMAs (S^T = means asks^T: a lane holds a row's scores of 16 blocks of
// each tile, its partner in lane ^ 32 the other 16). They are off by at most e = 2 (d + 8) 2^-24 |ask| |mean| (Cauchy-Schwarz over
// the terms; the norms with what their squares may lose below 2^-126, SP_LOST, and products that small below 1e-35 in all).
// A row's threshold is searched between its least and largest score, by counts; where the least score chosen and the
// largest left out are more than 2 e apart, 64 bits would choose the same. Where they are not, the blocks within 2 e of the
// threshold are scored again in 64 bits by a wave, up to 64 of them; a row with more of them (equal blocks,
// an ask of zeros), or with a norm that is not finite, is done by the whole workgroup, every block's rank counted.
// Eight tiles of a wave and the ask do not fit its 256 VGPRs: 14 to 18 are spilled (14400 queries of 8 heads of 64, 225 blocks: 108 us)
constexpr int SP_PICK = 1024;  // blocks, at most
constexpr float SP_LOST = 0x1p-118f;  // of a sum of up to 128 squares, should each lose 2^-126

template <int D, int NT, int W>
__global__ void __launch_bounds__(64 * W, W > 8 ? 4 : 2) sp_pick_kernel(const SparseP p, unsigned row_tiles) {
  constexpr int QN = D / 8;
  __shared__ float xf[3][W][32];  // exchanged by the waves: per row
  __shared__ int xi[W][32];
  __shared__ float wide[W];
  __shared__ unsigned redo[2];    // rows to do again: a few blocks, all of them
  __shared__ unsigned words[32][NT * W], cands[32][NT * W];
  __shared__ double ask64[D];
  __shared__ uint64_t keys[32 * NT * W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hl = lane >> 5;
  const unsigned nk = blockIdx.x / row_tiles, tile = blockIdx.x - nk * row_tiles;
  const int64_t n = nk / p.x.kv_heads, kvh = nk - n * p.x.kv_heads, rows = p.groups * p.x.rep;
  const int d = p.x.d;
  const int64_t row = (int64_t)tile * 32 + col;
  const bool there = row < rows;
  const int64_t g = (there ? row : rows - 1) / p.x.rep, head = kvh * p.x.rep + (there ? row : rows - 1) - g * p.x.rep;
  const int64_t ask = n * p.abs + g * p.lda + head * d, mld = (int64_t)p.x.kv_heads * d;
  const float* mp = p.means + (n * p.nb * p.x.kv_heads + kvh) * d;
  const int nb = (int)p.nb;

  f32x4 q[QN];
  float qq = 0.f;
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int c = 8 * i + 4 * hl;
    q[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (8 * i < d) {
      if (p.ask_dt == DT_BF16) {
        const u32x2 w = *reinterpret_cast<const u32x2*>((const unsigned short*)p.asks + ask + c);
#pragma unroll
        for (int e = 0; e < 2; ++e) q[i][2 * e] = __uint_as_float(w[e] << 16), q[i][2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        q[i] = *reinterpret_cast<const f32x4*>((const float*)p.asks + ask + c);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) qq = fmaf(q[i][e], q[i][e], qq);
  }
  qq = sum32(qq);

  f32x16 s[NT];
  float mm = 0.f, least = INFINITY, most = -INFINITY;
  int valid = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int b0 = 32 * (t * W + wave), b = b0 + col;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[t][j] = 0.f;
    if (b0 >= nb) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[t][j] = -INFINITY;
      continue;
    }
    const float* m = mp + (b < nb ? b : 0) * mld + 4 * hl;
    float norm = 0.f;
#pragma unroll
    for (int i = 0; i < QN; ++i)
      if (8 * i < d) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(m + 8 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          norm = fmaf(a[e], a[e], norm);
          s[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], q[i][e], s[t], 0, 0, 0);
        }
      }
    norm = sum32(norm);
    const bool ok = b < nb && norm == norm;  // a mean of NaN has no score, whatever the row asks
    if (ok) mm = fmaxf(mm, norm);
    const unsigned keep = (unsigned)__ballot(ok) >> (4 * hl);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int at = 8 * (j >> 2) + (j & 3);
      s[t][j] = keep_bit(s[t][j], keep, at);
      most = fmaxf(most, s[t][j]);
      least = fminf(least, keep >> at & 1 ? s[t][j] : INFINITY);
    }
    valid += __popc((unsigned)__ballot(ok));
  }
  // over the row's lanes and waves
  auto all_max = [&](float v, int slot) __attribute__((always_inline)) {
    v = max32(v);
    if constexpr (W > 1) {
      if (hl == 0) xf[slot][wave][col] = v;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) v = fmaxf(v, xf[slot][w][col]);
    }
    return v;
  };
  auto all_sum = [&](int v) __attribute__((always_inline)) {  // v of this lane's half of the blocks
    unsigned a = (unsigned)v, b = a;
    swap32(a, b);
    v = (int)(a + b);
    if constexpr (W > 1) {
      __syncthreads();  // the counts before have been read
      if (hl == 0) xi[wave][col] = v;
      __syncthreads();
      v = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) v += xi[w][col];
    }
    return v;
  };
  auto count = [&](float t) __attribute__((always_inline)) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) c += s[i][j] >= t;
    return all_sum(c);
  };
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));  // a wave's blocks lie over its lanes
  if (W > 1 && lane == 0) wide[wave] = mm;
  most = all_max(most, 0);
  least = -all_max(-least, 1);
  if constexpr (W > 1) {  // all_max's barriers lie behind
    mm = wide[0];
#pragma unroll
    for (int w = 1; w < W; ++w) mm = fmaxf(mm, wide[w]);
  }
  valid = all_sum(hl == 0 ? valid : 0);
  const float e = 2.f * (float)(d + 8) * 0x1p-24f * 1.01f * sqrtf(qq + SP_LOST) * sqrtf(mm + SP_LOST) + 1e-35f;
  const bool wild = !(qq < INFINITY && mm < INFINITY);  // products may leave fp32
  bool done = wild || valid <= p.top, exact = false;
  float thr = -3.402823466e38f;  // every block with a score
  // more than `top` scores from lo on, fewer from hi on: between them as far as the counts' logarithms say (the tail of
  // a bell falls about so), halfway every third time
  float lo = least, hi = most + fabsf(most) * 0x1p-20f + e, clo = (float)valid, chi = 0.5f;
  const float want = (float)p.top;
#pragma unroll 1
  for (int i = 0; i < 48 && !__all(done); ++i) {
    const float w = i % 3 == 2 ? 0.5f : __builtin_amdgcn_logf(clo / want) / __builtin_amdgcn_logf(clo / chi);
    const float mid = lo + (hi - lo) * fminf(fmaxf(w, 0.03f), 0.97f);
    const int c = count(mid);
    if (!done) {
      if (c == p.top) thr = mid, done = exact = true;
      else if (c > p.top) lo = mid, clo = (float)c;
      else hi = mid, chi = fmaxf((float)c, 0.5f);
      if (!(hi - lo > e)) done = true;
    }
  }
  float in = INFINITY, out = -INFINITY;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const bool sel = s[t][j] >= thr;
      in = fminf(in, sel ? s[t][j] : INFINITY);
      out = fmaxf(out, sel ? -INFINITY : s[t][j]);
    }
  in = -all_max(-in, 2);
  out = all_max(out, 0);
  const bool near = there && (wild || (valid > p.top && !(exact && in - out > 2.f * e)));
  unsigned* to = reinterpret_cast<unsigned*>(p.chosen + ((n * p.heads + head) * p.groups + g) * p.nw);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) w |= (unsigned)(s[t][j] >= thr) << (8 * (j >> 2) + (j & 3));
    w <<= 4 * hl;
    unsigned other = w;
    swap32(w, other);
    if (hl == 0 && there && !near && t * W + wave < 2 * p.nw) to[t * W + wave] = w | other;
  }
  if (!__any(near)) return;  // the same in every wave
  // the top-th largest score lies within [lo, hi]: what is more than 2 e above is chosen, what is more than 2 e below is not,
  // and 64 bits decide between them
  if (exact) lo = hi = in;
  const float sure = hi + 2.f * e, maybe = lo - 2.f * e;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    unsigned w = 0, c = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      w |= (unsigned)(s[t][j] > sure) << (8 * (j >> 2) + (j & 3));
      c |= (unsigned)(s[t][j] >= maybe && s[t][j] <= sure) << (8 * (j >> 2) + (j & 3));
    }
    w <<= 4 * hl, c <<= 4 * hl;
    unsigned w2 = w, c2 = c;
    swap32(w, w2);
    swap32(c, c2);
    if (hl == 0) words[col][t * W + wave] = w | w2, cands[col][t * W + wave] = c | c2;
  }
  if (wave == 0) {
    const unsigned few = (unsigned)__ballot(near && !wild), whole = (unsigned)__ballot(near && wild);
    if (lane == 0) redo[0] = few, redo[1] = whole;
  }
  __syncthreads();
  int turn = 0;
  for (unsigned left = __builtin_amdgcn_readfirstlane(redo[0]); left; left &= left - 1) {
    if (turn++ % W != wave) continue;
    const int at = __builtin_ctz(left);
    const int64_t r = (int64_t)tile * 32 + at, rg = r / p.x.rep, rh = kvh * p.x.rep + r - rg * p.x.rep;
    const int64_t from = n * p.abs + rg * p.lda + rh * d;
    double a[(D + 63) / 64];
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) a[i] = lane + 64 * i < d ? load1(p.asks, p.ask_dt, from + lane + 64 * i) : 0.f;
    int some = 0, taken = 0, mine = 0;  // candidates, chosen already, the lane's candidate
    for (int t = 0; t < NT * W; ++t) {
      taken += __popc(words[at][t]);
      for (unsigned c = __builtin_amdgcn_readfirstlane(cands[at][t]); c; c &= c - 1) {
        if (lane == some) mine = 32 * t + __builtin_ctz(c);
        ++some;
      }
    }
    if (some > 64) {
      if (lane == 0) atomicOr(&redo[1], 1u << at);
      continue;
    }
    uint64_t key = 0;
#pragma unroll 4
    for (int i = 0; i < some; ++i) {
      const float* m = mp + __builtin_amdgcn_readlane(mine, i) * mld;
      double v = 0.0;
#pragma unroll
      for (int k = 0; k < (D + 63) / 64; ++k)
        if (lane + 64 * k < d) v = fma(a[k], (double)m[lane + 64 * k], v);
#pragma unroll
      for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
      if (lane == i) key = sp_key(v);
    }
    int rank = 0;
    for (int i = 0; i < some; ++i) {
      const uint64_t k = (uint64_t)__builtin_amdgcn_readlane((unsigned)(key >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((unsigned)key, i);
      rank += k > key || (k == key && i < lane);
    }
    if (key != 0 && rank < p.top - taken) atomicOr(&words[at][mine >> 5], 1u << (mine & 31));
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own LDS operations, in order
    unsigned* rto = reinterpret_cast<unsigned*>(p.chosen + ((n * p.heads + rh) * p.groups + rg) * p.nw);
    for (int t = lane; t < 2 * p.nw; t += 64) rto[t] = words[at][t];
  }
  __syncthreads();
  for (unsigned left = __builtin_amdgcn_readfirstlane(redo[1]); left; left &= left - 1) {
    const int64_t r = (int64_t)tile * 32 + __builtin_ctz(left), rg = r / p.x.rep, rh = kvh * p.x.rep + r - rg * p.x.rep;
    for (int c = tid; c < d; c += 64 * W) ask64[c] = load1(p.asks, p.ask_dt, n * p.abs + rg * p.lda + rh * d + c);
    __syncthreads();
    for (int b = tid; b < nb; b += 64 * W) {
      double v = 0.0;
      for (int c = 0; c < d; ++c) v = fma(ask64[c], (double)mp[b * mld + c], v);
      keys[b] = sp_key(v);
    }
    __syncthreads();
    for (int b0 = 64 * wave; b0 < nb; b0 += 64 * W) {
      const int b = b0 + lane;
      const uint64_t k = b < nb ? keys[b] : 0;
      int rank = 0;
      for (int i = 0; i < nb; ++i) rank += keys[i] > k || (keys[i] == k && i < b);
      const uint64_t word = __ballot(k != 0 && rank < p.top);
      if (lane == 0) p.chosen[((n * p.heads + rh) * p.groups + rg) * p.nw + b0 / 64] = word;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- attention
__device__ __forceinline__ uint64_t or32(uint64_t v) {  // over the 32 lanes of a half
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) v |= __shfl_xor(v, o, 64);
  return v;
}

// The copies of one operand of a tile to LDS by W waves, 1 KiB each: XaCopy's layout. Where the rows of a wave's
// copies lie a multiple of 16 apart (what the swizzles repeat after), one offset serves all of them
template <int DT, int D, int W, bool V>
struct SpCopy {
  using T = XaTile<DT, D>;
  static constexpr int BYTES = T::BYTES, NI = (BYTES / 1024 + W - 1) / W;
  static constexpr bool EVEN = BYTES / 1024 % W == 0, SAME = W * 1024 % (16 * T::ROWB) == 0;
  uint32_t off[SAME ? 1 : NI];
  static __device__ __forceinline__ void place(int j, int wave, int lane, int& r, int& c) {
    const int at = (wave + W * j) * 1024 + lane * 16;
    r = at / T::ROWB;
    c = at % T::ROWB / 16;
    c ^= V ? T::swz_v(r) : T::swz_k(r);
  }
  __device__ __forceinline__ SpCopy(int64_t ld, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < (SAME ? 1 : NI); ++j) {
      int r, c;
      place(j, wave, lane, r, c);
      off[j] = (uint32_t)(r * ld * T::ES) + c * 16;
    }
  }
  // bits: the keys that count; the others, and columns from d on, are zeros
  __device__ __forceinline__ void operator()(const unsigned char* src, int64_t ld, int d, unsigned char* tile, uint64_t bits, int wave,
                                             int lane) const {
    unsigned char* dst = tile + wave * 1024;
#define SP_COPY(from)                                                                          \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from),     \
                                   (__attribute__((address_space(3))) void*)(dst + j * W * 1024), 16, 0, 0)
    const unsigned step = SAME ? (unsigned)(W * 1024 / T::ROWB * ld * T::ES) : 0;  // bytes between a wave's copies
    if (bits == T::ALL && d == D) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= BYTES / 1024) break;
        SP_COPY(src + (size_t)j * step + off[SAME ? 0 : j]);
      }
    } else {
      const unsigned char* zero = (const unsigned char*)xa_zeros;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if (!EVEN && wave + W * j >= BYTES / 1024) break;
        int r, c;
        place(j, wave, lane, r, c);
        SP_COPY((bits >> r & 1) && c * 16 < d * T::ES ? src + (size_t)j * step + off[SAME ? 0 : j] : zero);
      }
    }
#undef SP_COPY
  }
};

__device__ __forceinline__ const unsigned char* uniform(const unsigned char* p) {
  const uint64_t u = (uint64_t)p;
  return (const unsigned char*)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(u >> 32)) << 32 |
                                (unsigned)__builtin_amdgcn_readfirstlane((unsigned)u));
}

template <int DT, int D, int C, int MASK, int W>
__global__ void __launch_bounds__(64 * W, DT == DT_BF16 && D <= 64 ? 4 : 2) sp_kernel(const SparseP sp) {
  using T = XaTile<DT, D>;
  constexpr int KT = T::KT, KB = KT / 32, DB = D / 32;
  const CrossP& p = sp.x;
  const int tpb = sp.block / KT, lk = (int)p.lk, tiles = (int)((p.lk + KT - 1) / KT);  // tiles of a block; keys and tiles in all
  __shared__ __align__(16) unsigned char tile[2 * T::BYTES];
  __shared__ uint64_t wants[W][SP_WORDS];
  __shared__ unsigned short list[SP_WORDS * 64];  // blocks of the words at hand that a row of the workgroup has chosen

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hl = lane >> 5;
  // as xa_kernel: row blocks and splits of one (image, kv head) on one XCD
  const unsigned per = (unsigned)(p.nblk * p.splits), xcd = blockIdx.x & 7, j = blockIdx.x >> 3, whole = (unsigned)(p.nk >> 3) * per;
  unsigned nk, rest;
  if (j < whole) {
    nk = j / per;
    rest = j - nk * per;
    nk = nk * 8 + xcd;
  } else {
    const unsigned left = (unsigned)(p.nk & 7) * per, span = (left + 7) >> 3, i = xcd * span + (j - whole);
    if (j - whole >= span || i >= left) return;
    nk = i / per;
    rest = i - nk * per;
    nk += (unsigned)p.nk & ~7u;
  }
  const unsigned split = rest / (unsigned)p.nblk, rb = rest - split * (unsigned)p.nblk;
  const int n = (int)nk / p.kv_heads, kvh = (int)nk - n * p.kv_heads;
  const int64_t wrow = (int64_t)rb * (32 * W) + wave * 32;
  const bool busy = wrow < p.rows;
  // the lane's row, worked out anew where it is needed (kept over the loop it would spill); past the end the last one
  auto place = [&]() __attribute__((always_inline)) {
    int at = lane & 31;
    asm volatile("" : "+v"(at));
    return wrow + at < p.rows ? wrow + at : p.rows - 1;
  };
  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)kvh * p.d) * T::ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)kvh * p.d) * T::ES;
  const unsigned char* mkey = MASK == MASK_KEYS ? p.mask + n * p.mbs : nullptr;

  const SpCopy<DT, D, W, false> copy_k(p.ldk, wave, lane);
  const SpCopy<DT, D, W, true> copy_v(p.ldv, wave, lane);
  auto fill = [&](int t, uint64_t bits) __attribute__((always_inline)) {
    const int64_t base = (int64_t)t * KT;
    copy_k(uniform(kp + base * p.ldk * T::ES), p.ldk, p.d, tile, bits, wave, lane);
    copy_v(uniform(vp + base * p.ldv * T::ES), p.ldv, p.d, tile + T::BYTES, bits, wave, lane);
  };
  u32x4 qf[xa_qn<DT, C>];
  xa_load_q<DT, C>(p, n, xa_row(p, kvh, place()), hl, qf);
  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
  float m = XA_FLOOR, l = 0.f;
  bool far = false;

#pragma unroll 1
  for (int64_t w0 = 0; w0 < sp.nw; w0 += SP_WORDS) {
    const int wn = sp.nw - w0 < SP_WORDS ? (int)(sp.nw - w0) : SP_WORDS;
    if (w0) __syncthreads();  // the words and the last tile before have been read
    const XaRow r = xa_row(p, kvh, place());
    const uint64_t* words = sp.chosen + (((int64_t)n * sp.heads + r.head) * sp.groups + (unsigned)r.qi / (unsigned)sp.group) * sp.nw;
    for (int w = 0; w < wn; ++w) {
      const uint64_t any = or32(busy ? words[w0 + w] : 0);
      if (lane == 0) wants[wave][w] = any;
    }
    __syncthreads();
    // every wave lists the wanted blocks in order (the same list)
    int count = 0;
    for (int w = 0; w < wn; ++w) {
      uint64_t want = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) want |= wants[i][w];
      if (wave == 0 && (want >> lane & 1)) list[count + __popcll(want & ((1ull << lane) - 1))] = (unsigned short)(w * 64 + lane);
      count += __popcll(want);
    }
    count = __builtin_amdgcn_readfirstlane(count);
    __syncthreads();
    const int i1 = (int)((int64_t)count * (split + 1) / p.splits);
    // 32 listed blocks at a time: lane i holds the i-th, bit i of `keep` says whether the lane's row has chosen it, so that
    // the steps between the products read no list
#pragma unroll 1
    for (int i0 = (int)((int64_t)count * split / p.splits); i0 < i1; i0 += 32) {
      const int cn = i1 - i0 < 32 ? i1 - i0 : 32;
      const int blk = lane < cn ? list[i0 + lane] : 0;
      unsigned keep = 0;
      const unsigned* row_words = reinterpret_cast<const unsigned*>(words + w0);
      if (busy) {
#pragma unroll 4
        for (int i = 0; i < cn; ++i) {
          const int b = __builtin_amdgcn_readlane(blk, i);
          keep |= (row_words[b >> 5] >> (b & 31) & 1) << i;
        }
      }
      int e = -1, sub = tpb;
      auto pop = [&](int& i) __attribute__((always_inline)) {  // the next tile and its place in the list, -1 past the last
        if (++sub < tpb) {
          const int t = ((int)w0 * 64 + __builtin_amdgcn_readlane(blk, e)) * tpb + sub;
          if (t < tiles) return t;  // the last block's may end past 2^31
        }
        if (e + 1 >= cn) {
          sub = tpb;
          return -1;
        }
        i = ++e;
        sub = 0;
        return ((int)w0 * 64 + __builtin_amdgcn_readlane(blk, e)) * tpb;
      };
      auto key_byte = [&](int t) __attribute__((always_inline)) {  // this lane's key of a tile counts
        const bool in = t >= 0 && lane < KT && lane < lk - t * KT;
        if constexpr (MASK == MASK_KEYS) return in ? (int)mkey[t * KT + lane] : 0;
        return (int)in;
      };
      int i = 0, t = pop(i);
      int byte = key_byte(t);
#pragma unroll 1
      while (t >= 0) {
        const uint64_t bits = __ballot(byte);
        barrier_keep_vm();  // the tile before has been read
        fill(t, bits);
        const bool live = keep >> i & 1;  // this lane's row has chosen it
        t = pop(i);
        byte = key_byte(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's copies have landed
        barrier_keep_vm();                   // everybody's have
        constexpr bool ANEW = DT == DT_BF16 && (C == 64 || (D == 64 && W == 4));  // the forms that else spill
        if (__any(live)) xa_tile<DT, D, C, MASK_ROWS, KB, ANEW>(tile, tile + T::BYTES, qf, o, m, l, far, p.c, bits, bits == T::ALL, false, live);
      }
    }
  }
  if (!busy) return;
  l = sum32(l);
  const int64_t row = place();
  const bool there = wrow + col < p.rows;
  if (p.splits == 1) {
    xa_store<D>(p, n, xa_row(p, kvh, row), o, l, there);
    return;
  }
  if (!there) return;
  const int64_t to = ((int64_t)split * p.nk + nk) * p.rows + row, all = (int64_t)p.splits * p.nk * p.rows;
  float* po = p.part + to * D;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j4 = 0; j4 < 4; ++j4)
      *reinterpret_cast<f32x4*>(po + 32 * b + 8 * j4 + 4 * hl) = f32x4{o[b][4 * j4], o[b][4 * j4 + 1], o[b][4 * j4 + 2], o[b][4 * j4 + 3]};
  if (hl == 0) *reinterpret_cast<float2*>(p.part + all * D + 2 * to) = float2{m, l};
}

int sp_pad(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

// Waves of a workgroup, 32 rows each: they share the copies of a block, but wait for each other's blocks. Rows that choose
// together fill four; else two (fp32, bound by the products: one). us with 1 / 2 / 4 waves, one tile in LDS: 14400 queries
// of 8 heads of 64 each choosing 16 of 225 blocks 357 / 292 / 341; 57600, 64 choosing together, 16 of 900 354 / 242 / 298, 256
// together 329 / 224 / 195; 28800 of 128, 256 together 381 / 197 / 183; 7200 of 4 heads of 64 in fp32, each 453 / 659 / 435, 14400,
// 64 together 169 / 173 / 279; 14400 of 2 of 128 in fp32, 256 together 184 / 272 / 154. (A second tile in LDS, on its way
// during the first one's products, halves the workgroups of a CU: 57600, 64 together, 555 / 336 / 335)
int sp_waves(int32_t dt, int64_t rows, int64_t alike) { return rows <= 32 ? 1 : alike >= 128 ? 4 : dt == DT_BF16 ? 2 : 1; }

struct SpPlan {
  int64_t nb, nw, groups, nblk;
  int64_t slab, tiles;  // tiles of rows whose scores are held at a time; of an image and kv head
  int splits, waves, tile;  // tile: rows of one
  int pick_tiles, pick_waves;  // of 32 blocks per wave of sp_pick_kernel; 0: sp_score_kernel and sp_choose_kernel
  size_t means, asks, chosen, score, part;  // workspace bytes, each a multiple of 16
  size_t total() const { return means + asks + chosen + score + part; }
};

SpPlan sp_plan(int32_t dt, int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t d, int64_t top, int64_t block, int64_t group,
               bool has_means, bool has_chosen) {
  SpPlan g{};
  g.nb = cdiv(lk, block);
  g.nw = cdiv(g.nb, 64);
  g.groups = cdiv(lq, group);
  const int64_t rows = lq * (heads / kv_heads), nk = n * kv_heads, asks = n * heads * g.groups;
  if (!has_means) g.means = (size_t)(n * g.nb * kv_heads * d) * sizeof(float);
  if (group > 1) g.asks = (size_t)(n * g.groups * heads * d) * sizeof(float);
  if (!has_chosen) g.chosen = (size_t)cdiv(asks * g.nw, 2) * 16;
  if (g.nb <= SP_PICK) {
    // few rows: two tiles per wave and more waves
    const int64_t tiles = 2 * g.nw, wgs = nk * cdiv(g.groups * (heads / kv_heads), 32);
    const int most = wgs < 2 * device_cus() ? 2 : d <= 64 ? 8 : 4;
    g.pick_tiles = tiles <= 2 ? 2 : most;
    g.pick_waves = 1;
    while (g.pick_tiles * g.pick_waves < tiles) g.pick_waves *= 2;
  } else {
    g.tile = (int)std::min<int64_t>(SP_TILE, g.groups * (heads / kv_heads));
    g.tiles = cdiv(g.groups * (heads / kv_heads), g.tile);
    g.slab = std::min(nk * g.tiles, std::min<int64_t>(cdiv(SP_SLAB / 8, g.nb * g.tile), 1 << 16));
    g.score = (size_t)cdiv(g.slab * g.tile * g.nb, 2) * 16;
  }
  g.waves = sp_waves(dt, rows, group * (heads / kv_heads));
  g.nblk = cdiv(rows, 32 * g.waves);
  const int64_t blocks = g.nblk * nk, cus = device_cus();
  // few rows: the blocks that they can choose split until every CU has two workgroups
  const int64_t most = std::min(g.nb, std::min<int64_t>(rows, 32 * g.waves) * std::min(top, g.nb));
  g.splits = (int)std::max<int64_t>(1, std::min(2 * cus / blocks, most));
  if (g.splits > 1) g.part = (size_t)cdiv((int64_t)g.splits * nk * rows * (sp_pad(d) + 2), 4) * 16;
  return g;
}

bool sp_fits(int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t block, int64_t group) {
  const int64_t big = (int64_t)1 << 31;
  if (!(n < 65536 && kv_heads < 65536 && n * kv_heads < 65536 && heads < 65536 && lq < big && lk < big && lq * (heads / kv_heads) < big &&
        n * heads < big && n * kv_heads * (cdiv(lq * (heads / kv_heads), 128) * 128) < big - 4096))
    return false;
  const int64_t nb = cdiv(lk, block), groups = cdiv(lq, group);
  return nb < (1 << 21) && n * nb < (1 << 23) && (group == 1 || n * groups < (1 << 23)) && n * heads * groups < (1 << 26);
}

template <int D>
void sp_pick(const SparseP& k, const SpPlan& g, hipStream_t st) {
  const unsigned tiles = (unsigned)cdiv(k.groups * k.x.rep, 32);
  const dim3 grid((unsigned)k.x.nk * tiles), block(64 * g.pick_waves);
#define CLARUS_PICK(NT, W) \
  if (g.pick_tiles == NT && g.pick_waves == W) hipLaunchKernelGGL((sp_pick_kernel<D, NT, W>), grid, block, 0, st, k, tiles)
  CLARUS_PICK(2, 1);
  CLARUS_PICK(2, 2);
  CLARUS_PICK(2, 4);
  CLARUS_PICK(2, 8);
  CLARUS_PICK(2, 16);
  if constexpr (D <= 64) {
    CLARUS_PICK(8, 1);
    CLARUS_PICK(8, 2);
    CLARUS_PICK(8, 4);
  } else {
    CLARUS_PICK(4, 1);
    CLARUS_PICK(4, 2);
    CLARUS_PICK(4, 4);
    CLARUS_PICK(4, 8);
  }
#undef CLARUS_PICK
}

template <int DT, int D, int C, int MASK>
void sp_launch_mask(const SparseP& k, int waves, hipStream_t st) {
  const dim3 grid((unsigned)(8 * ((k.x.nblk * k.x.nk * k.x.splits + 7) / 8)));
  if (waves == 1) hipLaunchKernelGGL((sp_kernel<DT, D, C, MASK, 1>), grid, dim3(64), 0, st, k);
  else if (waves == 4) hipLaunchKernelGGL((sp_kernel<DT, D, C, MASK, 4>), grid, dim3(256), 0, st, k);
  else if constexpr (DT == DT_BF16) hipLaunchKernelGGL((sp_kernel<DT, D, C, MASK, 2>), grid, dim3(128), 0, st, k);
}

template <int DT, int D, int C>
void sp_launch(const SparseP& k, int waves, hipStream_t st) {
  if (k.x.mask) sp_launch_mask<DT, D, C, MASK_KEYS>(k, waves, st);
  else sp_launch_mask<DT, D, C, MASK_NONE>(k, waves, st);
  if (k.x.splits > 1) {
    constexpr int TPR = D <= 32 ? 8 : D <= 64 ? 16 : 32;
    int gs = 1;
    while (gs * TPR < XA_T && gs * XJ_BATCH < k.x.splits) gs *= 2;
    hipLaunchKernelGGL((xa_join_kernel<D>), dim3((unsigned)cdiv(k.x.rows * k.x.nk, XA_T / (TPR * gs))), dim3(XA_T), 0, st, k.x, gs);
  }
}

void sp_means(const void* x, int dt, int64_t xbs, int64_t ldx, const void* mask, int64_t mbs, float* out, int64_t n, int64_t rows, int64_t c,
              int64_t size, hipStream_t st) {
  const int64_t nb = cdiv(rows, size), oct = c / 8;
  int rg = 1;
  while (rg < 32 && rg < size && oct * rg * 2 <= SP_T) rg *= 2;
  // few blocks: fewer columns and more rows at a time (one group of 14400 rows of 512: 95 us, 1180 with all columns at once)
  while (rg < 64 && rg * 4 <= size && n * nb * cdiv(oct, SP_T / rg) < 2 * device_cus()) rg *= 2;
  const dim3 grid((unsigned)(n * nb), (unsigned)cdiv(oct, SP_T / rg));
  if (dt == DT_BF16)
    hipLaunchKernelGGL(sp_means_kernel<DT_BF16>, grid, dim3(SP_T), 0, st, (const unsigned char*)x, xbs, ldx, (const unsigned char*)mask, mbs, out,
                       rows, c, size, (unsigned)nb, rg);
  else
    hipLaunchKernelGGL(sp_means_kernel<DT_F32>, grid, dim3(SP_T), 0, st, (const unsigned char*)x, xbs, ldx, (const unsigned char*)mask, mbs, out,
                       rows, c, size, (unsigned)nb, rg);
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" int clarus_hip_block_means(const void* k, int32_t dtype, int64_t k_bstride, int64_t ldk, const void* mask, int64_t mask_bstride,
                                      float* means, int64_t n, int64_t lk, int64_t c, int64_t block, void* stream) {
  clear_error();
  CLARUS_REQUIRE(k && means, "block_means: null operand");
  CLARUS_REQUIRE(n > 0 && lk > 0 && c > 0 && block > 0, "block_means: empty problem");
  CLARUS_REQUIRE(dtype == DT_BF16 || dtype == DT_F32, "block_means: bf16 or fp32");
  CLARUS_REQUIRE(c % 8 == 0 && c < (1 << 20), "block_means: columns a multiple of 8, below 2^20");
  const int64_t es = dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(k, 16) && aligned(means, 16) && ldk * es % 16 == 0 && k_bstride * es % 16 == 0, "block_means: 16-byte aligned rows");
  CLARUS_REQUIRE(ldk >= 0 && k_bstride >= 0 && mask_bstride >= 0, "block_means: strides");
  CLARUS_REQUIRE(n < (1 << 23) && lk < ((int64_t)1 << 31) && block < ((int64_t)1 << 31) && n * cdiv(lk, block) < (1 << 23), "block_means: too large");
  note_kernel("sp_means_kernel");
  sp_means(k, dtype, k_bstride, ldk, mask, mask_bstride, means, n, lk, c, block, (hipStream_t)stream);
  return check_launch("block_means");
}

extern "C" size_t clarus_hip_sparse_attention_workspace(int32_t dtype, int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t d, int64_t top,
                                                        int64_t block, int64_t group, int32_t has_means, int32_t has_chosen) {
  if (n <= 0 || lq <= 0 || lk <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || d <= 0 || d > 128 || top <= 0 || block < 64 ||
      block % 64 || block >= (1 << 20) || group <= 0 || !sp_fits(n, lq, lk, heads, kv_heads, block, std::min(group, lq)))
    return 0;
  return sp_plan(dtype, n, lq, lk, heads, kv_heads, d, std::min(top, lk), block, std::min(group, lq), has_means != 0, has_chosen != 0).total();
}

extern "C" int clarus_hip_sparse_attention(const ClarusSparseArgs* a, void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  CLARUS_REQUIRE(a, "sparse_attention: null arguments");
  CLARUS_REQUIRE(a->q && a->k && a->v && a->out, "sparse_attention: null operand");
  CLARUS_REQUIRE(a->n > 0 && a->lq > 0 && a->lk > 0 && a->heads > 0 && a->kv_heads > 0, "sparse_attention: empty problem");
  CLARUS_REQUIRE(a->heads % a->kv_heads == 0, "sparse_attention: heads a multiple of kv_heads");
  CLARUS_REQUIRE(a->d >= 8 && a->d <= 128 && a->d % 8 == 0, "sparse_attention: head width a multiple of 8, at most 128");
  CLARUS_REQUIRE(a->top > 0 && a->group > 0 && a->block >= 64 && a->block % 64 == 0 && a->block < (1 << 20),
                 "sparse_attention: top and group positive, block a multiple of 64 below 2^20");
  CLARUS_REQUIRE((a->dtype == DT_BF16 || a->dtype == DT_F32) && (a->o_dtype == DT_BF16 || a->o_dtype == DT_F32),
                 "sparse_attention: bf16 or fp32");
  CLARUS_REQUIRE(a->scale > 0.f && a->scale < 2e38f, "sparse_attention: scale positive and below 2e38");
  const int64_t es = a->dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && aligned(a->means, 16) &&
                     aligned(a->chosen, 8) && a->ldq * es % 16 == 0 && a->ldk * es % 16 == 0 && a->ldv * es % 16 == 0 &&
                     a->q_bstride * es % 16 == 0 && a->k_bstride * es % 16 == 0 && a->v_bstride * es % 16 == 0,
                 "sparse_attention: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldk < (1 << 24) && a->ldv < (1 << 24), "sparse_attention: rows of k and v less than 2^24 elements apart");
  CLARUS_REQUIRE(a->ldq >= 0 && a->ldk >= 0 && a->ldv >= 0 && a->q_bstride >= 0 && a->k_bstride >= 0 && a->v_bstride >= 0 &&
                     a->mask_bstride >= 0,
                 "sparse_attention: strides");
  const int64_t group = std::min(a->group, a->lq), top = std::min(a->top, a->lk);
  CLARUS_REQUIRE(sp_fits(a->n, a->lq, a->lk, a->heads, a->kv_heads, a->block, group), "sparse_attention: too large");
  const SpPlan g = sp_plan(a->dtype, a->n, a->lq, a->lk, a->heads, a->kv_heads, a->d, top, a->block, group, a->means != nullptr, a->chosen != nullptr);
  CLARUS_REQUIRE(g.total() == 0 || (scratch && aligned(scratch, 16) && scratch_bytes >= g.total()),
                 "sparse_attention: scratch %zu < %zu bytes", scratch_bytes, g.total());
  char* at = (char*)scratch;
  auto take = [&](size_t bytes) { char* r = at; at += bytes; return r; };
  SparseP k{};
  CrossP& x = k.x;
  x.q = a->q; x.k = a->k; x.v = a->v; x.out = a->out; x.mask = (const unsigned char*)a->mask;
  x.qbs = a->q_bstride; x.ldq = a->ldq; x.kbs = a->k_bstride; x.ldk = a->ldk; x.vbs = a->v_bstride; x.ldv = a->ldv; x.mbs = a->mask_bstride;
  x.rep = (int)(a->heads / a->kv_heads); x.kv_heads = (int)a->kv_heads; x.d = (int)a->d; x.lq = (int)a->lq;
  x.rows = a->lq * x.rep; x.lk = a->lk; x.nk = a->n * a->kv_heads; x.nblk = g.nblk; x.splits = g.splits;
  x.o_dt = a->o_dtype; x.c = a->scale * 1.4426950408889634f;
  k.nw = g.nw; k.nb = g.nb; k.groups = g.groups; k.block = (int)a->block; k.group = (int)group; k.top = (int)top; k.heads = (int)a->heads;
  hipStream_t st = (hipStream_t)stream;
  const int64_t c = a->heads * a->d, ck = a->kv_heads * a->d;
  float* means = (float*)take(g.means);
  if (!a->means) sp_means(a->k, a->dtype, a->k_bstride, a->ldk, a->mask, a->mask_bstride, means, a->n, a->lk, ck, a->block, st);
  k.means = a->means ? a->means : means;
  float* asks = (float*)take(g.asks);
  if (group > 1) {
    sp_means(a->q, a->dtype, a->q_bstride, a->ldq, nullptr, 0, asks, a->n, a->lq, c, group, st);
    k.asks = asks; k.abs = g.groups * c; k.lda = c; k.ask_dt = DT_F32;
  } else {
    k.asks = a->q; k.abs = a->q_bstride; k.lda = a->ldq; k.ask_dt = a->dtype;
  }
  uint64_t* chosen = (uint64_t*)take(g.chosen);
  k.chosen = a->chosen ? a->chosen : chosen;
  k.score = (double*)take(g.score);
  x.part = (float*)take(g.part);
  if (g.pick_tiles) {
    if (a->d <= 64) sp_pick<64>(k, g, st);
    else sp_pick<128>(k, g, st);
  }
  k.tile = g.tile; k.tiles = g.tiles;
  for (k.first = 0; !g.pick_tiles && k.first < x.nk * g.tiles; k.first += g.slab) {
    const unsigned tiles = (unsigned)std::min(g.slab, x.nk * g.tiles - k.first);
    hipLaunchKernelGGL(sp_score_kernel, dim3(tiles, (unsigned)cdiv(g.nb, SP_TILE)), dim3(SP_T), 0, st, k);
    const dim3 rows(tiles * (unsigned)g.tile);
    if (g.nb <= 8 * SP_T) hipLaunchKernelGGL(sp_choose_kernel<8>, rows, dim3(SP_T), 0, st, k);
    else if (g.nb <= 16 * SP_T) hipLaunchKernelGGL(sp_choose_kernel<16>, rows, dim3(SP_T), 0, st, k);
    else if (g.nb <= 32 * SP_T) hipLaunchKernelGGL(sp_choose_kernel<32>, rows, dim3(SP_T), 0, st, k);
    else hipLaunchKernelGGL(sp_choose_kernel<0>, rows, dim3(SP_T), 0, st, k);
  }
  if (const int rc = check_launch("sparse_attention")) return rc;
  note_kernel("sp_kernel d=%d waves=%d splits=%d", sp_pad(a->d), g.waves, g.splits);
#define CLARUS_SP(DT)                                          \
  do {                                                         \
    if (a->d <= 32) sp_launch<DT, 32, 32>(k, g.waves, st);     \
    else if (a->d <= 48) sp_launch<DT, 64, 48>(k, g.waves, st); \
    else if (a->d <= 64) sp_launch<DT, 64, 64>(k, g.waves, st); \
    else if (a->d <= 80) sp_launch<DT, 96, 80>(k, g.waves, st); \
    else if (a->d <= 96) sp_launch<DT, 96, 96>(k, g.waves, st); \
    else if (a->d <= 112) sp_launch<DT, 128, 112>(k, g.waves, st); \
    else sp_launch<DT, 128, 128>(k, g.waves, st);              \
  } while (0)
  if (a->dtype == DT_BF16) CLARUS_SP(DT_BF16);
  else CLARUS_SP(DT_F32);
#undef CLARUS_SP
  return check_launch("sparse_attention");
}
