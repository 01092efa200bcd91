// Group norm of an NHWC map with its activation on gfx950.
//
// For image n and group g of cg = C / G channels, over the P pixels x cg channels of the group:
//   mean, var = biased;  y = act((x - mean) * rsqrt(var + eps) * weight[c] + bias[c])
//
// Statistics without cancellation: a thread takes UR rows of its channel octet into registers, has
// their mean and variance in two passes over registers, and joins them to its running (mean, var);
// threads, channels of a group and chunks of pixels are then joined by
//   mean = sum(w mean),  var = sum(w (var_i + (mean_i - mean)^2)),  w = cnt / sum(cnt)
// in a fixed order, all in fp32: no square of an uncentred value occurs, so a mean far from zero or
// a single large value costs no digits, and the result is deterministic. A variance is carried and no sum
// of squares, and nothing is joined to an empty part: whatever the count, values only have to lie within 2^60
// of their group's mean, whose size may be more than a square holds (up to 2^124, as eight of them are added).
// The mean of equal values is that value, and their variance 0: eight values are added in pairs, which is exact for
// equal ones, and means are joined by their differences from one of them.
//   gn_stats_kernel  per (image, chunk of pixels) the groups' mean and variance: one read of x
//   gn_join_kernel   per (image, group) the chunks joined: mean, rstd
//   gn_apply_kernel  y: one read of x, one write
//   gn_small_kernel  all in one launch, x held in registers between them, where the pixels of a few
//                    whole groups fit one workgroup
// What bounds it: memory. 720 x 1280 x 64 bf16 with GELU, 236 MB in and out: 62 us with x in the last-level cache
// (statistics 24, join 5, apply 36 us traced, the last at 97% VALU issue), 81 us cold; 2 x 173 x 251 x 128 fp32 with SiLU,
// 89 MB: 27 us. Small maps: the launches (90 x 160 x 512 bf16, 29 MB: 8 + 3 + 8 us).
#include <algorithm>

#include "capi.hpp"
#include "common.hpp"

namespace clarus {

namespace {

constexpr int GN_T = 256;    // threads of an apply workgroup
constexpr int GN_TS = 256;   // threads of a small workgroup
constexpr int GN_TT = 256;   // threads of a stats workgroup
constexpr int UR = 8;        // rows in flight per thread (stats; mean8's count)
constexpr int UA = 4;        // rows in flight per thread (apply)
constexpr int NRMAX = 8;     // rows held per thread (small), at most
constexpr int GN_JOIN = 8;   // partial statistics in flight per thread (join)
constexpr int GN_UNIT = 2048;  // channels that a workgroup has to hold together, at most
constexpr int64_t GN_GRID = 1 << 23;  // workgroups of a launch, at most
constexpr int GN_SILU = CLARUS_ACT_SILU;

struct GroupNormP {
  const void* x;
  void* out;
  const float* w;    // [C] or [N][C] (wbs = C), or null
  const float* b;
  float2* part;      // [n][G][chunk] mean, variance
  float2* stat;      // [n][G] mean, rstd
  int64_t xbs, ldx;  // image and pixel stride of x (elements)
  int64_t p;         // pixels
  int64_t chunk;     // pixels per workgroup of this launch
  int64_t schunk;    // pixels per statistics chunk
  int64_t wbs, bbs;
  int c, groups, cg, nchunk;
  int n, strips, chunks;  // images, strips of channels, chunks of this launch
  int tr, rpb;       // threads per row (octets of a strip), rows per pass of a workgroup
  int lpg;           // lanes that join a group: a power of two <= 64
  int act;
  float eps;
};

template <int DT>
__device__ __forceinline__ f32x8 gn_load(const void* x, int64_t i) {
  return load8<DT>((const unsigned char*)x + i * (DT == DT_BF16 ? 2 : 4));
}

// 8 values as they lie in memory, and widened
template <int DT> struct GnRaw { typedef u32x4 T; };
template <> struct GnRaw<DT_F32> { struct T { f32x4 a, b; }; };
template <int DT>
__device__ __forceinline__ typename GnRaw<DT>::T gn_raw(const void* x, int64_t i) {
  return *reinterpret_cast<const typename GnRaw<DT>::T*>((const unsigned char*)x + i * (DT == DT_BF16 ? 2 : 4));
}
template <int DT>
__device__ __forceinline__ f32x8 gn_widen(const typename GnRaw<DT>::T& v) { return load8<DT>(&v); }

// mean of 8 values, added in pairs
__device__ __forceinline__ float mean8(float a, float b, float c, float d, float e, float f, float g, float h) {
  return (((a + b) + (c + d)) + ((e + f) + (g + h))) * 0.125f;
}
__device__ __forceinline__ float mean8(const f32x8& x) { return mean8(x.v[0], x.v[1], x.v[2], x.v[3], x.v[4], x.v[5], x.v[6], x.v[7]); }

// sum over the lpg consecutive lanes of a group (lpg a power of two <= 64)
__device__ __forceinline__ float lanes_sum(float v, int lpg) {
  for (int o = 1; o < lpg; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

enum : int { GN_FRONT, GN_BACK, GN_PARTS };

// What a workgroup of a one-dimensional grid works on: (image, strip of channels, chunk of pixels). False past the last.
//   GN_FRONT, GN_BACK  one image after another (GN_BACK: the last first), its strips and chunks in equal parts over the
//                      XCDs where there are eight of them or more. The apply pass goes back over what the statistics pass
//                      has read, whose end is still in the last-level cache and, of its own part, in the XCD's L2 (90 x
//                      160 x 512 bf16 15.6 us dealt out one by one, 14.2 in parts; 2 x 173 x 251 x 128 fp32 29.1, 28.1 in
//                      parts, 26.7 back; images in parts over the XCDs: 64 x 4096 x 512 fp32 251 us, 301)
//   GN_PARTS           the whole in equal parts over the XCDs: neighbouring strips share the lines of a row, which an L2
//                      joins (64 images of 2048 pixels, 512 channels, 64 groups, bf16: 256 us dealt out, 71 in parts)
template <int ORDER>
__device__ __forceinline__ bool gn_at(const GroupNormP& p, int64_t& n, int& strip, int& chunk) {
  const unsigned per = (unsigned)p.strips * (unsigned)p.chunks, total = (unsigned)p.n * per, xcd = blockIdx.x & 7;
  unsigned i = blockIdx.x >> 3, rest;
  if (ORDER != GN_PARTS && per >= 8) {
    const unsigned m = (per + 7) >> 3;
    if (ORDER == GN_BACK) i = (unsigned)p.n * m - 1 - i;
    n = i / m;
    rest = xcd * m + i % m;
    if (rest >= per) return false;
  } else {
    const unsigned span = (total + 7) >> 3, id = ORDER == GN_PARTS ? xcd * span + i : ORDER == GN_BACK ? total - 1 - blockIdx.x : blockIdx.x;
    if (i >= span || id >= total) return false;
    n = id / per;
    rest = id % per;
  }
  strip = (int)(rest / (unsigned)p.chunks);
  chunk = (int)(rest - (unsigned)strip * (unsigned)p.chunks);
  return true;
}

// f(group) on the lpg consecutive threads of each of ng groups at a time, every lane of a wave in step
template <int T, class F>
__device__ __forceinline__ void for_groups(int ng, int lpg, F&& f) {
  const int per = T / lpg, mine = threadIdx.x / lpg;
  for (int g0 = 0; g0 < ng; g0 += per) f(g0 + mine < ng ? g0 + mine : ng - 1, g0 + mine < ng);
}

// WHOLE: cg % 8 == 0, an octet lies in one group and is one set of 8 values per row
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(GN_TT) gn_stats_kernel(const GroupNormP p) {
  constexpr int NA = WHOLE ? 1 : 8;  // (mean, var) pairs per thread
  constexpr int PER = WHOLE ? 8 : 1;
  __shared__ float sm[GN_TT * NA], sv[GN_TT * NA];
  const int tid = threadIdx.x;
  const int rl = tid / p.tr, oct = tid - rl * p.tr;
  int64_t n;
  int strip, at_chunk;
  if (!gn_at<GN_FRONT>(p, n, strip, at_chunk)) return;
  const int64_t r0 = (int64_t)at_chunk * p.chunk;
  const int rows = (int)((r0 + p.chunk < p.p ? r0 + p.chunk : p.p) - r0);
  const int c0 = strip * p.tr * 8;  // first channel of the strip
  const bool act = rl < p.rpb && c0 + oct * 8 < p.c;
  float mean[NA], var[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) mean[i] = var[i] = 0.f;
  int cnt = 0;  // rows so far
  // (m, v) of `part` of the rows with them joined to the rows so far (part 1: there are none)
  auto join = [&](int a, float m, float v, float part) __attribute__((always_inline)) {
    const float d = m - mean[a];
    mean[a] = fmaf(d, part, mean[a]);
    var[a] = fmaf(part, fmaf((1.f - part) * d, d, v - var[a]), var[a]);
  };
  if (act) {
    const int64_t base = n * p.xbs + r0 * p.ldx + c0 + oct * 8;
    int r = rl;
    typename GnRaw<DT>::T w[UR];  // the next batch
    auto fetch = [&](int at) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < UR; ++k) w[k] = gn_raw<DT>(p.x, base + (int64_t)(at + k * p.rpb) * p.ldx);
    };
    if (r + (UR - 1) * p.rpb < rows) fetch(r);
    for (; r + (UR - 1) * p.rpb < rows; r += UR * p.rpb) {
      f32x8 v[UR];
#pragma unroll
      for (int k = 0; k < UR; ++k) v[k] = gn_widen<DT>(w[k]);
      if (r + (2 * UR - 1) * p.rpb < rows) fetch(r + UR * p.rpb);
      const float part = cnt ? (float)UR * __builtin_amdgcn_rcpf((float)(cnt + UR)) : 1.f;
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        float t[UR], q = 0.f;
#pragma unroll
        for (int k = 0; k < UR; ++k) t[k] = WHOLE ? mean8(v[k]) : v[k].v[a];
        const float m = mean8(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7]);
#pragma unroll
        for (int k = 0; k < UR; ++k)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const float d = v[k].v[a * PER + i] - m;
            q = fmaf(d, d, q);
          }
        join(a, m, q * (1.f / (UR * PER)), part);
      }
      cnt += UR;
    }
    for (; r < rows; r += p.rpb) {
      const f32x8 v = gn_load<DT>(p.x, base + (int64_t)r * p.ldx);
      const float part = cnt ? __builtin_amdgcn_rcpf((float)(cnt + 1)) : 1.f;
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        float q = 0.f;
        const float m = WHOLE ? mean8(v) : v.v[a];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float d = v.v[a * PER + i] - m;
          q = fmaf(d, d, q);
        }
        join(a, m, q * (1.f / PER), part);
      }
      ++cnt;
    }
  }
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    sm[tid * NA + a] = mean[a];
    sv[tid * NA + a] = var[a];
  }
  __syncthreads();
  // entries of a group: row lanes (over the group's lanes) x its octets or channels of a row
  const int units = p.cg / PER, sub = tid & (p.lpg - 1);
  const int sgroups = min(p.tr * 8, p.c - c0) / p.cg;  // groups of the strip
  const int full = rows / p.rpb, rem = rows - full * p.rpb;
  // the part of the group's values that an entry with full rows, or one more, stands for
  const float w0 = (float)full / ((float)rows * (float)units), w1 = (float)(full + 1) / ((float)rows * (float)units);
  for_groups<GN_TT>(sgroups, p.lpg, [&](int g, bool mine) {
    const float base = sm[g * units];  // differences from one of the means: equal means come out as they are
    float ms = 0.f;
    for (int el = sub; el < p.rpb; el += p.lpg) {
      const float w = el < rem ? w1 : w0;
      for (int u = 0; u < units; ++u) ms = fmaf(w, sm[el * p.tr * NA + g * units + u] - base, ms);
    }
    const float mu = base + lanes_sum(ms, p.lpg);
    float q = 0.f;
    for (int el = sub; el < p.rpb; el += p.lpg) {
      const float w = el < rem ? w1 : w0;
      if (w == 0.f) continue;
      for (int u = 0; u < units; ++u) {
        const int at = el * p.tr * NA + g * units + u;
        const float d = sm[at] - mu;
        q = fmaf(w, fmaf(d, d, sv[at]), q);
      }
    }
    q = lanes_sum(q, p.lpg);
    if (mine && sub == 0) p.part[(n * p.groups + c0 / p.cg + g) * p.nchunk + at_chunk] = float2{mu, q};
  });
}

// GELU for an output rounded to bf16: x / (1 + e^-xP(x^2)), P an own minimax fit of ln(Phi(x) / Phi(-x)) / x on |x| < 5.5
// (its leading coefficient positive, so that it goes on to 0 and x). Off by at most 6.6e-6 and, down to -5.5, by 5.6e-4
// of the value, a seventh of a bf16 half step; further down the values are below 2e-7. 14 VALU slots against the 23 of
// the erf form, which make the apply pass wait for its arithmetic: 720 x 1280 x 64 bf16 72.4 us with it, 63.8
// with this
__device__ __forceinline__ float gelu_logistic(float x) {
  const float y = x * x;
  // coefficients times -log2(e)
  float p = fmaf(-1.38621534e-09f, y, 1.46396019e-07f);
  p = fmaf(p, y, -5.90224226e-06f);
  p = fmaf(p, y, 1.00142061e-04f);
  p = fmaf(p, y, 3.82605504e-04f);
  p = fmaf(p, y, -1.05382465e-01f);
  p = fmaf(p, y, -2.30192351f);
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * p));
}

template <int ODT>
__device__ __forceinline__ float gn_act(float y, int act) {
  if (act == ACT_GELU) return ODT == DT_BF16 ? gelu_logistic(y) : gelu_erf(y);
  if (act == GN_SILU) return y * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f));
  return y;
}

template <int ODT>
__device__ __forceinline__ void gn_store(void* out, int64_t at, const f32x8& y) {
  if constexpr (ODT == DT_BF16) {
    *reinterpret_cast<bf16x8*>((unsigned short*)out + at) = pack_bf16(y);
  } else {
    f32x4* o = reinterpret_cast<f32x4*>((float*)out + at);
    o[0] = f32x4{y.v[0], y.v[1], y.v[2], y.v[3]};
    o[1] = f32x4{y.v[4], y.v[5], y.v[6], y.v[7]};
  }
}

// One workgroup per (group, image): each thread takes GN_JOIN chunks at a time, all in flight, in two passes
__global__ void __launch_bounds__(64) gn_join_kernel(const GroupNormP p) {
  const int64_t n = blockIdx.y;
  const float full = (float)p.schunk * (float)p.cg, last = (float)(p.p - (p.nchunk - 1) * p.schunk) * (float)p.cg;
  const float2* part = p.part + (n * p.groups + blockIdx.x) * p.nchunk;
  float cnt = 0.f, mu = 0.f, q = 0.f;
  auto join = [&](float k, const float2& v) __attribute__((always_inline)) {
    if (k == 0.f) return;  // nothing there (its squared distance may be infinite, and 0 of it NaN)
    const float d = v.x - mu, f = cnt == 0.f ? 1.f : k * __builtin_amdgcn_rcpf(cnt + k);
    mu = fmaf(d, f, mu);
    q = fmaf(f, fmaf((1.f - f) * d, d, v.y - q), q);
    cnt += k;
  };
  for (int e0 = threadIdx.x; e0 < p.nchunk; e0 += 64 * GN_JOIN) {
    float2 t[GN_JOIN];
#pragma unroll
    for (int j = 0; j < GN_JOIN; ++j) t[j] = e0 + j * 64 < p.nchunk ? part[e0 + j * 64] : float2{0.f, 0.f};
    float ks = 0.f, ms = 0.f, qs = 0.f;
#pragma unroll
    for (int j = 0; j < GN_JOIN; ++j) {
      const int e = e0 + j * 64;
      const float k = e < p.nchunk - 1 ? full : e == p.nchunk - 1 ? last : 0.f;
      ks += k;
      if (e < p.nchunk) ms = fmaf(k, t[j].x - t[0].x, ms);
    }
    const float per = 1.f / ks, m = fmaf(ms, per, t[0].x);
#pragma unroll
    for (int j = 0; j < GN_JOIN; ++j) {
      const int e = e0 + j * 64;
      const float k = e < p.nchunk - 1 ? full : e == p.nchunk - 1 ? last : 0.f, d = t[j].x - m;
      if (e < p.nchunk) qs = fmaf(k * per, fmaf(d, d, t[j].y), qs);
    }
    join(ks, float2{m, qs});
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float k = __shfl_xor(cnt, o, 64);
    const float2 v = float2{__shfl_xor(mu, o, 64), __shfl_xor(q, o, 64)};
    join(k, v);
  }
  if (threadIdx.x == 0) p.stat[n * p.groups + blockIdx.x] = float2{mu, rsqrtf(q + p.eps)};
}

// the affine of 8 channels, all loads in flight together (4-byte aligned: a slice of a vector qualifies)
__device__ __forceinline__ void gn_affine(const GroupNormP& p, int64_t n, int c, float (&a)[8], float (&b)[8]) {
  struct __attribute__((packed, aligned(4))) Vec { float v[8]; };
  if (p.w) {
    const Vec t = *reinterpret_cast<const Vec*>(p.w + n * p.wbs + c);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = t.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = 1.f;
  }
  if (p.b) {
    const Vec t = *reinterpret_cast<const Vec*>(p.b + n * p.bbs + c);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = t.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.f;
  }
}

template <int DT, int ODT, int ACT, bool WHOLE>
__global__ void __launch_bounds__(GN_T) gn_apply_kernel(const GroupNormP p) {
  const int tid = threadIdx.x;
  int64_t n;
  int strip, at_chunk;
  if (!gn_at<GN_BACK>(p, n, strip, at_chunk)) return;
  const int rl = tid / p.tr, oct = tid - rl * p.tr, c0 = (strip * p.tr + oct) * 8;
  const bool act = rl < p.rpb && c0 < p.c;
  const int64_t r0 = (int64_t)at_chunk * p.chunk;
  const int rows = (int)((r0 + p.chunk < p.p ? r0 + p.chunk : p.p) - r0);
  const int64_t xb = n * p.xbs + r0 * p.ldx + c0, ob = (n * p.p + r0) * p.c + c0;
  // the first rows are on their way before the statistics and the affine are asked for
  typename GnRaw<DT>::T v[UA];
  auto fetch = [&](int at) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < UA; ++k) {  // rows past the end repeat the last one
      const int r = at + k * p.rpb < rows ? at + k * p.rpb : rows - 1;
      v[k] = gn_raw<DT>(p.x, xb + (int64_t)r * p.ldx);
    }
  };
  if (!act) return;
  fetch(rl);
  float a[8], b[8];
  gn_affine(p, n, c0, a, b);
  const float2* stat = p.stat + n * p.groups;
  float mean[8];
  int g = c0 / p.cg, gc = c0 - g * p.cg;
  float2 t = stat[g];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!WHOLE && i) {
      if (++gc == p.cg) gc = 0, ++g;
      t = stat[g];
    }
    mean[i] = t.x;
    a[i] *= t.y;
  }
  for (int r = rl; r < rows; r += UA * p.rpb) {
    typename GnRaw<DT>::T u[UA];
#pragma unroll
    for (int k = 0; k < UA; ++k) u[k] = v[k];
    if (r + UA * p.rpb < rows) fetch(r + UA * p.rpb);
#pragma unroll
    for (int k = 0; k < UA; ++k) {
      if (r + k * p.rpb >= rows) break;
      const f32x8 x = gn_widen<DT>(u[k]);
      f32x8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = gn_act<ODT>(fmaf(x.v[i] - mean[i], a[i], b[i]), ACT);
      gn_store<ODT>(p.out, ob + (int64_t)(r + k * p.rpb) * p.c, y);
    }
  }
}

// One workgroup per (image, strip of whole groups): x in registers (at most NR rows per thread), two exact passes
template <int DT, int ODT, bool WHOLE, int NR>
__global__ void __launch_bounds__(GN_TS) gn_small_kernel(const GroupNormP p) {
  constexpr int NA = WHOLE ? 1 : 8, PER = WHOLE ? 8 : 1;
  __shared__ float sm[GN_TS * NA];
  __shared__ float stat[2][GN_UNIT];
  const int tid = threadIdx.x, sub = tid & (p.lpg - 1);
  const int rl = tid / p.tr, oct = tid - rl * p.tr;
  int64_t n;
  int strip, at_chunk;
  if (!gn_at<GN_PARTS>(p, n, strip, at_chunk)) return;
  const int s0 = strip * p.tr * 8, c0 = s0 + oct * 8, P = (int)p.p;
  const bool act = rl < p.rpb && c0 < p.c;
  const int sgroups = min(p.tr * 8, p.c - s0) / p.cg;
  const int units = p.cg / PER;
  const float per = 1.f / ((float)P * (float)p.cg);
  const int64_t xb = n * p.xbs + (act ? c0 : s0);
  f32x8 v[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    const int r = rl + k * p.rpb < P ? rl + k * p.rpb : P - 1;  // rows past the end repeat the last one and count nothing
    v[k] = gn_load<DT>(p.x, xb + (int64_t)r * p.ldx);
  }
  float a[8], b[8];
  gn_affine(p, n, act ? c0 : 0, a, b);
  const int full = P / p.rpb, rem = P - full * p.rpb, mine_rows = full + (rl < rem);
  // the part of the group's values that an entry with full rows, or one more, stands for
  const float w0 = (float)full / ((float)P * (float)units), w1 = (float)(full + 1) / ((float)P * (float)units);
  float mean[NA], rstd[NA];
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      float s = 0.f, first = 0.f;
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        float t = 0.f;
        if (pass) {
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const float d = v[k].v[a * PER + i] - mean[a];
            t = fmaf(d, d, t);
          }
        } else {
          t = WHOLE ? mean8(v[k]) : v[k].v[a];
          if (k == 0) first = t;
          t -= first;
        }
        if (act && k < mine_rows) s += t;
      }
      sm[tid * NA + a] = pass ? s * per : fmaf(s, 1.f / (float)max(mine_rows, 1), first);
    }
    __syncthreads();
    for_groups<GN_TS>(sgroups, p.lpg, [&](int g, bool mine) {
      const float base = pass ? 0.f : sm[g * units];
      float s = 0.f;
      for (int el = sub; el < p.rpb; el += p.lpg) {
        const float w = pass ? 1.f : el < rem ? w1 : w0;
        for (int u = 0; u < units; ++u) s = fmaf(w, sm[el * p.tr * NA + g * units + u] - base, s);
      }
      s = lanes_sum(s, p.lpg);
      if (mine && sub == 0) stat[pass][g] = pass ? rsqrtf(s + p.eps) : base + s;
    });
    __syncthreads();
    int g = oct * 8 / p.cg, gc = oct * 8 - g * p.cg;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      const float t = act ? stat[pass][g] : 0.f;
      if (++gc == p.cg) gc = 0, ++g;
      if (pass) rstd[a] = t;
      else mean[a] = t;
    }
  }
  if (!act) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] *= rstd[i / PER];
  const int64_t ob = n * p.p * p.c + c0;
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    if (rl + k * p.rpb >= P) continue;
    f32x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = gn_act<ODT>(fmaf(v[k].v[i] - mean[i / PER], a[i], b[i]), p.act);
    gn_store<ODT>(p.out, ob + (int64_t)(rl + k * p.rpb) * p.c, y);
  }
}

// workgroups of a launch over per (strip, chunk) pairs of each of n images, as gn_at has them
unsigned gn_grid(int64_t n, int64_t per, bool parts) { return (unsigned)(parts || per < 8 ? 8 * cdiv(n * per, 8) : n * 8 * cdiv(per, 8)); }

// 32 bits: the pixels of an image, the workgroups of a launch; the join's grid has at most 65535 images
bool gn_fits(int64_t n, int64_t p, int64_t c) { return p < ((int64_t)1 << 31) && n < 65536 && c < ((int64_t)1 << 19); }

// least common multiple of 8 and cg
int64_t gn_unit(int64_t cg) { return cg % 8 == 0 ? cg : cg % 4 == 0 ? 2 * cg : cg % 2 == 0 ? 4 * cg : 8 * cg; }

// lanes that join one of `groups` groups of `ents` rows of entries in a workgroup of t threads
int gn_lanes(int64_t groups, int64_t ents, int t) {
  int l = 1;
  while (l < 64 && 2 * l * groups <= t && l < ents) l *= 2;
  return l;
}

struct GnPlan {
  bool small;
  int tr, strips;     // octets per row of a workgroup, strips of them
  int nchunk;         // statistics chunks of an image
  int64_t schunk, achunk;
};

GnPlan gn_plan(int64_t n, int64_t p, int64_t c, int64_t groups) {
  GnPlan g{};
  const int64_t u = gn_unit(c / groups) / 8;  // octets a workgroup has to hold together
  // One launch where a unit's pixels are at most NRMAX rows per thread of one workgroup: past that few workgroups with
  // long chains of loads lose to the three launches over the whole chip (us, one / three launches, bf16, 32 groups: 500
  // pixels of 512 channels at 4 rows 6.0 / 9.5, 1024 at 8 rows 7.8 / 9.4, 1536 at 12 rows 10.4 / 9.4, 2048 at 16 rows
  // 11.9 / 9.4; 64 images of the first 18.6 / 24.6, of the second 30.3 / 37.4, of the last 63.5 / 67.3)
  g.small = p <= (int64_t)(GN_TS / u) * NRMAX && n * (c / 8 / u) < GN_GRID;
  if (g.small) {
    g.tr = (int)u;
    g.strips = (int)(c / 8 / u);
    g.nchunk = 1;
    return g;
  }
  g.tr = (int)(c / 8 <= GN_T ? c / 8 : u * (GN_T / u));
  g.strips = (int)cdiv(c / 8, g.tr);
  // statistics: two workgroups per CU; apply: four. Each at least UR (UA) rows per thread
  auto split = [&](int64_t blocks, int64_t least) {
    const int64_t want = cdiv(blocks, n * g.strips), len = cdiv(p, want);
    return len < least ? least : len;
  };
  g.schunk = split(2LL * device_cus(), (int64_t)UR * (GN_TT / g.tr));
  g.achunk = split(4LL * device_cus(), (int64_t)UA * (GN_T / g.tr));
  g.nchunk = (int)cdiv(p, g.schunk);
  return g;
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" size_t clarus_hip_group_norm_workspace(int64_t n, int64_t p, int64_t c, int64_t groups) {
  if (n <= 0 || p <= 0 || c <= 0 || groups <= 0 || c % groups || c % 8 || !gn_fits(n, p, c) || gn_unit(c / groups) > GN_UNIT) return 0;
  const GnPlan g = gn_plan(n, p, c, groups);
  return g.small ? 0 : (size_t)(n * groups * (g.nchunk + 1)) * sizeof(float2);
}

extern "C" int clarus_hip_group_norm(const void* x, int32_t x_dtype, int64_t x_bstride, int64_t ldx, const float* w,
                                     int64_t w_bstride, const float* b, int64_t b_bstride, void* out, int32_t o_dtype,
                                     int64_t n, int64_t p, int64_t c, int64_t groups, float eps, int32_t act,
                                     void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  CLARUS_REQUIRE(x && out, "group_norm: null operand");
  CLARUS_REQUIRE(n > 0 && p > 0 && c > 0 && groups > 0, "group_norm: empty problem");
  CLARUS_REQUIRE((x_dtype == DT_BF16 || x_dtype == DT_F32) && (o_dtype == DT_BF16 || o_dtype == DT_F32),
                 "group_norm: bf16 or fp32");
  CLARUS_REQUIRE(c % 8 == 0 && c % groups == 0, "group_norm: channels a multiple of 8 and of the groups");
  CLARUS_REQUIRE(gn_fits(n, p, c), "group_norm: too large");
  CLARUS_REQUIRE(gn_unit(c / groups) <= GN_UNIT, "group_norm: lcm(8, channels per group) at most %d", GN_UNIT);
  CLARUS_REQUIRE(act == ACT_NONE || act == ACT_GELU || act == CLARUS_ACT_SILU, "group_norm: act none, GELU or SiLU");
  const int64_t es = x_dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(ldx >= c && (n == 1 || x_bstride >= 0), "group_norm: strides");
  CLARUS_REQUIRE(aligned(x, 16) && aligned(out, 16) && ldx * es % 16 == 0 && x_bstride * es % 16 == 0,
                 "group_norm: x and out 16-byte aligned rows");
  CLARUS_REQUIRE((w_bstride == 0 || w_bstride >= c) && (b_bstride == 0 || b_bstride >= c), "group_norm: affine strides");
  CLARUS_REQUIRE(eps >= 0.f && eps < INFINITY, "group_norm: eps finite and not negative");
  const size_t need = clarus_hip_group_norm_workspace(n, p, c, groups);
  CLARUS_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && aligned(scratch, 8)), "group_norm: scratch %zu < %zu bytes", scratch_bytes, need);
  const GnPlan g = gn_plan(n, p, c, groups);
  const int64_t achunks = g.small ? 1 : cdiv(p, g.achunk);
  CLARUS_REQUIRE(n * g.strips * std::max<int64_t>(g.nchunk, achunks) < GN_GRID, "group_norm: too large");
  GroupNormP k{};
  k.x = x; k.out = out; k.w = w; k.b = b;
  k.stat = (float2*)scratch;
  k.part = k.stat + n * groups;
  k.xbs = x_bstride; k.ldx = ldx; k.p = p; k.schunk = g.schunk;
  k.wbs = w_bstride; k.bbs = b_bstride;
  k.c = (int)c; k.groups = (int)groups; k.cg = (int)(c / groups); k.nchunk = g.nchunk;
  k.n = (int)n; k.strips = g.strips; k.chunks = 1; k.tr = g.tr; k.eps = eps; k.act = act;
  hipStream_t st = (hipStream_t)stream;
  const bool whole = k.cg % 8 == 0;
  const int64_t sgroups = (c < 8 * g.tr ? c : 8 * g.tr) / k.cg;
  k.rpb = (g.small ? GN_TS : GN_TT) / g.tr;
  k.lpg = gn_lanes(sgroups, k.rpb, g.small ? GN_TS : GN_TT);
  if (g.small) {
    const int nr = (int)cdiv(p, k.rpb);
    const dim3 grid(gn_grid(n, g.strips, true));
    note_kernel("gn_small_kernel strips=%d rows=%d", g.strips, nr);
#define CLARUS_GN_S(DT, ODT, W)                                                                                  \
  do {                                                                                                           \
    if (nr <= 4) hipLaunchKernelGGL((gn_small_kernel<DT, ODT, W, 4>), grid, dim3(GN_TS), 0, st, k);              \
    else hipLaunchKernelGGL((gn_small_kernel<DT, ODT, W, NRMAX>), grid, dim3(GN_TS), 0, st, k);                  \
  } while (0)
#define CLARUS_GN(DT, ODT)                \
  do {                                    \
    if (whole) CLARUS_GN_S(DT, ODT, true); \
    else CLARUS_GN_S(DT, ODT, false);     \
  } while (0)
    if (x_dtype == DT_BF16) {
      if (o_dtype == DT_BF16) CLARUS_GN(DT_BF16, DT_BF16);
      else CLARUS_GN(DT_BF16, DT_F32);
    } else {
      if (o_dtype == DT_BF16) CLARUS_GN(DT_F32, DT_BF16);
      else CLARUS_GN(DT_F32, DT_F32);
    }
#undef CLARUS_GN
#undef CLARUS_GN_S
    return check_launch("group_norm");
  }
  k.chunk = g.schunk;
  k.chunks = g.nchunk;
  const dim3 sgrid(gn_grid(n, (int64_t)g.strips * g.nchunk, false));
  note_kernel("gn_stats_kernel + gn_apply_kernel nchunk=%d strips=%d", g.nchunk, g.strips);
  if (x_dtype == DT_BF16) {
    if (whole) hipLaunchKernelGGL((gn_stats_kernel<DT_BF16, true>), sgrid, dim3(GN_TT), 0, st, k);
    else hipLaunchKernelGGL((gn_stats_kernel<DT_BF16, false>), sgrid, dim3(GN_TT), 0, st, k);
  } else {
    if (whole) hipLaunchKernelGGL((gn_stats_kernel<DT_F32, true>), sgrid, dim3(GN_TT), 0, st, k);
    else hipLaunchKernelGGL((gn_stats_kernel<DT_F32, false>), sgrid, dim3(GN_TT), 0, st, k);
  }
  hipLaunchKernelGGL(gn_join_kernel, dim3((unsigned)groups, (unsigned)n), dim3(64), 0, st, k);
  k.chunk = g.achunk;
  k.chunks = (int)achunks;
  k.rpb = GN_T / g.tr;
  const dim3 grid(gn_grid(n, g.strips * achunks, false));
#define CLARUS_GN_A(DT, ODT, ACT)                                                                      \
  do {                                                                                                 \
    if (whole) hipLaunchKernelGGL((gn_apply_kernel<DT, ODT, ACT, true>), grid, dim3(GN_T), 0, st, k);  \
    else hipLaunchKernelGGL((gn_apply_kernel<DT, ODT, ACT, false>), grid, dim3(GN_T), 0, st, k);       \
  } while (0)
#define CLARUS_GN(DT, ODT)                                  \
  do {                                                      \
    if (act == ACT_NONE) CLARUS_GN_A(DT, ODT, ACT_NONE);    \
    else if (act == ACT_GELU) CLARUS_GN_A(DT, ODT, ACT_GELU); \
    else CLARUS_GN_A(DT, ODT, GN_SILU);                     \
  } while (0)
  if (x_dtype == DT_BF16) {
    if (o_dtype == DT_BF16) CLARUS_GN(DT_BF16, DT_BF16);
    else CLARUS_GN(DT_BF16, DT_F32);
  } else {
    if (o_dtype == DT_BF16) CLARUS_GN(DT_F32, DT_BF16);
    else CLARUS_GN(DT_F32, DT_F32);
  }
#undef CLARUS_GN
#undef CLARUS_GN_A
  return check_launch("group_norm");
}
