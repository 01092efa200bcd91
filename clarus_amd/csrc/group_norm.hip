// Group norm of an NHWC map with its activation on gfx950.
//
// For image n and group g of cg = C / G channels, over the P pixels x cg channels of the group:
//   mean, var = biased;  y = act((x - mean) * rsqrt(var + eps) * weight[c] + bias[c])
//
// Statistics without cancellation: a thread takes UR rows of its channel octet into registers, has
// their mean and squared distances exactly (two passes over registers), and joins them to its
// running (mean, M2); threads, channels of a group and chunks of pixels are then joined by
//   mean = sum(cnt mean) / sum(cnt),  M2 = sum(M2 + cnt (mean_i - mean)^2)
// in a fixed order, all in fp32: no sum of squares of uncentred values occurs, so a mean far from
// zero or a single large value costs no digits, and the result is deterministic.
//   1. gn_stats_kernel: per (image, chunk of pixels) the groups' mean and M2
//   2. gn_join_kernel:  per (image, group) the chunks joined: mean, rstd
//   3. gn_apply_kernel: y, one read of x and one write
#include "capi.hpp"
#include "common.hpp"

namespace clarus {

namespace {

constexpr int GN_T = 256;   // threads of a workgroup
constexpr int UR = 8;       // rows in flight per thread
constexpr int GN_SILU = 3;  // CLARUS_ACT_SILU

struct GroupNormP {
  const void* x;
  void* out;
  const float* w;    // [C] or [N][C] (wbs = C), or null
  const float* b;
  float2* part;      // [n][chunk][G] mean, M2
  float2* stat;      // [n][G] mean, rstd
  int64_t xbs, ldx;  // image and pixel stride of x (elements)
  int64_t p, chunk;  // pixels, pixels per chunk
  int64_t wbs, bbs;
  int c, groups, cg, nchunk;
  int tr, rpb;       // threads per row (octets of a strip), rows per pass of a workgroup
  float eps;
};

template <int DT>
__device__ __forceinline__ f32x8 gn_load(const void* x, int64_t i) {
  return load8<DT>((const unsigned char*)x + i * (DT == DT_BF16 ? 2 : 4));
}

__device__ __forceinline__ float wave_sum(float v) { return group_sum<64>(v); }

// WHOLE: cg % 8 == 0, an octet lies in one group and is one set of 8 values per row
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(GN_T) gn_stats_kernel(const GroupNormP p) {
  constexpr int NA = WHOLE ? 1 : 8;  // (mean, M2) pairs per thread
  constexpr int PER = WHOLE ? 8 : 1;
  __shared__ float sm[GN_T * NA], s2[GN_T * NA];
  const int tid = threadIdx.x;
  const int rl = tid / p.tr, oct = tid - rl * p.tr;
  const int64_t n = blockIdx.z, r0 = (int64_t)blockIdx.x * p.chunk;
  const int rows = (int)((r0 + p.chunk < p.p ? r0 + p.chunk : p.p) - r0);
  const int c0 = blockIdx.y * p.tr * 8;  // first channel of the strip
  const bool act = rl < p.rpb && c0 + oct * 8 < p.c;
  float mean[NA], m2[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) mean[i] = m2[i] = 0.f;
  int cnt = 0;  // rows so far
  if (act) {
    const int64_t base = n * p.xbs + r0 * p.ldx + c0 + oct * 8;
    int r = rl;
    for (; r + (UR - 1) * p.rpb < rows; r += UR * p.rpb) {
      f32x8 v[UR];
#pragma unroll
      for (int k = 0; k < UR; ++k) v[k] = gn_load<DT>(p.x, base + (int64_t)(r + k * p.rpb) * p.ldx);
      const float join = (float)cnt / (float)(cnt + UR), part = (float)UR / (float)(cnt + UR);
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < UR; ++k)
#pragma unroll
          for (int i = 0; i < PER; ++i) s += v[k].v[a * PER + i];
        const float m = s * (1.f / (UR * PER));
#pragma unroll
        for (int k = 0; k < UR; ++k)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const float d = v[k].v[a * PER + i] - m;
            q = fmaf(d, d, q);
          }
        const float d = m - mean[a];
        mean[a] = fmaf(d, part, mean[a]);
        m2[a] += q + d * d * (join * (UR * PER));
      }
      cnt += UR;
    }
    for (; r < rows; r += p.rpb) {
      const f32x8 v = gn_load<DT>(p.x, base + (int64_t)r * p.ldx);
      const float join = (float)cnt / (float)(cnt + 1), part = 1.f / (float)(cnt + 1);
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) s += v.v[a * PER + i];
        const float m = s * (1.f / PER);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float d = v.v[a * PER + i] - m;
          q = fmaf(d, d, q);
        }
        const float d = m - mean[a];
        mean[a] = fmaf(d, part, mean[a]);
        m2[a] += q + d * d * (join * PER);
      }
      ++cnt;
    }
  }
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    sm[tid * NA + a] = mean[a];
    s2[tid * NA + a] = m2[a];
  }
  __syncthreads();
  // a wave joins one group at a time: entries (row lane, unit), unit = an octet or a channel
  const int wave = tid >> 6, lane = tid & 63;
  const int units = p.cg / PER;                 // entries of a group per row lane
  const int sgroups = min(p.tr * 8, p.c - c0) / p.cg;  // groups of the strip
  for (int g = wave; g < sgroups; g += GN_T / 64) {
    float cs = 0.f, ms = 0.f;
    for (int e = lane; e < units * p.rpb; e += 64) {
      const int el = e / units, u = e - el * units;
      const float k = (float)(PER * ((rows - el + p.rpb - 1) / p.rpb));  // el < rpb: 0 where el >= rows
      cs += k;
      ms = fmaf(k, sm[el * p.tr * NA + g * units + u], ms);
    }
    cs = wave_sum(cs);
    const float mu = wave_sum(ms) / cs;
    float q = 0.f;
    for (int e = lane; e < units * p.rpb; e += 64) {
      const int el = e / units, u = e - el * units;
      const float k = (float)(PER * ((rows - el + p.rpb - 1) / p.rpb));
      const int at = el * p.tr * NA + g * units + u;
      const float d = sm[at] - mu;
      q += fmaf(d * d, k, s2[at]);
    }
    q = wave_sum(q);
    if (lane == 0) p.part[((int64_t)n * p.nchunk + blockIdx.x) * p.groups + c0 / p.cg + g] = float2{mu, q};
  }
}

__global__ void __launch_bounds__(64) gn_join_kernel(const GroupNormP p) {
  const int g = blockIdx.x, lane = threadIdx.x;
  const int64_t n = blockIdx.y;
  const float2* part = p.part + n * p.nchunk * p.groups + g;
  const float last = (float)(p.p - (p.nchunk - 1) * p.chunk) * (float)p.cg, full = (float)p.chunk * (float)p.cg;
  float ms = 0.f;
  for (int e = lane; e < p.nchunk; e += 64) ms = fmaf(e == p.nchunk - 1 ? last : full, part[(int64_t)e * p.groups].x, ms);
  const float total = (float)p.p * (float)p.cg;
  const float mu = wave_sum(ms) / total;
  float q = 0.f;
  for (int e = lane; e < p.nchunk; e += 64) {
    const float2 v = part[(int64_t)e * p.groups];
    const float d = v.x - mu;
    q += fmaf(d * d, e == p.nchunk - 1 ? last : full, v.y);
  }
  q = wave_sum(q);
  if (lane == 0) p.stat[n * p.groups + g] = float2{mu, rsqrtf(q / total + p.eps)};
}

template <int ACT>
__device__ __forceinline__ float gn_act(float y) {
  if constexpr (ACT == ACT_GELU) return gelu_erf(y);
  if constexpr (ACT == GN_SILU) return y * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f));
  return y;
}

template <int DT, int ODT, int ACT>
__global__ void __launch_bounds__(GN_T) gn_apply_kernel(const GroupNormP p) {
  const int tid = threadIdx.x;
  const int rl = tid / p.tr, oct = tid - rl * p.tr;
  const int c0 = (blockIdx.y * p.tr + oct) * 8;
  if (rl >= p.rpb || c0 >= p.c) return;
  const int64_t n = blockIdx.z, r0 = (int64_t)blockIdx.x * p.chunk;
  const int rows = (int)((r0 + p.chunk < p.p ? r0 + p.chunk : p.p) - r0);
  float mean[8], a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 s = p.stat[n * p.groups + (c0 + i) / p.cg];
    mean[i] = s.x;
    a[i] = s.y * (p.w ? p.w[n * p.wbs + c0 + i] : 1.f);
    b[i] = p.b ? p.b[n * p.bbs + c0 + i] : 0.f;
  }
  const int64_t xb = n * p.xbs + r0 * p.ldx + c0, ob = (n * p.p + r0) * p.c + c0;
  auto put = [&](const f32x8& v, int r) __attribute__((always_inline)) {
    f32x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = gn_act<ACT>(fmaf(v.v[i] - mean[i], a[i], b[i]));
    const int64_t at = ob + (int64_t)r * p.c;
    if constexpr (ODT == DT_BF16) {
      *reinterpret_cast<bf16x8*>((unsigned short*)p.out + at) = pack_bf16(y);
    } else {
      f32x4* o = reinterpret_cast<f32x4*>((float*)p.out + at);
      o[0] = f32x4{y.v[0], y.v[1], y.v[2], y.v[3]};
      o[1] = f32x4{y.v[4], y.v[5], y.v[6], y.v[7]};
    }
  };
  constexpr int UA = 4;
  int r = rl;
  for (; r + (UA - 1) * p.rpb < rows; r += UA * p.rpb) {
    f32x8 v[UA];
#pragma unroll
    for (int k = 0; k < UA; ++k) v[k] = gn_load<DT>(p.x, xb + (int64_t)(r + k * p.rpb) * p.ldx);
#pragma unroll
    for (int k = 0; k < UA; ++k) put(v[k], r + k * p.rpb);
  }
  for (; r < rows; r += p.rpb) put(gn_load<DT>(p.x, xb + (int64_t)r * p.ldx), r);
}

struct GnPlan {
  int tr, rpb, strips, nchunk;
  int64_t chunk;
};

// least common multiple of 8 and cg
int64_t gn_unit(int64_t cg) { return cg % 8 == 0 ? cg : cg % 4 == 0 ? 2 * cg : cg % 2 == 0 ? 4 * cg : 8 * cg; }

GnPlan gn_plan(int64_t n, int64_t p, int64_t c, int64_t groups) {
  GnPlan g;
  const int64_t u = gn_unit(c / groups) / 8;  // octets a workgroup has to hold together
  g.tr = (int)(c / 8 <= GN_T ? c / 8 : u * (GN_T / u));
  g.strips = (int)cdiv(c / 8, g.tr);
  g.rpb = GN_T / g.tr;
  // about four workgroups per CU, each at least UR rows per thread
  int64_t want = cdiv(4LL * device_cus(), n * g.strips);
  int64_t chunk = cdiv(p, want < 1 ? 1 : want);
  const int64_t least = (int64_t)UR * g.rpb;
  chunk = cdiv(chunk < least ? least : chunk, g.rpb) * g.rpb;
  g.chunk = chunk < p ? chunk : p;
  g.nchunk = (int)cdiv(p, g.chunk);
  return g;
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" size_t clarus_hip_group_norm_workspace(int64_t n, int64_t p, int64_t c, int64_t groups) {
  if (n <= 0 || p <= 0 || c <= 0 || groups <= 0 || c % groups || c % 8 || gn_unit(c / groups) > 8 * GN_T) return 0;
  const GnPlan g = gn_plan(n, p, c, groups);
  return (size_t)(n * groups * (g.nchunk + 1)) * sizeof(float2);
}

extern "C" int clarus_hip_group_norm(const void* x, int32_t x_dtype, int64_t x_bstride, int64_t ldx, const float* w,
                                     int64_t w_bstride, const float* b, int64_t b_bstride, void* out, int32_t o_dtype,
                                     int64_t n, int64_t p, int64_t c, int64_t groups, float eps, int32_t act,
                                     void* scratch, size_t scratch_bytes, void* stream) {
  clear_error();
  CLARUS_REQUIRE(x && out && scratch, "group_norm: null operand");
  CLARUS_REQUIRE(n > 0 && p > 0 && c > 0 && groups > 0, "group_norm: empty problem");
  CLARUS_REQUIRE((x_dtype == DT_BF16 || x_dtype == DT_F32) && (o_dtype == DT_BF16 || o_dtype == DT_F32),
                 "group_norm: bf16 or fp32");
  CLARUS_REQUIRE(c % 8 == 0 && c % groups == 0, "group_norm: channels a multiple of 8 and of the groups");
  CLARUS_REQUIRE(gn_unit(c / groups) <= 8 * GN_T, "group_norm: lcm(8, channels per group) at most %d", 8 * GN_T);
  CLARUS_REQUIRE(act == ACT_NONE || act == ACT_GELU || act == CLARUS_ACT_SILU, "group_norm: act none, GELU or SiLU");
  const int64_t es = x_dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(ldx >= c && (n == 1 || x_bstride >= 0), "group_norm: strides");
  CLARUS_REQUIRE(aligned(x, 16) && aligned(out, 16) && ldx * es % 16 == 0 && x_bstride * es % 16 == 0,
                 "group_norm: x and out 16-byte aligned rows");
  CLARUS_REQUIRE((w_bstride == 0 || w_bstride >= c) && (b_bstride == 0 || b_bstride >= c), "group_norm: affine strides");
  // float counts and the pixel index of a chunk: 2^31 pixels, 65535 images and strips are the launch's limits
  CLARUS_REQUIRE(p < ((int64_t)1 << 31) && n < 65536 && c < ((int64_t)1 << 24), "group_norm: too large");
  const size_t need = clarus_hip_group_norm_workspace(n, p, c, groups);
  CLARUS_REQUIRE(scratch_bytes >= need && aligned(scratch, 8), "group_norm: scratch %zu < %zu bytes", scratch_bytes, need);
  const GnPlan g = gn_plan(n, p, c, groups);
  GroupNormP k{};
  k.x = x; k.out = out; k.w = w; k.b = b;
  k.stat = (float2*)scratch;
  k.part = k.stat + n * groups;
  k.xbs = x_bstride; k.ldx = ldx; k.p = p; k.chunk = g.chunk;
  k.wbs = w_bstride; k.bbs = b_bstride;
  k.c = (int)c; k.groups = (int)groups; k.cg = (int)(c / groups); k.nchunk = g.nchunk;
  k.tr = g.tr; k.rpb = g.rpb; k.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)g.nchunk, (unsigned)g.strips, (unsigned)n);
  note_kernel("gn_stats_kernel + gn_apply_kernel nchunk=%d strips=%d", g.nchunk, g.strips);
  const bool whole = k.cg % 8 == 0;
  if (x_dtype == DT_BF16) {
    if (whole) hipLaunchKernelGGL((gn_stats_kernel<DT_BF16, true>), grid, dim3(GN_T), 0, st, k);
    else hipLaunchKernelGGL((gn_stats_kernel<DT_BF16, false>), grid, dim3(GN_T), 0, st, k);
  } else {
    if (whole) hipLaunchKernelGGL((gn_stats_kernel<DT_F32, true>), grid, dim3(GN_T), 0, st, k);
    else hipLaunchKernelGGL((gn_stats_kernel<DT_F32, false>), grid, dim3(GN_T), 0, st, k);
  }
  hipLaunchKernelGGL(gn_join_kernel, dim3((unsigned)groups, (unsigned)n), dim3(64), 0, st, k);
#define CLARUS_GN(DT, ODT)                                                                               \
  do {                                                                                                   \
    if (act == ACT_NONE) hipLaunchKernelGGL((gn_apply_kernel<DT, ODT, ACT_NONE>), grid, dim3(GN_T), 0, st, k);       \
    else if (act == ACT_GELU) hipLaunchKernelGGL((gn_apply_kernel<DT, ODT, ACT_GELU>), grid, dim3(GN_T), 0, st, k);  \
    else hipLaunchKernelGGL((gn_apply_kernel<DT, ODT, GN_SILU>), grid, dim3(GN_T), 0, st, k);                        \
  } while (0)
  if (x_dtype == DT_BF16) {
    if (o_dtype == DT_BF16) CLARUS_GN(DT_BF16, DT_BF16);
    else CLARUS_GN(DT_BF16, DT_F32);
  } else {
    if (o_dtype == DT_BF16) CLARUS_GN(DT_F32, DT_BF16);
    else CLARUS_GN(DT_F32, DT_F32);
  }
#undef CLARUS_GN
  return check_launch("group_norm");
}
