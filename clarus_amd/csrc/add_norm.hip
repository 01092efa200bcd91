// A block's output added to the residual stream, and the norm that the next block reads, on gfx950; per row of C channels:
//   sum = x + scale gate (post(y) pw + pb),   norm = pre(sum) w + b,
// post and pre nothing, LayerNorm or RMS. One pass: a row lies in the registers of G lanes (up to 4096 channels in one
// wave, up to 16384 in four), its statistics cross the lanes by DPP, and each of x, y, sum and norm moves once.
//
// Statistics: the mean of the row, then mean and mean square of the differences from it, which also takes away what the
// first sum had rounded: no cancellation, whatever the mean's size, and equal values have a variance of 0 to 2^-46 of their
// square. Differences are scaled by 2^-7 or so before they are squared: values within 2^60 stay finite.
// What bounds it: memory. 28800 rows of 512, an fp32 stream and a bf16 norm: 38.2 us, 4.6 TB/s (34.3 at a large copy's rate).
// Past 1024 channels a lane's part of the affine does not stay in registers: it is read again for every row (from L2), and lanes hold
// 4 or 8 octets whether the row fills them or not. As many elements as 57600 rows of 512, fp32 / bf16 stream, 69 / 46 us at a copy's rate:
// 1024 channels 73 / 48 us, 1536 95 / 76, 2048 84 / 60, 4096 94 / 71, 6144 148 / 126, 8192 134 / 107, 16384 98 / 75.
#include <algorithm>

#include "capi.hpp"
#include "common.hpp"

namespace clarus {

namespace {

constexpr int AN_T = 256;
constexpr int AN_ROWS = 8;  // rows of a workgroup's slot, at most

enum : int { NORM_NONE = CLARUS_PRO_NONE, NORM_LN = CLARUS_PRO_LN, NORM_RMS = CLARUS_PRO_RMS };

struct AddNormP {
  const void *x, *y;
  void *sum, *norm;
  const float *gate, *pw, *pb, *w, *b;
  int64_t xbs, ldx, ybs, ldy;
  int64_t gbs, pwbs, pbbs, wbs, bbs;
  int64_t rows;
  unsigned chunks;   // workgroups of an image
  int per;           // rows of a workgroup
  int oct;           // octets of a row
  int g;             // lanes of a row within a wave
  int s_dt, n_dt, post, pre;
  float scale, eps, inv_c;
  float down, up;    // 2^-k and 2^2k / c: the mean square of differences from the sum of (2^-k difference)^2
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// sum over the g consecutive lanes of a row (a power of two), WPR waves of them
template <int WPR>
__device__ __forceinline__ float an_sum(float v, int g, float* lds) {
  if (g >= 2) v = dpp_add<0xB1>(v);    // quad_perm 1 0 3 2
  if (g >= 4) v = dpp_add<0x4E>(v);    // quad_perm 2 3 0 1
  if (g >= 8) v = dpp_add<0x141>(v);   // mirror of 8
  if (g >= 16) v = dpp_add<0x140>(v);  // mirror of 16
  if (g >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (g >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (WPR > 1) {
    __syncthreads();  // the sums before have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v += lds[i];
  }
  return v;
}

// v normed in place; octets past the row's end hold 0 and stay 0
template <int NO, int WPR>
__device__ __forceinline__ void an_norm(const AddNormP& p, int kind, const bool (&in)[NO], f32x8 (&v)[NO], float* lds) {
  float mean = 0.f;
  if (kind == NORM_LN) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[i].v[e];
    mean = an_sum<WPR>(s, p.g, lds) * p.inv_c;
  }
  float d1 = 0.f, d2 = 0.f;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = in[i] ? v[i].v[e] - mean : 0.f, t = d * p.down;
      v[i].v[e] = d;
      d1 += d;
      d2 = fmaf(t, t, d2);
    }
  float var = an_sum<WPR>(d2, p.g, lds) * p.up, off = 0.f;
  if (kind == NORM_LN) {
    off = an_sum<WPR>(d1, p.g, lds) * p.inv_c;
    var = fmaxf(fmaf(-off, off, var), 0.f);
  }
  const float rstd = 1.f / sqrtf(var + p.eps);
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i].v[e] = (v[i].v[e] - off) * rstd;
}

__device__ __forceinline__ f32x8 an_vec(const float* p, int64_t at, float none) {
  if (p) return load8<DT_F32>(p + at);
  f32x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = none;
  return r;
}

__device__ __forceinline__ void an_store(void* p, int dt, int64_t at, const f32x8& v) {
  if (dt == DT_BF16) {
    *reinterpret_cast<bf16x8*>((unsigned short*)p + at) = pack_bf16(v);
  } else {
    f32x4* q = reinterpret_cast<f32x4*>((float*)p + at);
    q[0] = f32x4{v.v[0], v.v[1], v.v[2], v.v[3]};
    q[1] = f32x4{v.v[4], v.v[5], v.v[6], v.v[7]};
  }
}

// NO: octets of a row per lane; WPR: waves per row
template <int XDT, int YDT, int NO, int WPR>
__global__ void __launch_bounds__(AN_T) add_norm_kernel(const AddNormP p) {
  constexpr bool KEEP = NO <= 2;  // the affine stays in registers over the rows
  __shared__ float lds[4];
  const int tid = threadIdx.x, g = WPR > 1 ? AN_T : p.g, slots = AN_T / g, slot = tid / g, lane = tid - slot * g;
  const unsigned n = blockIdx.x / p.chunks, chunk = blockIdx.x - n * p.chunks;
  const int64_t r0 = (int64_t)chunk * p.per, r1 = r0 + p.per < p.rows ? r0 + p.per : p.rows;
  const int64_t c = (int64_t)p.oct * 8;
  bool in[NO];
  int64_t col[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) {
    in[i] = lane + i * g < p.oct;
    col[i] = (in[i] ? lane + i * g : 0) * 8;
  }
  const bool has_y = p.y != nullptr;
  f32x8 ga[KEEP ? NO : 1], gb[KEEP ? NO : 1], wa[KEEP ? NO : 1], wb[KEEP ? NO : 1];
  auto outer = [&](int i, f32x8& a, f32x8& b) __attribute__((always_inline)) {  // scale gate pw, scale gate pb
    const f32x8 gate = an_vec(p.gate, n * p.gbs + col[i], 1.f);
    a = an_vec(p.pw, n * p.pwbs + col[i], 1.f);
    b = an_vec(p.pb, n * p.pbbs + col[i], 0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = gate.v[e] * p.scale;
      a.v[e] *= s;
      b.v[e] *= s;
    }
  };
  auto inner = [&](int i, f32x8& a, f32x8& b) __attribute__((always_inline)) {
    a = an_vec(p.w, n * p.wbs + col[i], 1.f);
    b = an_vec(p.b, n * p.bbs + col[i], 0.f);
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      if (has_y) outer(i, ga[i], gb[i]);
      if (p.norm) inner(i, wa[i], wb[i]);
    }
  }
  const unsigned char *xp = (const unsigned char*)p.x, *yp = (const unsigned char*)p.y;
  constexpr int XS = XDT == DT_BF16 ? 2 : 4, YS = YDT == DT_BF16 ? 2 : 4;
  // the slots of a wave stay together (a row past the end repeats the last and is not written)
#pragma unroll 1
  for (int64_t r = r0; r < r1; r += slots) {
    const bool live = r + slot < r1;
    const int64_t row = live ? r + slot : r1 - 1;
    f32x8 v[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) v[i] = load8<XDT>(xp + (n * p.xbs + row * p.ldx + col[i]) * XS);
    const int64_t to = (n * p.rows + row) * c;
    if (has_y) {
      f32x8 y[NO];
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        y[i] = load8<YDT>(yp + (n * p.ybs + row * p.ldy + col[i]) * YS);
        if (!in[i]) y[i] = zero8();
      }
      if (p.post != NORM_NONE) an_norm<NO, WPR>(p, p.post, in, y, lds);
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        if constexpr (!KEEP) outer(i, ga[0], gb[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i].v[e] += fmaf(y[i].v[e], ga[KEEP ? i : 0].v[e], gb[KEEP ? i : 0].v[e]);
        if (in[i] && live) an_store(p.sum, p.s_dt, to + col[i], v[i]);
      }
    }
    if (p.norm) {
#pragma unroll
      for (int i = 0; i < NO; ++i)
        if (!in[i]) v[i] = zero8();
      if (p.pre != NORM_NONE) an_norm<NO, WPR>(p, p.pre, in, v, lds);
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        if constexpr (!KEEP) inner(i, wa[0], wb[0]);
        f32x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h.v[e] = fmaf(v[i].v[e], wa[KEEP ? i : 0].v[e], wb[KEEP ? i : 0].v[e]);
        if (in[i] && live) an_store(p.norm, p.n_dt, to + col[i], h);
      }
    }
  }
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" int clarus_hip_add_norm(const ClarusAddNormArgs* a, void* stream) {
  clear_error();
  CLARUS_REQUIRE(a, "add_norm: null arguments");
  CLARUS_REQUIRE(a->x && (!a->y || a->sum) && (a->y || a->norm), "add_norm: null operand");
  CLARUS_REQUIRE(a->n > 0 && a->rows > 0 && a->c > 0, "add_norm: empty problem");
  const int64_t big = (int64_t)1 << 31;
  CLARUS_REQUIRE(a->n < (1 << 23) && a->rows < big && a->n * a->rows < big, "add_norm: fewer than 2^31 rows and 2^23 images");
  CLARUS_REQUIRE(a->c % 8 == 0 && a->c <= 16384, "add_norm: channels a multiple of 8 up to 16384");
  for (const int32_t dt : {a->x_dtype, a->y_dtype, a->sum_dtype, a->norm_dtype})
    CLARUS_REQUIRE(dt == DT_BF16 || dt == DT_F32, "add_norm: bf16 or fp32");
  for (const int32_t k : {a->post, a->pre}) CLARUS_REQUIRE(k == NORM_NONE || k == NORM_LN || k == NORM_RMS, "add_norm: norms");
  CLARUS_REQUIRE(a->eps >= 0.f && a->eps < INFINITY && a->scale == a->scale && fabsf(a->scale) < INFINITY, "add_norm: eps, scale");
  const int64_t xs = a->x_dtype == DT_BF16 ? 2 : 4, ys = a->y_dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->x, 16) && a->ldx * xs % 16 == 0 && a->x_bstride * xs % 16 == 0 &&
                     (!a->y || (aligned(a->y, 16) && a->ldy * ys % 16 == 0 && a->y_bstride * ys % 16 == 0)) && aligned(a->sum, 16) &&
                     aligned(a->norm, 16),
                 "add_norm: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldx >= 0 && a->x_bstride >= 0 && a->ldy >= 0 && a->y_bstride >= 0, "add_norm: strides");
  for (const float* f : {a->gate, a->post_w, a->post_b, a->w, a->b}) CLARUS_REQUIRE(aligned(f, 16), "add_norm: 16-byte aligned affine");
  for (const int64_t s : {a->gate_bstride, a->post_w_bstride, a->post_b_bstride, a->w_bstride, a->b_bstride})
    CLARUS_REQUIRE(s >= 0 && s % 4 == 0, "add_norm: strides of the affine");
  AddNormP k{};
  k.x = a->x; k.y = a->y; k.sum = a->sum; k.norm = a->norm;
  k.gate = a->gate; k.pw = a->post_w; k.pb = a->post_b; k.w = a->w; k.b = a->b;
  k.xbs = a->x_bstride; k.ldx = a->ldx; k.ybs = a->y_bstride; k.ldy = a->ldy;
  k.gbs = a->gate_bstride; k.pwbs = a->post_w_bstride; k.pbbs = a->post_b_bstride; k.wbs = a->w_bstride; k.bbs = a->b_bstride;
  k.rows = a->rows; k.oct = (int)(a->c / 8);
  k.s_dt = a->sum_dtype; k.n_dt = a->norm_dtype; k.post = a->post; k.pre = a->pre;
  k.scale = a->scale; k.eps = a->eps; k.inv_c = 1.f / (float)a->c;
  int half = 0;
  while ((1ll << (2 * half)) < a->c) ++half;
  k.down = ldexpf(1.f, -half);
  k.up = ldexpf(1.f, 2 * half) / (float)a->c;
  const bool wide = k.oct > 512;
  k.g = 1;
  while (k.g < 64 && k.g < k.oct) k.g *= 2;
  const int slots = wide ? 1 : AN_T / k.g;
  int64_t each = AN_ROWS;
  while (each > 1 && a->n * cdiv(a->rows, slots * each) < 8 * device_cus()) each /= 2;
  // a launch holds fewer than 2^32 threads
  while (a->n * cdiv(a->rows, slots * each) >= (1 << 23)) each *= 2;
  k.per = (int)(slots * each);
  k.chunks = (unsigned)cdiv(a->rows, k.per);
  const dim3 grid((unsigned)(a->n * k.chunks));
  hipStream_t st = (hipStream_t)stream;
  const int no = (int)cdiv(k.oct, wide ? AN_T : k.g);
  note_kernel("add_norm_kernel octets=%d lanes=%d rows=%d", no, wide ? AN_T : k.g, k.per);
#define CLARUS_AN(X, Y)                                                                                             \
  do {                                                                                                              \
    if (wide) hipLaunchKernelGGL((add_norm_kernel<X, Y, 8, 4>), grid, dim3(AN_T), 0, st, k);                        \
    else if (no == 1) hipLaunchKernelGGL((add_norm_kernel<X, Y, 1, 1>), grid, dim3(AN_T), 0, st, k);                \
    else if (no == 2) hipLaunchKernelGGL((add_norm_kernel<X, Y, 2, 1>), grid, dim3(AN_T), 0, st, k);                \
    else if (no <= 4) hipLaunchKernelGGL((add_norm_kernel<X, Y, 4, 1>), grid, dim3(AN_T), 0, st, k);                \
    else hipLaunchKernelGGL((add_norm_kernel<X, Y, 8, 1>), grid, dim3(AN_T), 0, st, k);                             \
  } while (0)
  if (a->x_dtype == DT_BF16) {
    if (a->y_dtype == DT_BF16) CLARUS_AN(DT_BF16, DT_BF16);
    else CLARUS_AN(DT_BF16, DT_F32);
  } else {
    if (a->y_dtype == DT_BF16) CLARUS_AN(DT_F32, DT_BF16);
    else CLARUS_AN(DT_F32, DT_F32);
  }
#undef CLARUS_AN
  return check_launch("add_norm");
}
