// Rotary positions with several axes (time, height, width) on the heads of NHWC rows, on gfx950:
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = 2 pi pos[token, axis(j)] turn[j]
// for the pairs j of every head's columns; the other columns are copied. The heads of a token share its angles.
//
// A workgroup works out cos and sin of its tokens' pairs into LDS, then its threads, each with a place of its own in a
// row (one head's V pairs, or V columns that stay), go over the tokens, four in flight. The turns pos * turn[j] and
// their fraction are held in 64 bits (a position of a million is a million radians of the fastest pair, of which fp32
// keeps one digit behind the point); the fraction is below 1/2 and goes through sincospi in 32.
// What bounds it: memory, each element read and written once. 57600 tokens of 1024 columns in bf16 55.9 us (4.2 TB/s; 45.8 at
// the rate of a large copy), 36450 of 432 in fp32 28.3 (24.5); below some 1000 tokens the launch.
#include <algorithm>

#include "capi.hpp"
#include "common.hpp"

namespace clarus {

namespace {

constexpr int RO_T = 256;
constexpr int RO_TOKENS = 32;    // tokens of a workgroup, at most
constexpr int RO_FLIGHT = 4;     // tokens in flight per thread
constexpr int RO_AXES = CLARUS_ROTARY_AXES;
constexpr int RO_PAIRS = CLARUS_ROTARY_PAIRS;

enum : int { POS_GRID = 0, POS_F32 = 1, POS_I32 = 2, POS_I64 = 3 };

struct RotaryP {
  const void* x;
  void* out;
  const void* pos;
  int64_t xbs, ldx, pbs, ldp;
  int64_t total;       // tokens of all images
  unsigned l;          // tokens of an image
  int c, d, p;         // columns of a row, of a head; pairs
  int per_row, rpp;    // places of a row that this launch's workgroups take, rows per pass
  int units;           // places of a row in all
  int turned, whole;   // places of a head: turned, in all
  int tokens;          // of a workgroup
  int pos_kind, o_dt;
  unsigned grid[RO_AXES];
  double turn[RO_PAIRS];
  unsigned char axis[RO_PAIRS];
};

// V consecutive elements, V x the type's size aligned
template <int DT, int V>
__device__ __forceinline__ void ro_load(const void* p, float (&r)[V]) {
  if constexpr (V == 8) {
    const f32x8 t = load8<DT>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = t.v[i];
  } else if constexpr (DT == DT_BF16) {
    typedef __attribute__((ext_vector_type(V))) unsigned short T;
    const T t = *reinterpret_cast<const T*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = bf16_to_f32(t[i]);
  } else {
    typedef __attribute__((ext_vector_type(V))) float T;
    const T t = *reinterpret_cast<const T*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = t[i];
  }
}

template <int V>
__device__ __forceinline__ void ro_store(void* p, int dt, int64_t at, const float (&r)[V]) {
  if (dt == DT_BF16) {
    unsigned short* q = (unsigned short*)p + at;
    if constexpr (V == 8) *reinterpret_cast<u32x4*>(q) = u32x4{pack2_bf16(r[0], r[1]), pack2_bf16(r[2], r[3]), pack2_bf16(r[4], r[5]), pack2_bf16(r[6], r[7])};
    else if constexpr (V == 4) *reinterpret_cast<u32x2*>(q) = u32x2{pack2_bf16(r[0], r[1]), pack2_bf16(r[2], r[3])};
    else if constexpr (V == 2) *reinterpret_cast<unsigned*>(q) = pack2_bf16(r[0], r[1]);
    else *q = f32_to_bf16_bits(r[0]);
  } else {
    float* q = (float*)p + at;
    if constexpr (V == 8) {
      reinterpret_cast<f32x4*>(q)[0] = f32x4{r[0], r[1], r[2], r[3]};
      reinterpret_cast<f32x4*>(q)[1] = f32x4{r[4], r[5], r[6], r[7]};
    } else if constexpr (V == 4) *reinterpret_cast<f32x4*>(q) = f32x4{r[0], r[1], r[2], r[3]};
    else if constexpr (V == 2) *reinterpret_cast<f32x2*>(q) = f32x2{r[0], r[1]};
    else *q = r[0];
  }
}

__device__ __forceinline__ void ro_turn(float& a, float& b, float2 cs) {
  const float x = a, y = b;
  a = fmaf(x, cs.x, -(y * cs.y));
  b = fmaf(x, cs.y, y * cs.x);
}

// HALVES: pair j is columns (j, p + j), a place V pairs (two runs of V columns); else columns (2 j, 2 j + 1), a place
// V / 2 pairs (one run of V columns)
template <int DT, int V, bool HALVES>
__global__ void __launch_bounds__(RO_T) rotary_kernel(const RotaryP p) {
  extern __shared__ float2 cs[];  // [token][pair] cos, sin
  __shared__ int64_t from[RO_TOKENS];
  constexpr int ES = DT == DT_BF16 ? 2 : 4, NP = HALVES ? V : V / 2;
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int nt = (int)(p.total - t0 < p.tokens ? p.total - t0 : p.tokens);
  for (int i = tid; i < nt * p.p; i += RO_T) {
    const int t = i / p.p, j = i - t * p.p, ax = p.axis[j];
    const unsigned row = (unsigned)(t0 + t), n = row / p.l, at = row - n * p.l;
    double where;
    if (p.pos_kind == POS_GRID) {
      unsigned rest = at, mine = 0;
#pragma unroll
      for (int a = RO_AXES - 1; a >= 0; --a) {
        const unsigned q = rest / p.grid[a], m = rest - q * p.grid[a];
        if (a == ax) mine = m;
        rest = q;
      }
      where = mine;
    } else {
      const int64_t e = n * p.pbs + at * p.ldp + ax;
      where = p.pos_kind == POS_F32 ? (double)((const float*)p.pos)[e]
              : p.pos_kind == POS_I32 ? (double)((const int*)p.pos)[e] : (double)((const int64_t*)p.pos)[e];
    }
    const double turns = where * p.turn[j];
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = float2{c, s};
  }
  if (tid < nt) {
    const unsigned row = (unsigned)(t0 + tid), n = row / p.l;
    from[tid] = n * p.xbs + (int64_t)(row - n * p.l) * p.ldx;
  }
  __syncthreads();
  const int r0 = tid / p.per_row, place = blockIdx.y * p.per_row + tid - r0 * p.per_row;
  if (r0 >= p.rpp || place >= p.units) return;
  const int head = place / p.whole, u = place - head * p.whole;
  const bool turned = u < p.turned;
  const int run = HALVES ? (turned ? u * V : 2 * p.p + (u - p.turned) * V) : u * V;
  const int col = head * p.d + run, j0 = HALVES ? u * V : u * (V / 2);
  const unsigned char* xp = (const unsigned char*)p.x;
#pragma unroll 1
  for (int t = r0; t < nt; t += p.rpp * RO_FLIGHT) {
    float a[RO_FLIGHT][V], b[RO_FLIGHT][V];
#pragma unroll
    for (int f = 0; f < RO_FLIGHT; ++f) {
      const int at = t + f * p.rpp < nt ? t + f * p.rpp : t;
      const unsigned char* q = xp + (from[at] + col) * ES;
      ro_load<DT, V>(q, a[f]);
      if (HALVES && turned) ro_load<DT, V>(q + p.p * ES, b[f]);
    }
#pragma unroll
    for (int f = 0; f < RO_FLIGHT; ++f) {
      const int at = t + f * p.rpp;
      if (at >= nt) break;
      const int64_t to = (t0 + at) * p.c + col;
      if (turned) {
        const float2* w = cs + at * p.p + j0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float2 w1 = w[i];
          if constexpr (HALVES) ro_turn(a[f][i], b[f][i], w1);
          else ro_turn(a[f][2 * i], a[f][2 * i + 1], w1);
        }
        if constexpr (HALVES) ro_store<V>(p.out, p.o_dt, to + p.p, b[f]);
      }
      ro_store<V>(p.out, p.o_dt, to, a[f]);
    }
  }
}

template <int DT, int V, bool HALVES>
void ro_launch(const RotaryP& k, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((rotary_kernel<DT, V, HALVES>), grid, dim3(RO_T), (unsigned)(k.tokens * k.p * sizeof(float2)), st, k);
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" int clarus_hip_rotary(const ClarusRotaryArgs* a, void* stream) {
  clear_error();
  CLARUS_REQUIRE(a, "rotary: null arguments");
  CLARUS_REQUIRE(a->x && a->out, "rotary: null operand");
  const int64_t big = (int64_t)1 << 28;
  CLARUS_REQUIRE(a->n > 0 && a->l > 0 && a->heads > 0 && a->d > 0, "rotary: empty problem");
  CLARUS_REQUIRE(a->n < big && a->l < big && a->n * a->l < big, "rotary: fewer than 2^28 tokens");
  CLARUS_REQUIRE(a->d % 8 == 0 && a->d <= 2 * RO_PAIRS && a->heads < (1 << 20) && a->heads * a->d < (1 << 24),
                 "rotary: head width a multiple of 8 up to %d, rows below 2^24 columns", 2 * RO_PAIRS);
  CLARUS_REQUIRE(a->axes >= 1 && a->axes <= RO_AXES, "rotary: 1 to %d axes", RO_AXES);
  CLARUS_REQUIRE((a->dtype == DT_BF16 || a->dtype == DT_F32) && (a->o_dtype == DT_BF16 || a->o_dtype == DT_F32),
                 "rotary: bf16 or fp32");
  CLARUS_REQUIRE(a->pairs_mode == 0 || a->pairs_mode == 1, "rotary: pairs adjacent (0) or in halves (1)");
  CLARUS_REQUIRE(a->pos_kind >= POS_GRID && a->pos_kind <= POS_I64 && (a->pos_kind == POS_GRID || a->positions), "rotary: positions");
  const int64_t es = a->dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->x, 16) && aligned(a->out, 16) && a->ldx * es % 16 == 0 && a->x_bstride * es % 16 == 0,
                 "rotary: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldx >= 0 && a->x_bstride >= 0 && a->pos_bstride >= 0 && a->ldpos >= 0, "rotary: strides");
  const bool halves = a->pairs_mode == 1;
  RotaryP k{};
  int64_t cells = 1;
  for (int i = 0; i < RO_AXES; ++i) {
    k.grid[i] = 1;
    if (i < a->axes && a->pos_kind == POS_GRID) {
      CLARUS_REQUIRE(a->grid[i] > 0 && a->grid[i] <= a->l, "rotary: grid");
      k.grid[i] = (unsigned)a->grid[i];
      cells *= a->grid[i];
      CLARUS_REQUIRE(cells <= a->l, "rotary: grid");
    }
  }
  CLARUS_REQUIRE(a->pos_kind != POS_GRID || cells == a->l, "rotary: a grid of l tokens");
  int64_t p = 0;
  for (int i = 0; i < a->axes; ++i) {
    CLARUS_REQUIRE(a->sections[i] >= 0 && a->sections[i] <= RO_PAIRS, "rotary: sections");
    for (int64_t j = 0; j < a->sections[i] && p < RO_PAIRS; ++j) k.axis[p] = (unsigned char)i, k.turn[p] = a->turn[p], ++p;
  }
  int64_t sum = 0;
  for (int i = 0; i < a->axes; ++i) sum += a->sections[i];
  CLARUS_REQUIRE(sum >= 1 && 2 * sum <= a->d, "rotary: sections of 1 to d / 2 pairs in all");
  for (int i = 0; i < p; ++i) CLARUS_REQUIRE(a->turn[i] == a->turn[i] && a->turn[i] < 1e300 && a->turn[i] > -1e300, "rotary: turn %d", i);
  int v = 8;  // columns (halves: pairs) of a place
  while ((halves ? p : 2 * p) % v || a->d % v) v /= 2;
  if (halves)
    while ((a->d - 2 * p) % v) v /= 2;
  k.x = a->x; k.out = a->out; k.pos = a->positions;
  k.xbs = a->x_bstride; k.ldx = a->ldx; k.pbs = a->pos_bstride; k.ldp = a->ldpos;
  k.total = a->n * a->l; k.l = (unsigned)a->l;
  k.c = (int)(a->heads * a->d); k.d = (int)a->d; k.p = (int)p;
  k.turned = (int)(halves ? p / v : 2 * p / v);
  k.whole = (int)(k.turned + (a->d - 2 * p) / v);
  k.units = (int)(a->heads * k.whole);
  k.per_row = std::min(k.units, RO_T);
  k.rpp = RO_T / k.per_row;
  k.pos_kind = a->pos_kind; k.o_dt = a->o_dtype;
  const int64_t strips = cdiv(k.units, k.per_row);
  CLARUS_REQUIRE(strips < 65536, "rotary: too large");
  // as many tokens as make two passes of a workgroup, fewer while CUs idle (and, for 2^32 threads of a launch, more)
  int64_t tokens = std::min<int64_t>(RO_TOKENS, 2LL * RO_FLIGHT * k.rpp);
  if (k.total >= (1 << 22)) tokens = RO_TOKENS;
  while (tokens > k.rpp && cdiv(k.total, tokens) * strips < 4 * device_cus()) tokens = std::max<int64_t>(tokens / 2, k.rpp);
  k.tokens = (int)std::min<int64_t>(tokens, RO_TOKENS);
  const dim3 grid((unsigned)cdiv(k.total, k.tokens), (unsigned)strips);
  hipStream_t st = (hipStream_t)stream;
  note_kernel("rotary_kernel v=%d tokens=%d", v, k.tokens);
#define CLARUS_RO(DT)                                                              \
  do {                                                                             \
    if (halves) {                                                                  \
      if (v == 8) ro_launch<DT, 8, true>(k, grid, st);                             \
      else if (v == 4) ro_launch<DT, 4, true>(k, grid, st);                        \
      else if (v == 2) ro_launch<DT, 2, true>(k, grid, st);                        \
      else ro_launch<DT, 1, true>(k, grid, st);                                    \
    } else {                                                                       \
      if (v == 8) ro_launch<DT, 8, false>(k, grid, st);                            \
      else if (v == 4) ro_launch<DT, 4, false>(k, grid, st);                       \
      else ro_launch<DT, 2, false>(k, grid, st);                                   \
    }                                                                              \
  } while (0)
  if (a->dtype == DT_BF16) CLARUS_RO(DT_BF16);
  else CLARUS_RO(DT_F32);
#undef CLARUS_RO
  return check_launch("rotary");
}
