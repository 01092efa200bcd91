// Attention of one sequence of positions (pixels, or a few tokens) over the states of an encoder of
// another length, on gfx950:
//   o[q] = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  over the keys the mask keeps; 0 where it keeps none.
//
// One pass over the keys with the running maximum m and sum l of the softmax; no score is written to
// memory. A row is a query and one of the heads that share a kv head, so shared heads fill the tile of
// a single query. A wave holds 32 rows:
//   S^T = K Q^T       a lane of a 32 x 32 MFMA holds one row's scores of 16 keys: sums stay in the lane to
//                     the end, a maximum needs one exchange, with lane ^ 32
//   O^T = V^T P^T     P^T is the B operand as it is: lane l holds keys 8 (i / 4) + 4 (l / 32) + i % 4
//                     of each 16, and V^T is read in that order (bf16: transposing LDS reads; fp32: one
//                     float per lane), so P moves through no LDS
// K and V go from memory straight to LDS, 16 bytes a lane, without passing through registers.
//   xa_resident_kernel  up to XR_KEYS keys: all of them stay in LDS, rows stream by (few rows of wide fp32 heads: below)
//   xa_kernel           any number of keys: 128 or 256 rows (4 or 8 waves) per workgroup, tiles of 64 (fp32: 32)
//                       keys, the next one on its way during the current one's products
//   xa_join_kernel      joins the (O, m, l) of keys split over workgroups, where rows are few
//   xa_bits_kernel      a mask of pairs as bits
// m, l and O are fp32. bf16: products of bf16 q, k, v are exact in fp32; P is rounded once to bf16 for
// the product with V (at most half a step, 2^-8, of each weight, of independent signs: together about
// as much as the result's own rounding to bf16). fp32: every product runs on fp32 MFMAs.
// A masked or padding key's score is taken as -inf whatever its K holds; where no query keeps it (a mask of
// keys, the end of the keys) its V row is taken as 0.
//
// What bounds it (bf16, the GPU's time alone, without the call's).
//   Many rows and keys: the softmax's arithmetic and the matrix cores, which overlap in part. 14400 queries x 3600 keys, 8
//   heads of 64: 117 to 129 us by the card, 822 to 907 TFLOP/s (a large library product reaches 1190); 57600 x 3600, 4 heads of
//   128: 434 to 477 us, 890 to 979. In the first the VALU is busy for 70% of the cycles (an exponential counts twice), the
//   matrix cores for 44%, in the second for 43% and 45%, at clocks that the load lowers to 1.8 and 1.9 GHz.
//   A prompt (57600 x 77, 4 heads of 64): 12 us of reading q and writing o at the rate of a large copy; 18.3 us, a wave
//   loading, multiplying and weighing its few keys in turn: the VALU is busy for 55% of the cycles.
//   One query of 8 images x 30001 keys: reading K and V, 492 MB in 94 us, 5.2 TB/s (a large copy: 4.8 TB/s).
#include <algorithm>

#include "attention_tile.hpp"
#include "capi.hpp"

namespace clarus {

namespace {

constexpr int64_t XA_BITS_GRID = 1 << 20;  // workgroups of a bits launch, at most

// ---------------------------------------------------------------- few keys
// Up to XR_KEYS keys (a prompt): all keys of an (image, kv head) stay in a workgroup's LDS: copied once, one barrier,
// then its 8 waves take 32 rows each, chunk after chunk, the next chunk's queries in flight. Workgroups of the same rows
// and other heads run on one XCD, whose L2 then reads and writes each line of q and out once.
constexpr int XR_T = 512;
constexpr int XR_KEYS = 128;

template <int DT, int D, int C, int MASK>
__global__ void __launch_bounds__(XR_T, (DT == DT_BF16 ? D <= 64 : D <= 32) ? 4 : 2) xa_resident_kernel(const CrossP p) {
  using T = XaTile<DT, D>;
  constexpr int KT = T::KT, W = XR_T / 64, QN = xa_qn<DT, C>;
  extern __shared__ __attribute__((aligned(16))) unsigned char tiles[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hl = lane >> 5;
  const unsigned total = (unsigned)(p.nblk * p.nk), span = (total + 7) >> 3;
  const unsigned id = (blockIdx.x & 7) * span + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= span || id >= total) return;
  const int part = (int)(id / (unsigned)p.nk);
  const int nk = (int)(id - part * (unsigned)p.nk);
  const int n = nk / p.kv_heads, kvh = nk - n * p.kv_heads;
  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)kvh * p.d) * T::ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)kvh * p.d) * T::ES;
  const unsigned char* mkey = MASK == MASK_KEYS ? p.mask + n * p.mbs : nullptr;
  const int lk = (int)p.lk, ntile = (lk + KT - 1) / KT;

  // chunks of 32 rows: part `part` of nblk equal parts, wave after wave
  const int chunks = (int)((p.rows + 31) / 32), each = (int)((chunks + p.nblk - 1) / p.nblk);
  const int c1 = min((part + 1) * each, chunks);
  int ch = part * each + wave;
  auto at = [&](int c) __attribute__((always_inline)) {  // rows past the end repeat the last one
    const int64_t r = (int64_t)c * 32 + col;
    return xa_row(p, kvh, r < p.rows ? r : p.rows - 1);
  };
  constexpr bool ANEW = DT == DT_BF16 && MASK == MASK_PAIRS && C == 64;  // (57600 x 77, 4 heads of 64: 24.6 us, 25.2 kept)
  constexpr bool AHEAD = QN <= 8;  // the next chunk's queries in flight (where registers allow it)
  u32x4 qn[QN];
  if (AHEAD && ch < c1) xa_load_q<DT, C>(p, n, at(ch), hl, qn);
  constexpr int MT = XR_KEYS / KT;
  uint64_t kept[MT];  // the keys of each tile that count
  {
    int byte[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) byte[t] = t < ntile ? xa_key_byte<KT, MASK>(mkey, (int64_t)t * KT, lk, lane) : 0;
    const XaCopy<DT, D, W> copy(p, wave, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      kept[t] = __ballot(byte[t]);
      if (kept[t])
        copy(p, kp + (int64_t)t * KT * p.ldk * T::ES, vp + (int64_t)t * KT * p.ldv * T::ES, tiles + t * 2 * T::BYTES, kept[t]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies have landed
  barrier_keep_vm();
#pragma unroll 1
  for (; ch < c1; ch += W) {
    u32x4 qf[QN];
    const XaRow r = at(ch);
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < QN; ++i) qf[i] = qn[i];
      if (ch + W < c1) xa_load_q<DT, C>(p, n, at(ch + W), hl, qn);
    } else {
      xa_load_q<DT, C>(p, n, r, hl, qf);
    }
    const unsigned char* mrow = MASK == MASK_PAIRS ? p.mask + n * p.mbs + r.qi * p.mqs : nullptr;
    f32x16 o[D / 32];
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[b][j] = 0.f;
    float m = XA_FLOOR, l = 0.f;
    bool far = false, fresh = true;  // fresh: o is 0
    // 32 keys at a time (a row of 32 keys starts where the swizzles do), half of a tile in bf16
#pragma unroll 1
    for (int h = 0; h < lk; h += 32) {
      const unsigned char* ks = tiles + h / KT * 2 * T::BYTES + h % KT * T::ROWB;
      uint32_t bits = 0;
#pragma unroll
      for (int t = 0; t < MT; ++t)
        if (h / KT == t) bits = (unsigned)(kept[t] >> (h % KT));
      if constexpr (MASK == MASK_PAIRS) {  // a row's 32 bytes by its two lanes
        unsigned lo = xa_bits16(mrow + h + 16 * hl, lk - h - 16 * hl) << (16 * hl), hi = lo;
        swap32(lo, hi);
        bits = lo | hi;
        if (!__any(bits)) continue;
      } else if (!bits) {
        continue;
      }
      xa_tile<DT, D, C, MASK, 1, ANEW>(ks, ks + T::BYTES, qf, o, m, l, far, p.c, bits, bits == 0xffffffffu, fresh);
      fresh = false;
    }
    l = sum32(l);
    xa_store<D>(p, n, r, o, l, ch * 32ll + col < p.rows);
  }
}

// ---------------------------------------------------------------- keys streamed through LDS
// W waves of 32 rows. (MASK_PAIRS at 3 waves per SIMD: at 4 it spills. Of those at 4, two forms of masked keys in four waves keep
// a few registers in scratch: bf16 heads of 40 and 48 three, fp32 heads of 56 and 64 four.)
template <int DT, int D, int C, int MASK, int W>
__global__ void __launch_bounds__(64 * W, D <= 64 ? (MASK == MASK_PAIRS ? 3 : 4) : 2) xa_kernel(const CrossP p) {
  using T = XaTile<DT, D>;
  constexpr int KT = T::KT, KB = KT / 32, DB = D / 32;
  __shared__ __align__(16) unsigned char tiles[2][2 * T::BYTES];
  __shared__ uint64_t wants[MASK == MASK_PAIRS ? W : 1];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hl = lane >> 5;
  // row blocks and splits of one (image, kv head) run on one XCD, whose L2 then holds that head's K and V: eight
  // (image, kv head) pairs at a time, one on each XCD (padded batches stay balanced), the blocks of the last few
  // pairs dealt out in equal parts
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

  const int64_t wrow = (int64_t)rb * (32 * W) + wave * 32;  // the wave's first row
  const bool busy = wrow < p.rows;
  const int64_t row = wrow + col < p.rows ? wrow + col : p.rows - 1;  // rows past the end repeat the last one
  const XaRow r = xa_row(p, kvh, row);

  const unsigned char* kp = (const unsigned char*)p.k + (n * p.kbs + (int64_t)kvh * p.d) * T::ES;
  const unsigned char* vp = (const unsigned char*)p.v + (n * p.vbs + (int64_t)kvh * p.d) * T::ES;
  // MASK_PAIRS: a row's mask as bits, a word per tile
  using Word = std::conditional_t<KT == 64, uint64_t, uint32_t>;
  const Word* words = MASK == MASK_PAIRS ? (const Word*)(p.bits + n * p.bbs + r.qi * p.nw) + (int64_t)split * (p.split_len / KT) : nullptr;
  const unsigned char* mkey = MASK == MASK_KEYS ? p.mask + n * p.mbs : nullptr;

  const int64_t k0 = (int64_t)split * p.split_len, k1 = k0 + p.split_len < p.lk ? k0 + p.split_len : p.lk;
  const int ntile = (int)((k1 - k0 + KT - 1) / KT);

  const XaCopy<DT, D, W> copy(p, wave, lane);
  auto key_byte = [&](int t) __attribute__((always_inline)) {  // 0 for t < 0
    return t < 0 ? 0 : xa_key_byte<KT, MASK>(mkey, k0 + (int64_t)t * KT, k1, lane);
  };
  auto fill = [&](int t, uint64_t bits, int buf) __attribute__((always_inline)) {
    const int64_t base = k0 + (int64_t)t * KT;
    copy(p, kp + base * p.ldk * T::ES, vp + base * p.ldv * T::ES, tiles[buf], bits);
  };

  u32x4 qf[xa_qn<DT, C>];
  xa_load_q<DT, C>(p, n, r, hl, qf);
  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[b][j] = 0.f;
  float m = XA_FLOOR, l = 0.f;
  bool far = false;

  // 64 tiles at a time: the tiles of which the workgroup (want) and the wave (mine) keep a key, one bit each; the others
  // are neither copied nor waited for
#pragma unroll 1
  for (int c0 = 0; c0 < ntile; c0 += 64) {
    const int cn = ntile - c0 < 64 ? ntile - c0 : 64;
    uint64_t want = ~0ull >> (64 - cn), mine = want;
    if constexpr (MASK == MASK_KEYS) {
      want = __ballot(lane < cn && xa_any<KT>(mkey + k0 + (int64_t)(c0 + lane) * KT, k1 - k0 - (int64_t)(c0 + lane) * KT));
    } else if constexpr (MASK == MASK_PAIRS) {
      // lane (row, hl): 32 tiles' words of its row, 16 in flight
      mine = 0;
#pragma unroll 1
      for (int t0 = 0; t0 < 32 && t0 < cn; t0 += 16) {
        Word w[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const int tile = 32 * hl + t0 + t;
          w[t] = words[c0 + (tile < cn ? tile : 0)];
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const uint64_t any = __ballot(32 * hl + t0 + t < cn && w[t] != 0);
          mine |= (uint64_t)((unsigned)any != 0) << (t0 + t) | (uint64_t)((any >> 32) != 0) << (32 + t0 + t);
        }
      }
      if (!busy) mine = 0;
      __syncthreads();  // the words of the 64 tiles before have been read
      if (lane == 0) wants[wave] = mine;
      __syncthreads();
      want = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) want |= wants[w];
      want = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(want >> 32)) << 32 |
             (unsigned)__builtin_amdgcn_readfirstlane((unsigned)want);
    }
    auto pop = [&]() __attribute__((always_inline)) {  // the next wanted tile, -1 past the last
      if (!want) return -1;
      const int t = __builtin_ctzll(want);
      want &= want - 1;
      return c0 + t;
    };
    int t = pop(), t1 = pop();
    if (t < 0) continue;
    if (c0) barrier_keep_vm();  // the last tile of the 64 before has been read
    // the kept keys of a tile, one bit each; the bytes of the tile after the next are on their way
    uint64_t bits = __ballot(key_byte(t));
    int byte = key_byte(t1), buf = 0;
    fill(t, bits, 0);
    Word next = MASK == MASK_PAIRS ? words[t] : 0;
#pragma unroll 1
    while (t >= 0) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies of tile t have landed
      barrier_keep_vm();                   // everybody's have, and the tile before has been read
      const uint64_t now = MASK == MASK_PAIRS ? (uint64_t)next : bits;
      const int t2 = pop();
      if (t1 >= 0) {
        bits = __ballot(byte);
        byte = key_byte(t2);
        fill(t1, bits, buf ^ 1);
        if constexpr (MASK == MASK_PAIRS) next = words[t1];
      }
      if (busy && (MASK != MASK_PAIRS || (mine >> (t - c0) & 1)))
        xa_tile<DT, D, C, MASK, KB, false>(tiles[buf], tiles[buf] + T::BYTES, qf, o, m, l, far, p.c, now, now == T::ALL, false);
      t = t1;
      t1 = t2;
      buf ^= 1;
    }
  }
  if (!busy) return;
  l = sum32(l);
  if (p.splits == 1) {
    xa_store<D>(p, n, r, o, l, wrow + col < p.rows);
    return;
  }
  if (wrow + col >= p.rows) return;
  const int64_t at = ((int64_t)split * p.nk + nk) * p.rows + row, all = (int64_t)p.splits * p.nk * p.rows;
  float* po = p.part + at * D;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int j4 = 0; j4 < 4; ++j4)
      *reinterpret_cast<f32x4*>(po + 32 * b + 8 * j4 + 4 * hl) = f32x4{o[b][4 * j4], o[b][4 * j4 + 1], o[b][4 * j4 + 2], o[b][4 * j4 + 3]};
  if (hl == 0) *reinterpret_cast<float2*>(p.part + all * D + 2 * at) = float2{m, l};
}

// MASK_PAIRS: the mask's bytes as bits, 64 keys a word, zeros behind the last key: read once for all heads, and an eighth
// of the bytes for the kernels' gathers. A thread makes 16 bits. first: what the launches before have made
__global__ void __launch_bounds__(XA_T) xa_bits_kernel(const unsigned char* mask, int64_t mbs, int64_t mqs, int64_t lq, int64_t lk,
                                                       int64_t nw, int64_t first, int64_t total, unsigned short* out) {
  const int64_t i = first + (int64_t)blockIdx.x * XA_T + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / (4 * nw), w = i - row * 4 * nw, n = row / lq, key = 16 * w;
  out[i] = key < lk ? (unsigned short)xa_bits16(mask + n * mbs + (row - n * lq) * mqs + key, lk - key) : 0;
}

int xa_pad(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

// Into how many parts the keys are split: as many as make the time of a part's tiles in a row and, with more than one
// part, of writing and joining the parts least, and less than most_of the time in one; at most two workgroups per CU. The
// constants are measured (us): a tile 0.73 / 0.96 / 1.4 with heads of 32 / 64 / 128, fp32 1.2 / 2.25 / 4.3; a second
// workgroup on a CU adds a quarter of that, in fp32, where the matrix core is the bound, 0.8; parts 2.8 and, a MB of one
// part, 0.56 + 0.3 for each. What it
// decides, in one / the chosen / more parts (us, bf16): one query, 8 heads of 64, 400 keys 9.6 / 7.6 (7); 8 x 256 queries,
// 8 heads of 40, 400 keys 11.2 / - / 15.8 (2), 1600 keys 30.7 / 21.8 (4); 900 queries, 8 heads of 64, 800 keys 16.3 / 14.7
// (4); 2 x 3600 queries, 4 heads of 64, 1000 keys 18.7 / - / 28.0 (2). One query of 8 images, 16 heads on 4 of 128, 30001
// keys: 119 in 8 parts, 94 in 16 (two workgroups per CU), 107 in 24
int64_t xa_splits(int32_t dt, int64_t blocks, int64_t rows, int64_t tiles, int D, double most_of) {
  const int64_t cus = device_cus(), most = std::min(tiles, std::max<int64_t>(2 * cus / blocks, 1));
  const double tile = dt == DT_BF16 ? 0.5 + 0.0072 * D : 0.2 + 0.032 * D, share = dt == DT_BF16 ? 0.25 : 0.8;
  const double mb = 1e-6 * (double)rows * (D + 2) * sizeof(float);
  int64_t best = 1;
  double least = 1e30, whole = 0.0;
  for (int64_t s = 1; s <= most; ++s) {
    const double t = cdiv(tiles, s) * tile * (1 + share * (cdiv(blocks * s, cus) - 1)) + (s > 1 ? 2.8 + mb * (0.56 + 0.3 * s) : 0.0);
    if (s == 1) whole = t;
    if (t < least && (s == 1 || t < most_of * whole)) least = t, best = s;
  }
  return best;
}

// Waves of a workgroup: eight (bf16, heads up to 64, no mask of pairs) fill half the tiles for the same rows, 0.9 of the
// time per row, where there are more of them than CUs; but rows are dealt out in twos as large, so the fuller CU counts
// (us in four / eight: 14400 x 3600, 8 heads of 64 142 / 126; 57600 x 1000, 4 heads of 64 82 / 76; 10000 x 2000, 8 heads of
// 64, 632 / 320 workgroups, 59 / 62; 5000 x 2000, 8 heads of 64, 320 / 160 workgroups, 40 / 44; fp32 and wider heads within
// 2% or slower in eight; masks of pairs from 0.85 to 1.06 of the time)
int xa_waves(int32_t dt, int64_t rows, int64_t nk, int D, int mask) {
  if (dt != DT_BF16 || D > 64 || mask == MASK_PAIRS) return 4;
  const int64_t cus = device_cus(), four = cdiv(rows, 128) * nk, eight = cdiv(rows, 256) * nk;
  return eight > cus && 9 * 2 * cdiv(eight, cus) < 10 * cdiv(four, cus) ? 8 : 4;
}

struct XaPlan {
  bool resident;
  int64_t nblk, split_len;  // row blocks (resident: workgroups) of an (image, kv head); keys of a split
  int splits, waves;        // waves of a workgroup of xa_kernel
  size_t bits, part;        // workspace bytes: the mask's words, the splits' parts
};

XaPlan xa_plan(int32_t dt, int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t d, int mask) {
  XaPlan g{};
  const int kt = dt == DT_BF16 ? 64 : 32, D = xa_pad(d);
  const int64_t rows = lq * (heads / kv_heads), nk = n * kv_heads;
  // keys that fit LDS are split only where it takes a third off the modelled time, which knows no masks: few rows of wide fp32
  // heads (4 x 1 queries, 8 heads on 2 of 128, 128 keys 19.8 us / 10.9 split; 71 queries 16.0 / 13.4; 225 queries, 16 heads of
  // 80, not split, 12.4 / 13.7)
  if (lk <= XR_KEYS && xa_splits(dt, cdiv(rows, 128) * nk, nk * rows, cdiv(lk, kt), D, 0.7) == 1) {
    g.resident = true;
    g.splits = 1;
    g.split_len = lk;
    const int64_t want = cdiv((D <= 64 ? 2LL : 1LL) * device_cus(), nk), most = cdiv(rows, 32 * (XR_T / 64));
    // few rows: one chunk of 32 per workgroup while there are CUs, so that no two waves share a SIMD (900 queries, 8 heads of
    // 64: 4.8 us, 6.0 with eight chunks per workgroup, fp32 10.0 and 17.4)
    g.nblk = std::max(std::min(want, most), std::min(cdiv(rows, 32), device_cus() / nk));
    return g;
  }
  g.waves = xa_waves(dt, rows, nk, D, mask);
  g.nblk = cdiv(rows, 32 * g.waves);
  const int64_t blocks = g.nblk * nk;
  g.split_len = cdiv(cdiv(lk, xa_splits(dt, blocks, nk * rows, cdiv(lk, kt), D, 1.0)), kt) * kt;
  g.splits = (int)cdiv(lk, g.split_len);
  if (mask == MASK_PAIRS) g.bits = (size_t)(n * lq * cdiv(lk, 64) + 1) / 2 * 16;
  if (g.splits > 1) g.part = (size_t)g.splits * nk * rows * (D + 2) * sizeof(float);
  return g;
}

// What 32-bit counts and a launch of fewer than 2^32 threads (two for each of n * heads * lq rows) hold. Each size on its own
// first, so that no product wraps
bool xa_fits(int64_t n, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int mask) {
  const int64_t big = (int64_t)1 << 31;
  return n < 65536 && kv_heads < 65536 && n * kv_heads < 65536 && heads < big && lq < big && lk < big &&
         lq * (heads / kv_heads) < big && n * kv_heads * (lq * (heads / kv_heads)) < big &&
         (mask != MASK_PAIRS || n * lq < ((int64_t)1 << 38) / lk);
}

template <int DT, int D, int C>
void xa_launch(const CrossP& k, bool resident, int waves, int mask, hipStream_t st) {
  const dim3 grid((unsigned)(8 * ((k.nblk * k.nk * k.splits + 7) / 8)));
  if (resident) {
    using T = XaTile<DT, D>;
    const unsigned lds = (unsigned)(cdiv(k.lk, T::KT) * 2 * T::BYTES);
    if (mask == MASK_NONE) hipLaunchKernelGGL((xa_resident_kernel<DT, D, C, MASK_NONE>), grid, dim3(XR_T), lds, st, k);
    else if (mask == MASK_KEYS) hipLaunchKernelGGL((xa_resident_kernel<DT, D, C, MASK_KEYS>), grid, dim3(XR_T), lds, st, k);
    else hipLaunchKernelGGL((xa_resident_kernel<DT, D, C, MASK_PAIRS>), grid, dim3(XR_T), lds, st, k);
    return;
  }
  if constexpr (DT == DT_BF16 && D <= 64) {
    if (waves == 8) {
      if (mask == MASK_NONE) hipLaunchKernelGGL((xa_kernel<DT, D, C, MASK_NONE, 8>), grid, dim3(512), 0, st, k);
      else hipLaunchKernelGGL((xa_kernel<DT, D, C, MASK_KEYS, 8>), grid, dim3(512), 0, st, k);
      return;  // not split
    }
  }
  if (mask == MASK_NONE) hipLaunchKernelGGL((xa_kernel<DT, D, C, MASK_NONE, 4>), grid, dim3(256), 0, st, k);
  else if (mask == MASK_KEYS) hipLaunchKernelGGL((xa_kernel<DT, D, C, MASK_KEYS, 4>), grid, dim3(256), 0, st, k);
  else hipLaunchKernelGGL((xa_kernel<DT, D, C, MASK_PAIRS, 4>), grid, dim3(256), 0, st, k);
  if (k.splits > 1) {
    constexpr int TPR = D <= 32 ? 8 : D <= 64 ? 16 : 32;
    int gs = 1;
    while (gs * TPR < XA_T && gs * XJ_BATCH < k.splits) gs *= 2;
    hipLaunchKernelGGL((xa_join_kernel<D>), dim3((unsigned)cdiv(k.rows * k.nk, XA_T / (TPR * gs))), dim3(XA_T), 0, st, k, gs);
  }
}

}  // namespace

}  // namespace clarus

using namespace clarus;

extern "C" size_t clarus_hip_cross_attention_workspace(int32_t dtype, int64_t n, int64_t lq, int64_t lk, int64_t heads,
                                                       int64_t kv_heads, int64_t d, int32_t mask_mode) {
  if (n <= 0 || lq <= 0 || lk <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || d <= 0 || d > 128 ||
      !xa_fits(n, lq, lk, heads, kv_heads, mask_mode))
    return 0;
  const XaPlan g = xa_plan(dtype, n, lq, lk, heads, kv_heads, d, mask_mode);
  return g.bits + g.part;
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
  CLARUS_REQUIRE(a->scale > 0.f && a->scale < 2e38f, "cross_attention: scale positive and below 2e38");
  const int64_t es = a->dtype == DT_BF16 ? 2 : 4;
  CLARUS_REQUIRE(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && a->ldq * es % 16 == 0 &&
                     a->ldk * es % 16 == 0 && a->ldv * es % 16 == 0 && a->q_bstride * es % 16 == 0 &&
                     a->k_bstride * es % 16 == 0 && a->v_bstride * es % 16 == 0,
                 "cross_attention: 16-byte aligned rows");
  CLARUS_REQUIRE(a->ldk < (1 << 24) && a->ldv < (1 << 24), "cross_attention: rows of k and v less than 2^24 elements apart");
  CLARUS_REQUIRE(a->ldq >= 0 && a->ldk >= 0 && a->ldv >= 0 && a->q_bstride >= 0 && a->k_bstride >= 0 && a->v_bstride >= 0,
                 "cross_attention: strides");
  CLARUS_REQUIRE(a->mask_mode >= MASK_NONE && a->mask_mode <= MASK_PAIRS && (a->mask_mode == MASK_NONE || a->mask) &&
                     a->mask_bstride >= 0 && a->mask_qstride >= 0,
                 "cross_attention: mask");
  CLARUS_REQUIRE(xa_fits(a->n, a->lq, a->lk, a->heads, a->kv_heads, a->mask_mode), "cross_attention: too large");
  const XaPlan g = xa_plan(a->dtype, a->n, a->lq, a->lk, a->heads, a->kv_heads, a->d, a->mask_mode);
  CLARUS_REQUIRE(8 * ((g.nblk * a->n * a->kv_heads * g.splits + 7) / 8) < ((int64_t)1 << 32) / (g.resident ? XR_T : 64 * g.waves),
                 "cross_attention: too large");  // rows that fill few of their workgroups
  const size_t need = g.bits + g.part;
  CLARUS_REQUIRE(need == 0 || (scratch && aligned(scratch, 16) && scratch_bytes >= need),
                 "cross_attention: scratch %zu < %zu bytes", scratch_bytes, need);
  CrossP k{};
  k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out; k.mask = (const unsigned char*)a->mask; k.part = (float*)((char*)scratch + g.bits);
  k.qbs = a->q_bstride; k.ldq = a->ldq; k.kbs = a->k_bstride; k.ldk = a->ldk; k.vbs = a->v_bstride; k.ldv = a->ldv;
  k.mbs = a->mask_bstride; k.mqs = a->mask_qstride;
  k.rep = (int)(a->heads / a->kv_heads); k.kv_heads = (int)a->kv_heads; k.d = (int)a->d; k.lq = (int)a->lq;
  k.rows = a->lq * k.rep; k.lk = a->lk; k.nk = a->n * a->kv_heads;
  k.nblk = g.nblk; k.split_len = g.split_len; k.splits = g.splits;
  k.o_dt = a->o_dtype;
  k.c = a->scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  if (g.bits) {
    // images or queries that share one mask row (stride 0) share its words
    const int64_t nw = cdiv(a->lk, 64), lq = a->mask_qstride ? a->lq : 1, total = (a->mask_bstride ? a->n : 1) * lq * 4 * nw;
    k.bits = (const uint64_t*)scratch;
    k.nw = a->mask_qstride ? nw : 0;
    k.bbs = a->mask_bstride ? lq * nw : 0;
    for (int64_t first = 0; first < total; first += XA_BITS_GRID * XA_T)
      hipLaunchKernelGGL(xa_bits_kernel, dim3((unsigned)std::min(cdiv(total - first, XA_T), XA_BITS_GRID)), dim3(XA_T), 0, st,
                         k.mask, a->mask_bstride, a->mask_qstride, lq, a->lk, nw, first, total, (unsigned short*)scratch);
    if (const int rc = check_launch("cross_attention")) return rc;
  }
  const int D = xa_pad(a->d);
  note_kernel("%s d=%d waves=%d splits=%d", g.resident ? "xa_resident_kernel" : "xa_kernel", D, g.resident ? XR_T / 64 : g.waves, g.splits);
  // V's columns come in blocks of 32, the columns that a score sums over in sixteens (14400 x 3600, 8 heads of 40: 113 us over
  // 48 columns, 121 over 64, fp32 807 and 894; 14400 x 2000, 4 heads of 80 54 / 57, of 104 67 / 69, fp32 347 / 377, 459 / 493)
#define CLARUS_XA(DT)                                        \
  do {                                                       \
    if (D == 32) xa_launch<DT, 32, 32>(k, g.resident, g.waves, a->mask_mode, st);           \
    else if (a->d <= 48) xa_launch<DT, 64, 48>(k, g.resident, g.waves, a->mask_mode, st);   \
    else if (D == 64) xa_launch<DT, 64, 64>(k, g.resident, g.waves, a->mask_mode, st);      \
    else if (a->d <= 80) xa_launch<DT, 96, 80>(k, g.resident, g.waves, a->mask_mode, st);   \
    else if (D == 96) xa_launch<DT, 96, 96>(k, g.resident, g.waves, a->mask_mode, st);      \
    else if (a->d <= 112) xa_launch<DT, 128, 112>(k, g.resident, g.waves, a->mask_mode, st); \
    else xa_launch<DT, 128, 128>(k, g.resident, g.waves, a->mask_mode, st);                 \
  } while (0)
  if (a->dtype == DT_BF16) CLARUS_XA(DT_BF16);
  else CLARUS_XA(DT_F32);
#undef CLARUS_XA
  return check_launch("cross_attention");
}
