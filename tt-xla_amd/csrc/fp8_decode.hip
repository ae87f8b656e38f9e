// Decode attention over the 8-bit cache: entry points, and the choice of blocks for its sparse form.
//
// Sparse form.  For every (user, KV head) the blocks of the context are scored by what their key bounds allow,
//   score(block) = max over the group's heads of  sum_d  max(q_d, 0) high_d + min(q_d, 0) low_d,
// an upper bound of q . k over the block's keys as they were written (their rounding to e4m3 may pass it by a little); the block that holds the newest token, the first block and the best of the others are
// attended, `kept` in all, of equal scores the lower column.  A choice flips with the last bit of a score, so scores are
// sums in 64 bits: products of bfloat16 values are exact there and a sum of 512 of them keeps 28 bits to spare, so that neither
// the order of the sum nor its split matters in practice.  But 64-bit sums for all blocks took 13 and 21 us (27 000 blocks with four heads, 46 000
// with eight), three times what reading the bounds takes, and hardly any of them decides anything.  So:
//   block_scores_kernel   scores by the matrix pipe, in 32 bits, and with them the sums of the products' magnitudes, which bound their
//                         error.  Memory bound: a block's bounds are 4 D bytes, read once.
//   choose_blocks_kernel  one workgroup per (user, KV head): finds the last score that is kept, T (a histogram over the scores' range, ranks inside the bin
//                         T lies in).  With scores at most e from the true ones, what is more than 2 e above T is kept and what is more
//                         than 2 e below is not; the few blocks between (about one in practice) are scored again in 64 bits and
//                         the best of them kept.  The columns come out in order, as a page table of their own.
// The attention is the decode kernel on that table: each (user, KV head) is a user with one KV head, its blocks the slabs of the cache.
#include "fp8_decode_kernel.h"

#include <algorithm>
#include <cstdlib>
#include <cstring>

namespace ttpa {
namespace fp8 {
int check_cache(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table, int kv_heads,
                int head_size, int block_size, int table_width, int num_blocks);
}
namespace decode {

bool launch_fp8_d64(const void *args, hipStream_t st);
bool launch_fp8_d128(const void *args, hipStream_t st);
bool launch_fp8_d256(const void *args, hipStream_t st);

namespace {

// ---- scores ----------------------------------------------------------------------------------------
using fp8::u32x4;
struct ScoreArgs {
  const uint16_t *q;
  int64_t q_us, q_hs;
  const uint16_t *bounds;
  const int32_t *pt;
  int64_t pt_rs;
  const void *cur;
  int cur_i64;
  int users, hkv, g, bs, w, nb, kept;
  int64_t row;     // elements of a row of the next two
  float2 *scores;  // [users * hkv][row]: score in 32 bits, sum of its products' magnitudes
  uint64_t *keys;  // [users * hkv][row]: exact scores, where too many are in question for LDS
  int32_t *table;  // [users * hkv][kept]
  int32_t *pos;    // [users * hkv]
  int32_t *columns;  // [users, hkv, kept], the caller's
  int *arrived;      // [users * hkv], zeroed for the attention
};

// Blocks of a user's context; 0 for a padded row.
__device__ __forceinline__ int blocks_of(const ScoreArgs &a, int u, int64_t &pos) {
  pos = load_index(a.cur, a.cur_i64, u);
  const int64_t cap = (int64_t)a.w * a.bs;
  if (pos >= cap) pos = cap - 1;
  return pos < 0 ? 0 : (int)(pos / a.bs) + 1;
}

constexpr uint64_t kUnbounded = ~0ull;
// Whole numbers in the order of the scores; what is no number, or no finite one above, comes first.
__device__ __forceinline__ uint64_t score_key(double s) {
  if (!(s < (double)INFINITY)) return kUnbounded;
  const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
  return (b >> 63) ? ~b : b | (1ull << 63);
}

template <int CTRL>
__device__ __forceinline__ double dpp_move_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A wavefront scores 16 blocks at a time: A = 16 rows of bounds x 32 features (lane n: block n), B = the heads' queries, positive parts against
// highs, negative ones against lows.
template <int D>
constexpr int score_tiles() {
  return D == 64 ? 2 : 1;
}
template <int D>
__global__ __launch_bounds__(256) void block_scores_kernel(ScoreArgs a) {
  constexpr int KSTEPS = D / 32, TILES = score_tiles<D>();
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int seg = blockIdx.x, u = seg / a.hkv, h = seg - u * a.hkv;
  int c0 = ((int)blockIdx.y * 4 + wave) * 16 * TILES;
  // (the table row is as wide for every user: a page that the context does not reach is looked up, too, and goes no further)
  int page[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) page[t] = a.pt[u * a.pt_rs + min(c0 + 16 * t + n, a.w - 1)];
  u32x4 q[KSTEPS];
  const uint32_t head = n < a.g ? 0xffffffffu : 0u;
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) {
    q[s] = *reinterpret_cast<const u32x4 *>(a.q + u * a.q_us + (int64_t)(h * a.g + min(n, a.g - 1)) * a.q_hs + 32 * s + 8 * quad);
#pragma unroll
    for (int i = 0; i < 4; ++i) q[s][i] &= head;
  }
  int64_t pos;
  const int nblk = blocks_of(a, u, pos);
  if (nblk <= a.kept || c0 >= nblk) return;  // (up to `kept` blocks: all are attended)
#pragma unroll 1
  for (;;) {
    u32x4 low[TILES][KSTEPS], high[TILES][KSTEPS];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int64_t slab = (int64_t)((unsigned)page[t] < (unsigned)a.nb ? page[t] : 0) * a.hkv + h;
      const uint16_t *b = a.bounds + slab * (2 * D) + 8 * quad;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) low[t][s] = *reinterpret_cast<const u32x4 *>(b + 32 * s);
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) high[t][s] = *reinterpret_cast<const u32x4 *>(b + D + 32 * s);
    }
    floatx4 sum[TILES], size[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) sum[t] = size[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      // the parts of the queries; a NaN stays one in both (it counts as positive and as negative)
      u32x4 plus, minus, less;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = q[s][i];
        const uint32_t lo_nan = (w & 0x7fffu) > 0x7f80u ? 0xffffu : 0u, hi_nan = (w & 0x7fff0000u) > 0x7f800000u ? 0xffff0000u : 0u;
        const uint32_t negative = ((w >> 15) & 0x00010001u) * 0xffffu;
        plus[i] = w & (~negative | lo_nan | hi_nan), minus[i] = w & (negative | lo_nan | hi_nan), less[i] = minus[i] & 0x7fff7fffu;
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        u32x4 low_size, high_size;
#pragma unroll
        for (int i = 0; i < 4; ++i) low_size[i] = low[t][s][i] & 0x7fff7fffu, high_size[i] = high[t][s][i] & 0x7fff7fffu;
        sum[t] = mma16<false>(high[t][s], plus, sum[t]);
        size[t] = mma16<false>(high_size, plus, size[t]);
        sum[t] = mma16<false>(low[t][s], minus, sum[t]);
        size[t] = mma16<false>(low_size, less, size[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      // lane (head n, quad) holds blocks 4 quad + r: the largest over the heads; a sum that is no number is as good as infinite
      float best[4], most[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        best[r] = row16_max(n < a.g ? (sum[t][r] == sum[t][r] ? sum[t][r] : INFINITY) : -INFINITY);
        most[r] = row16_max(n < a.g ? (size[t][r] == size[t][r] ? size[t][r] : INFINITY) : 0.f);
      }
      const int c = c0 + 16 * t + 4 * quad + n;
      if (n < 4 && c < nblk)
        a.scores[seg * a.row + c] = make_float2(n == 0 ? best[0] : n == 1 ? best[1] : n == 2 ? best[2] : best[3],
                                                       n == 0 ? most[0] : n == 1 ? most[1] : n == 2 ? most[2] : most[3]);
    }
    c0 += (int)gridDim.y * 64 * TILES;
    if (c0 >= nblk) return;
#pragma unroll
    for (int t = 0; t < TILES; ++t) page[t] = a.pt[u * a.pt_rs + min(c0 + 16 * t + n, a.w - 1)];
  }
}

// ---- choice ----------------------------------------------------------------------------------------
constexpr int kBins = 1024, kRanked = 256;

__device__ __forceinline__ uint32_t wave_max(uint32_t v) { return wave_max_u32(v); }
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, m);
    v = v > o ? v : o;
  }
  return v;
}

// Whole numbers in the order of 32-bit scores.
__device__ __forceinline__ uint32_t float_key(float s) {
  const uint32_t b = __builtin_bit_cast(uint32_t, s + 0.f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}

struct Choice {
  uint64_t threshold;  // keys above it are kept, and of those equal to it the first `ties`
  int ties;
};
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kHeld = 4, kLdsColumns = 8192;
struct ChoiceLds {
  uint32_t bins[kBins];
  uint64_t cand[kRanked], high[kWaves], low[kWaves];
  int num[kHeld][kWaves], column[kRanked], bin, over, count, next;
  float size[kWaves];
  uint8_t kept[kRanked];
};
// This thread's places in the first `used` of N running counts over the workgroup, and the counts of all.  (Between two calls lies a barrier.)
template <int N>
struct Counts {
  int before[N], all[N];
};
template <int N>
__device__ __forceinline__ Counts<N> running_counts(ChoiceLds &s, const int (&x)[N], int used = N) {
  static_assert(N <= kHeld, "");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Counts<N> c;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c.before[i] = c.all[i] = 0;
    if (i < used) {
      const int upto = wave_prefix_sum(x[i]);
      if (lane == 63) s.num[i][wave] = upto;
      c.before[i] = upto - x[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < used)
      for (int w = 0; w < kWaves; ++w) {
        const int n = s.num[i][w];
        if (w < wave) c.before[i] += n;
        c.all[i] += n;
      }
  return c;
}

__device__ __forceinline__ void clear_bins(ChoiceLds &s) {
#pragma unroll
  for (int j = 0; j < kBins / kThreads; ++j) s.bins[threadIdx.x + j * kThreads] = 0;
  if (threadIdx.x == 0) s.next = 0;
}
// The largest and the least of the workgroup's keys, and the largest of `size`; also in front of whatever the bins are used for.
template <typename Key>
__device__ __forceinline__ void extent(ChoiceLds &s, Key &hi, Key &lo, float &size) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  hi = wave_max(hi), lo = ~wave_max((Key)~lo);
  // (magnitudes: their order is that of their bits)
  size = __builtin_bit_cast(float, wave_max_u32(__builtin_bit_cast(uint32_t, size)));
  if (lane == 0) s.high[wave] = hi, s.low[wave] = lo, s.size[wave] = size;
  clear_bins(s);
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) hi = max(hi, (Key)s.high[w]), lo = min(lo, (Key)s.low[w]), size = fmaxf(size, s.size[w]);
}

// Where the `need` largest of the keys between lo and hi end; all threads.  visit(f) calls f for every key that the thread has.  A
// histogram over the keys' range finds the bin; the keys in it are ranked, or its range is the next histogram's.  The bins come cleared.
template <typename Key, typename Visit>
__device__ __forceinline__ Choice last_kept(ChoiceLds &s, int need, Key hi, Key lo, const Visit &visit) {
  constexpr int OWN = kBins / kThreads;
  const int tid = threadIdx.x;
#pragma unroll 1
  for (;;) {
    if (need == 0) return {hi, 0};
    if (lo == hi) return {lo, need};
    const int shift = max(0, 64 - __builtin_clzll((uint64_t)(hi - lo)) - 10);  // (hi - lo) >> shift < 1024
    visit([&](Key k) {
      if (k >= lo && k <= hi) atomicAdd(&s.bins[(k - lo) >> shift], 1u);
    });
    __syncthreads();
    // the bin, from the top, where the count reaches `need`: each thread owns neighbouring bins
    const int base = kBins - OWN * (tid + 1);
    int mine[OWN], sum = 0;
#pragma unroll
    for (int j = 0; j < OWN; ++j) mine[j] = (int)s.bins[base + j], sum += mine[j];
    int above = running_counts<1>(s, {sum}).before[0];
    if (above < need && above + sum >= need) {  // one thread
      int b = OWN - 1;
      while (above + mine[b] < need) above += mine[b], --b;
      s.bin = base + b, s.over = above, s.count = mine[b];
    }
    __syncthreads();
    const int count = s.count;
    need -= s.over;
    const Key span = ((Key)1 << shift) - 1;
    lo += (Key)s.bin << shift;
    hi = hi - lo < span ? hi : lo + span;  // (the last bin may reach past the largest number)
    if (shift == 0) return {lo, need};     // all of the bin are alike
    if (count <= kRanked) {
      visit([&](Key k) {
        if (k >= lo && k <= hi) s.cand[atomicAdd(&s.next, 1)] = k;
      });
      __syncthreads();
      if (tid < count) {
        // the need-th largest: fewer than `need` keys are larger, and with its equals there are enough
        const uint64_t k = s.cand[tid];
        int larger = 0, equal = 0;
#pragma unroll 1
        for (int i = 0; i < count; ++i) larger += s.cand[i] > k, equal += s.cand[i] == k;
        if (larger < need && larger + equal >= need) s.high[0] = k, s.over = need - larger;  // (equal keys write the same)
      }
      __syncthreads();
      return {s.high[0], s.over};
    }
    clear_bins(s);
    __syncthreads();
  }
}

// The exact score in 64 bits of one head's query over one page's bounds, as a key: D / 4 lanes, each with a page and a head of their own per such group.
template <int D>
__device__ __forceinline__ uint64_t exact_key(const ScoreArgs &a, int u, int h, int g, int page) {
  constexpr int LPB = D / 4;
  const int in_block = (int)(threadIdx.x & 63) % LPB;
  const bool high = in_block >= LPB / 2;
  const int f = 8 * (in_block % (LPB / 2));
  const int64_t slab = (int64_t)((unsigned)page < (unsigned)a.nb ? page : 0) * a.hkv + h;
  const u32x4 raw = *reinterpret_cast<const u32x4 *>(a.bounds + slab * (2 * D) + (high ? D : 0) + f);
  const u32x4 t = *reinterpret_cast<const u32x4 *>(a.q + u * a.q_us + (int64_t)(h * a.g + g) * a.q_hs + f);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v0 = bf16_lo(t[i]), v1 = bf16_hi(t[i]);
    // (a NaN stays one in both parts)
    const double q0 = high ? (v0 < 0.f ? 0.f : v0) : (v0 > 0.f ? 0.f : v0), q1 = high ? (v1 < 0.f ? 0.f : v1) : (v1 > 0.f ? 0.f : v1);
    s = __builtin_fma(q0, (double)bf16_lo(raw[i]), s);
    s = __builtin_fma(q1, (double)bf16_hi(raw[i]), s);
  }
  s += dpp_move_f64<kDppXor1>(s);
  s += dpp_move_f64<kDppXor2>(s);
  s += dpp_move_f64<kDppHalfMirror>(s);
  s += dpp_move_f64<kDppMirror>(s);
  if constexpr (LPB >= 32) s += __shfl_xor(s, 16);
  if constexpr (LPB >= 64) s += __shfl_xor(s, 32);
  return score_key(s);
}

// The choice among the blocks but the first and the last of a context of nblk > kept, each handed to `emit`.  HELD: contexts of up to kHeld blocks
// per thread, whose scores and pages every thread has in registers (column tid + kThreads j; x0, id0: those of the first); the scores of longer ones lie in LDS,
// where the table has up to kLdsColumns, or stay where they are, and each thread has neighbouring columns.
template <int D, bool HELD, typename Emit>
__device__ __forceinline__ void choose_among(const ScoreArgs &a, ChoiceLds &s, float *s_score, int seg, int u, int h, int nblk, float2 x0, int id0,
                                             const Emit &emit) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t *pt = a.pt + u * a.pt_rs;
  const float2 *scores = a.scores + seg * a.row;
  const int held = HELD ? (nblk + kThreads - 1) / kThreads : 0;  // of the registers
  float2 x[HELD ? kHeld : 1];
  int id[HELD ? kHeld : 1];
  if constexpr (HELD) {
    x[0] = x0, id[0] = id0;
#pragma unroll
    for (int j = 1; j < kHeld; ++j)
      if (j < held) x[j] = scores[min(tid + kThreads * j, nblk - 1)], id[j] = pt[min(tid + kThreads * j, nblk - 1)];
  }
  // The thread's columns, of the blocks but the first and the last: visit(f) calls f(column, score, place in `id`).
  const int per = (nblk + kThreads - 1) / kThreads, from = max(min(tid * per, nblk), 1), to = min(tid * per + per, nblk - 1);  // (not HELD)
  const bool in_lds = !HELD && a.w <= kLdsColumns;
  const auto visit = [&](const auto &f) {
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        const int c = tid + kThreads * j;
        if (j < held && c > 0 && c < nblk - 1) f(c, x[j].x, j);
      }
    } else {
#pragma unroll 1
      for (int c = from; c < to; ++c) f(c, in_lds ? s_score[c] : scores[c].x, c);
    }
  };
  const auto page = [&](int j) {
    if constexpr (HELD) return id[j];
    return pt[j];
  };
  uint32_t hi = 0, lo = ~0u;
  float size = 0.f;  // largest sum of magnitudes
  if constexpr (HELD) {
    visit([&](int, float v, int j) { size = fmaxf(size, x[j].y), hi = max(hi, float_key(v)), lo = min(lo, float_key(v)); });
  } else {
#pragma unroll 4
    for (int c = 1 + tid; c < nblk - 1; c += kThreads) {
      const float2 v = scores[c];
      if (in_lds) s_score[c] = v.x;
      size = fmaxf(size, v.y), hi = max(hi, float_key(v.x)), lo = min(lo, float_key(v.x));
    }
  }
  extent(s, hi, lo, size);
  const int need = a.kept - 2;
  const Choice approx = last_kept<uint32_t>(s, need, hi, lo, [&](const auto &f) { visit([&](int, float v, int) { f(float_key(v)); }); });
  // T, and how far a score may be from the exact one: at most 512 additions, each off by at most a unit in the last place of what the magnitudes
  // add up to (2^-23), twice that for what the matrix pipe's own order and rounding may be; and what falls below the smallest normal number.
  const uint32_t tb = (uint32_t)approx.threshold;
  const float t = __builtin_bit_cast(float, (tb >> 31) ? tb & 0x7fffffffu : ~tb);
  const float e = size * 0x1p-13f + 0x1p-100f;
  const bool exact_all = !(size < INFINITY) || !(fabsf(t) < INFINITY);  // infinities among the scores: no bound says anything
  const float sure = exact_all ? INFINITY : t + 2.f * e, out = exact_all ? -INFINITY : t - 2.f * e;
  const auto kept_surely = [&](float v) { return !exact_all && need > 0 && v > sure; };
  const auto in_question = [&](float v) { return exact_all || (need > 0 && v >= out && !(v > sure)); };
  // Two running counts over the columns in order, of those that p and q hold for: the counts in front of the thread's columns (HELD: of each), and of all.
  struct Places {
    int p[HELD ? kHeld : 1], q[HELD ? kHeld : 1], all_p, all_q;
  };
  const auto count = [&](const auto &p, const auto &q) {
    Places o;
    if constexpr (HELD) {
      // (for each row of kThreads columns both counts in a word)
      int n[kHeld] = {};
      visit([&](int c, float v, int j) { n[j] = (int)p(c, v) | (int)q(c, v) << 16; });
      const Counts<kHeld> r = running_counts<kHeld>(s, n, held);
      o.all_p = o.all_q = 0;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        o.p[j] = o.all_p + (r.before[j] & 0xffff), o.q[j] = o.all_q + (r.before[j] >> 16);
        o.all_p += r.all[j] & 0xffff, o.all_q += r.all[j] >> 16;
      }
    } else {
      int n[2] = {0, 0};
      visit([&](int c, float v, int) { n[0] += p(c, v), n[1] += q(c, v); });
      const Counts<2> r = running_counts<2>(s, n);
      o.p[0] = r.before[0], o.q[0] = r.before[1], o.all_p = r.all[0], o.all_q = r.all[1];
    }
    return o;
  };
  // f(column, score, place in `id`, the two counts in front of it)
  const auto walk = [&](const Places &o, const auto &p, const auto &q, const auto &f) {
    if constexpr (HELD) {
      visit([&](int c, float v, int j) { f(c, v, j, o.p[j], o.q[j]); });
    } else {
      int np = o.p[0], nq = o.q[0];
      visit([&](int c, float v, int j) {
        f(c, v, j, np, nq);
        np += p(c, v), nq += q(c, v);
      });
    }
  };
  const auto is_sure = [&](int, float v) { return kept_surely(v); };
  const auto is_open = [&](int, float v) { return in_question(v); };
  const Places n = count(is_sure, is_open);
  const int open = n.all_q, need_open = need - n.all_p;
  constexpr int GROUPS = 256 / D;  // of lanes with a score of their own, in a wavefront
  const int group = wave * GROUPS + lane / (D / 4);
  uint64_t *const keys = a.keys + seg * a.row;
  if (open <= kRanked) {
    // few in question: their exact scores and ranks in LDS
    walk(n, is_sure, is_open, [&](int, float v, int j, int, int at) {
      if (in_question(v)) s.column[at] = page(j), s.cand[at] = 0;
    });
    __syncthreads();
#pragma unroll 1
    for (int i = group; i - group < open * a.g; i += kWaves * GROUPS) {
      const int y = min(i, open * a.g - 1), o = y / a.g;
      const uint64_t k = exact_key<D>(a, u, h, y - o * a.g, s.column[o]);
      if (lane % (D / 4) == 0 && i < open * a.g) atomicMax(reinterpret_cast<unsigned long long *>(&s.cand[o]), (unsigned long long)k);
    }
    __syncthreads();
    if (tid < open) {
      const uint64_t k = s.cand[tid];
      int better = 0;  // (columns are in order: of equals the first ones)
#pragma unroll 1
      for (int i = 0; i < open; ++i) better += s.cand[i] > k || (s.cand[i] == k && i < tid);
      s.kept[tid] = better < need_open;
    }
    __syncthreads();
    walk(n, is_sure, is_open, [&](int c, float v, int j, int at, int open_at) {
      if (!kept_surely(v) && !(in_question(v) && s.kept[open_at])) return;
      ++at;  // (column 0 is in front)
#pragma unroll 1
      for (int i = 0; i < open_at; ++i) at += s.kept[i];
      emit(at, c, page(j));
    });
  } else {
    // many (scores alike, infinities): exact scores of all in memory, and the choice among those in question by them
#pragma unroll 1
    for (int i = group; i - group < nblk; i += kWaves * GROUPS) {
      const int c = min(i, nblk - 1);
      uint64_t k = 0;
#pragma unroll 1
      for (int g = 0; g < a.g; ++g) k = max(k, exact_key<D>(a, u, h, g, pt[c]));
      if (lane % (D / 4) == 0 && i < nblk) keys[i] = k;
    }
    __syncthreads();
    const auto those = [&](const auto &f) {
      visit([&](int c, float v, int) {
        if (in_question(v)) f(keys[c]);
      });
    };
    uint64_t high = 0, low = ~0ull;
    those([&](uint64_t k) { high = max(high, k), low = min(low, k); });
    extent(s, high, low, size);
    const Choice exact = last_kept<uint64_t>(s, need_open, high, low, those);
    // what is kept for sure or by its exact score; of the blocks tied for the last places the first ones
    const auto is_kept = [&](int c, float v) { return kept_surely(v) || (in_question(v) && keys[c] > exact.threshold); };
    const auto is_tied = [&](int c, float v) { return in_question(v) && keys[c] == exact.threshold; };
    __syncthreads();
    walk(count(is_kept, is_tied), is_kept, is_tied, [&](int c, float v, int j, int at, int tied_at) {
      if (is_kept(c, v) || (is_tied(c, v) && tied_at < exact.ties)) emit(1 + at + min(tied_at, exact.ties), c, page(j));
    });
  }
}

// One workgroup per (user, KV head); what bounds it is its own chain (three round trips to memory, a dozen barriers) and, as every launch begins with a cold
// instruction cache, its code.  128 (user, head) pairs of 64 ... 512 blocks 6.5 us, 32 of 1024 ... 2048 9.2 (scores and pages in LDS throughout 7.1 and 12.4; unrolled
// over sixteen columns and with 1024 threads 21); a pass over 8192 columns, in LDS / where they lie, 46.1 / 51.8.  Scores made in the same workgroup instead of a
// launch of their own: 35.2 / 32.5 the first pass, 54.9 / 30.4 the second.
template <int D, bool LONG>
__global__ __launch_bounds__(kThreads) void choose_blocks_kernel(ScoreArgs a) {
  __shared__ ChoiceLds s;
  extern __shared__ float s_score[];
  const int tid = threadIdx.x;
  const int seg = blockIdx.x, u = seg / a.hkv, h = seg - u * a.hkv;
  const int32_t *pt = a.pt + u * a.pt_rs;
  // (asked for before it is known how many there are; scores that nobody has written are not used)
  const float2 x0 = a.scores[seg * a.row + min(tid, a.w - 1)];
  const int id0 = pt[min(tid, a.w - 1)];
  int64_t pos = load_index(a.cur, a.cur_i64, u);
  const int nblk = blocks_of(a, u, pos);
  int32_t *table = a.table + (int64_t)seg * a.kept, *columns = a.columns + (int64_t)seg * a.kept;
  const int chosen = min(nblk, a.kept);
  const auto emit = [&](int at, int c, int page) {
    table[at] = ((unsigned)page < (unsigned)a.nb ? page : 0) * a.hkv + h;
    columns[at] = c;
  };
#pragma unroll 1
  for (int i = chosen + tid; i < a.kept; i += kThreads) table[i] = h, columns[i] = -1;
  if (tid == 0) {
    a.pos[seg] = nblk ? (int)((int64_t)(chosen - 1) * a.bs + (pos - (int64_t)(nblk - 1) * a.bs)) : -1;
    a.arrived[seg] = 0;
  }
  if (nblk <= a.kept) {
#pragma unroll 1
    for (int c = tid; c < nblk; c += kThreads) emit(c, c, pt[c]);
    return;
  }
  if (tid == 0) emit(0, 0, pt[0]), emit(a.kept - 1, nblk - 1, pt[nblk - 1]);
  if constexpr (LONG) {
    if (nblk > kHeld * kThreads) {
      choose_among<D, false>(a, s, s_score, seg, u, h, nblk, x0, id0, emit);
      return;
    }
  }
  choose_among<D, true>(a, s, s_score, seg, u, h, nblk, x0, id0, emit);
}

constexpr int kScoreWorkgroups = 1024;
template <int D>
int launch_choice(const ScoreArgs &a, hipStream_t st) {
  const int segments = a.users * a.hkv;
  if (a.w > a.kept) {
    // Tables are wide where contexts may grow long: not more workgroups than are at work at once about, each of which goes on until its context ends, and
    // a context's workgroups as far apart as there are contexts, so that those that have work are on all XCDs.  (Side by side, and as many as the table is
    // wide, 16 users of 4096 ... 32768 tokens took 31.9 us where the table ended with them and 68 in a table of 16384 columns; so 31.6 and 32.1.)
    constexpr int kBlocks = 4 * 16 * score_tiles<D>();
    const int most = std::max(kScoreWorkgroups / segments, 1);
    block_scores_kernel<D><<<dim3(segments, std::min((a.w + kBlocks - 1) / kBlocks, most)), dim3(256), 0, st>>>(a);
    if (const int rc = check_launch("fp8 sparse decode (scores)")) return rc;
  }
  if (a.w <= kHeld * kThreads)
    choose_blocks_kernel<D, false><<<dim3(segments), dim3(kThreads), 0, st>>>(a);
  else
    choose_blocks_kernel<D, true><<<dim3(segments), dim3(kThreads), a.w <= kLdsColumns ? 4 * (size_t)a.w : 0, st>>>(a);
  return check_launch("fp8 sparse decode (choice)");
}

// ---- the attention's launch ----------------------------------------------------------------------------
// Wavefronts of the workgroup that reads a whole segment, or 0.  The limit is where lists of few segments turn (us a pass whole / cut, one user of
// 32/8 heads of 128: 1024 tokens 8.1 / 10.9, 2048 14.1 / 10.8; 8 users 11.1 / 10.8 and 17.3 / 12.4).  With a segment for every CU and contexts about
// alike whole segments stay ahead beyond it (128 users, 1024 ... 2048 tokens 67.5 / 75.2), but not over ragged ones, and the host cannot
// tell them apart (64 users of 32 ... 2048 24.5 / 20.2).
int fp8_direct_waves(int users, int kv_heads, int head_size, int64_t tokens) {
  const int64_t segments = (int64_t)users * kv_heads, bytes = tokens * head_size * 2;
  const char *forced_name = getenv("TTPA_DECODE_KERNEL");
  const bool ranges = (forced_name && !strcmp(forced_name, "ranges")) || getenv("TTPA_DECODE_WAVES_PER_CU");
  const bool direct = forced_name && !strcmp(forced_name, "direct");
  if (!direct && (ranges || bytes > 272 * 1024)) return 0;
  int cus = device_cus();
  if (cus <= 0) cus = 256;
  const int tile = head_size <= 128 ? 64 : 32;
  return head_size > 128 || segments > cus || tokens <= 4 * tile ? 4 : 8;
}

// Workgroups that a sparse pass's scratch has room for, beyond one per segment: so many may share a segment.
int sparse_slots() { return 4 * std::max(device_cus(), 256); }
int most_sparse_parts(int segments) { return sparse_slots() / segments; }

// arrived: counters of the segments, at zero, with which several workgroups may share a segment of equal ones; or null.
int attend(DecodeArgs a, const float *k_scales, const float *v_scales, int head_size, int *arrived, hipStream_t st) {
  const int g = a.hq / a.hkv;
  int64_t tokens = (int64_t)a.w * a.bs;
  if (a.window > 0) tokens = std::min<int64_t>(tokens, a.window);
  a.slot_floats = slot_floats_for(g, head_size);
  a.kv_format = -1;
  a.direct = fp8_direct_waves(a.users, a.hkv, head_size, tokens);
  const int segments = a.users * a.hkv;
  int parts = 1;
  if (arrived) {
    // Segments of one length, about: as many workgroups each as make the rounds of workgroups, one per CU, times a wavefront's tiles and about two more for
    // its beginning and end fewest.  us a pass, as many as there are CUs for, rounded up / so, 32 blocks of 64 tokens of 32/8 heads of 128: 10 users 33.4 / 27.2, 20
    // 44.2 / 35.1, 24 45.8 / 37.7; of 64: 10 users 26.7 / 22.7, 24 33.1 / 26.3; 16/4 heads of 256: 33 users 57.6 / 51.6.  (Two per CU, which there is room for at 64 and
    // 256: 16 users of 64 25.0 / 28.9, 4 of 256 29.9 / 33.6.)  Wavefronts: 128 segments of 2048 tokens 4 x 2 36.2, 8 x 2 35.7; 32 of 4096 4 x 8 35.9, 8 x 8 35.1.
    const int tile = head_size <= 128 ? 64 : 32, tiles = (int)((tokens + tile - 1) / tile), cus = std::max(device_cus(), 1);
    a.direct = head_size <= 128 ? 8 : 4;
    int64_t best = INT64_MAX;
    for (int p = 1; p <= std::min({(tiles + a.direct - 1) / a.direct, kMostParts, std::max(most_sparse_parts(segments), 1)}); ++p) {
      const int64_t cost = ((int64_t)segments * p + cus - 1) / cus * ((tiles + a.direct * p - 1) / (a.direct * p) + 2);
      if (cost < best) best = cost, parts = p;
    }
  }
  // Four wavefronts per CU, and eight over a long list at head size 64, whose tiles are half as large.  How long the list is the kernel
  // knows, and then leaves half of the ranges empty.  us a pass at four / eight, 32/8 heads of 64: 8 users of 2048 ... 4096 tokens (3000 tiles) 11.8 / 12.7,
  // 24 of 32 ... 4096 (6000) 12.0 / 12.2, 24 of 32 ... 8192 (12 000) 15.4 / 14.3, 32 of 8000 ... 16384 (49 000) 74.4 / 67.5; at 128 and 256 lists of
  // 50 000 tiles gain 1 %, shorter ones lose 3 - 15 %.
  const int larger_grid = waves_for_device(8.0);
  a.n_waves = waves_for_device(4.0);
  // (few_ranges also keeps the merge in whole pieces where its slices do not fit the chip at once, with 128 segments and wide groups: 32 users of
  // 2000 ... 6000 tokens, 64/4 heads of 128 36.4 / 33.1, of 256 62.1 / 55.9.)
  a.few_ranges = a.n_waves, a.many_from = 0;
  if (head_size == 64 && segments * ((tokens + 63) / 64 + 1) >= 3 * (int64_t)larger_grid) a.n_waves = larger_grid, a.many_from = 3 * (int64_t)larger_grid;
  a.seg_units = segment_units(1);
  if (!segment_units_forced()) a.seg_free_tiles = a.n_waves;
  if (!a.direct && segments > (int64_t)a.n_waves * kWave)
    return fail(TTPA_ERR_UNSUPPORTED, "fp8 decode: %d segments need a grid of more than %d wavefronts", segments, a.n_waves);
  const uint32_t runs = (uint32_t)a.bs / (head_size <= 128 ? 16 : 8);
  const uint32_t negate = a.scale_log2e < 0.f ? 0x80008000u : 0u;
  a.scale_log2e = fabsf(a.scale_log2e);
  const Fp8Args fa = {a, k_scales, v_scales, negate, runs, 0xffffffffu / runs, parts, arrived};
  const bool ok = head_size == 64 ? launch_fp8_d64(&fa, st) : head_size == 128 ? launch_fp8_d128(&fa, st) : launch_fp8_d256(&fa, st);
  hipEvent_t ev0, ev1;
  take_profile_events(ev0, ev1);  // still armed only if the launch did not happen
  if (!ok) return fail(TTPA_ERR_LAUNCH, "fp8 decode: cannot configure the kernel");
  if (!a.direct) launch_combine(a, segments, g, head_size, st);
  return check_launch("paged_fp8_decode");
}

int check_decode(const void *out, int64_t out_us, int64_t out_hs, const void *q, int64_t q_us, int64_t q_hs, const void *cur_pos, int users,
                 int q_heads, int kv_heads) {
  TTPA_REQUIRE(out && q && cur_pos, "fp8 decode: null pointer argument");
  TTPA_REQUIRE(users > 0 && q_heads > 0, "fp8 decode: non-positive dimension");
  TTPA_REQUIRE(q_heads % kv_heads == 0, "fp8 decode: q_heads %d not divisible by kv_heads %d", q_heads, kv_heads);
  if (q_heads / kv_heads > 16)
    return fail(TTPA_ERR_UNSUPPORTED, "fp8 decode: %d query heads per KV head; built for up to 16", q_heads / kv_heads);
  TTPA_REQUIRE(aligned16(q) && aligned16(out), "fp8 decode: q / out must be 16-byte aligned");
  TTPA_REQUIRE(q_us % 8 == 0 && q_hs % 8 == 0, "fp8 decode: q strides must be multiples of 8 elements");
  (void)out_us, (void)out_hs;
  return TTPA_OK;
}

// A sparse call's scratch behind the attention's: the scores' keys, the tables, the positions.
struct SparseLayout {
  size_t slots, row, keys, table, total;
};
SparseLayout sparse_layout(int users, int q_heads, int kv_heads, int head_size, int table_width, int kept) {
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t segments = (size_t)users * kv_heads;
  const size_t slots = (size_t)sparse_slots() + segments;
  SparseLayout l;
  l.slots = up(slots * slot_floats_for(q_heads / kv_heads, head_size) * sizeof(float));
  l.row = ((size_t)table_width + 15) / 16 | 1;  // (an odd number of lines: rows that begin on the same channels of the memory wait for each other)
  l.row *= 16;
  l.keys = up(segments * l.row * 8);  // scores, and as much for exact ones
  l.table = up(segments * (size_t)kept * 4);
  l.total = l.slots + 2 * l.keys + l.table + 2 * up(segments * 4);
  return l;
}
constexpr int kSparseSegments = kMaxUsers;  // (user, KV head) pairs per pass
int sparse_users(int users, int kv_heads) { return std::max(1, std::min(users, kSparseSegments / std::max(kv_heads, 1))); }

}  // namespace
}  // namespace decode
}  // namespace ttpa

using namespace ttpa;
using namespace ttpa::decode;

extern "C" int ttpa_paged_fp8_decode(void *out, int64_t out_user_stride, int64_t out_head_stride, const void *q, int64_t q_user_stride,
                                     int64_t q_head_stride, const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
                                     const int32_t *page_table, int64_t page_table_row_stride, const void *cur_pos, int cur_pos_is_i64,
                                     int32_t users, int32_t q_heads, int32_t kv_heads, int32_t head_size, int32_t block_size, int32_t table_width,
                                     int32_t num_blocks, float scale, int32_t sliding_window, const float *attention_sink, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  if (int rc = check_decode(out, out_user_stride, out_head_stride, q, q_user_stride, q_head_stride, cur_pos, users, q_heads, kv_heads)) return rc;
  TTPA_REQUIRE(sliding_window >= 0, "fp8 decode: sliding_window %d is negative", sliding_window);
  if (users > kMaxUsers) return fail(TTPA_ERR_UNSUPPORTED, "fp8 decode: %d users exceeds the limit of %d", users, kMaxUsers);
  const size_t need = ttpa_paged_decode_workspace_bytes(users, q_heads, kv_heads, head_size);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(TTPA_ERR_WORKSPACE, "fp8 decode: workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace_bytes);
  DecodeArgs a = {};
  a.out = static_cast<uint16_t *>(out), a.out_us = out_user_stride, a.out_hs = out_head_stride;
  a.q = static_cast<const uint16_t *>(q), a.q_us = q_user_stride, a.q_hs = q_head_stride;
  a.k = static_cast<const uint8_t *>(k_cache), a.v = static_cast<const uint8_t *>(v_cache);
  a.pt = page_table, a.pt_rs = page_table_row_stride, a.cur = cur_pos, a.cur_i64 = cur_pos_is_i64;
  a.users = users, a.hq = q_heads, a.hkv = kv_heads, a.bs = block_size, a.w = table_width, a.nb = num_blocks;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.ws_seg = static_cast<int *>(workspace);
  a.ws_slots = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + header_bytes(users, kv_heads));
  a.window = sliding_window, a.sink = attention_sink;
  return attend(a, k_scales, v_scales, head_size, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" size_t ttpa_paged_fp8_sparse_decode_workspace_bytes(int32_t users, int32_t q_heads, int32_t kv_heads, int32_t head_size,
                                                               int32_t table_width, int32_t kept_blocks) {
  if (users <= 0 || q_heads <= 0 || kv_heads <= 0 || head_size <= 0 || q_heads % kv_heads || table_width <= 0 || kept_blocks <= 0) return 0;
  return sparse_layout(sparse_users(users, kv_heads), q_heads, kv_heads, head_size, table_width, kept_blocks).total;
}

extern "C" int ttpa_paged_fp8_sparse_decode(void *out, int64_t out_head_stride, int32_t *columns, const void *q, int64_t q_head_stride,
                                            const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
                                            const void *key_bounds, const int32_t *page_table, int64_t page_table_row_stride, const void *cur_pos,
                                            int cur_pos_is_i64, int32_t users, int32_t q_heads, int32_t kv_heads, int32_t head_size,
                                            int32_t block_size, int32_t table_width, int32_t num_blocks, int32_t kept_blocks, float scale,
                                            void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  if (int rc = check_decode(out, 0, out_head_stride, q, 0, q_head_stride, cur_pos, users, q_heads, kv_heads)) return rc;
  TTPA_REQUIRE(key_bounds && columns && aligned16(key_bounds), "fp8 sparse decode: bounds must be 16-byte aligned, columns not null");
  TTPA_REQUIRE(kept_blocks >= 2 && (int64_t)kept_blocks * block_size < (1ll << 31) - 4096, "fp8 sparse decode: kept_blocks %d; at least 2", kept_blocks);
  if (kv_heads > kSparseSegments) return fail(TTPA_ERR_UNSUPPORTED, "fp8 sparse decode: %d KV heads exceeds the limit of %d", kv_heads, kSparseSegments);
  const int per = sparse_users(users, kv_heads), g = q_heads / kv_heads;
  const SparseLayout l = sparse_layout(per, q_heads, kv_heads, head_size, table_width, kept_blocks);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(TTPA_ERR_WORKSPACE, "fp8 sparse decode: workspace of %zu bytes (256-byte aligned) required, got %zu", l.total, workspace_bytes);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int u0 = 0; u0 < users; u0 += per) {
    const int n = std::min(per, users - u0), segments = n * kv_heads;
    ScoreArgs s = {};
    s.q = static_cast<const uint16_t *>(q) + (int64_t)u0 * q_heads * q_head_stride, s.q_us = (int64_t)q_heads * q_head_stride, s.q_hs = q_head_stride;
    s.bounds = static_cast<const uint16_t *>(key_bounds);
    s.pt = page_table + u0 * page_table_row_stride, s.pt_rs = page_table_row_stride;
    s.cur = static_cast<const uint8_t *>(cur_pos) + (int64_t)u0 * (cur_pos_is_i64 ? 8 : 4), s.cur_i64 = cur_pos_is_i64;
    s.users = n, s.hkv = kv_heads, s.g = g, s.bs = block_size, s.w = table_width, s.nb = num_blocks, s.kept = kept_blocks;
    s.row = (int64_t)l.row;
    s.scores = reinterpret_cast<float2 *>(ws + l.slots);
    s.keys = reinterpret_cast<uint64_t *>(ws + l.slots + l.keys);
    s.table = reinterpret_cast<int32_t *>(ws + l.slots + 2 * l.keys);
    s.pos = reinterpret_cast<int32_t *>(ws + l.slots + 2 * l.keys + l.table);
    s.arrived = s.pos + (segments + 63) / 64 * 64;
    s.columns = columns + (int64_t)u0 * kv_heads * kept_blocks;
    if (const int rc = head_size == 64 ? launch_choice<64>(s, st) : head_size == 128 ? launch_choice<128>(s, st) : launch_choice<256>(s, st)) return rc;
    DecodeArgs a = {};
    a.out = static_cast<uint16_t *>(out) + (int64_t)u0 * q_heads * out_head_stride, a.out_us = g * out_head_stride, a.out_hs = out_head_stride;
    a.q = s.q, a.q_us = g * q_head_stride, a.q_hs = q_head_stride;
    a.k = static_cast<const uint8_t *>(k_cache), a.v = static_cast<const uint8_t *>(v_cache);
    a.pt = s.table, a.pt_rs = kept_blocks, a.cur = s.pos, a.cur_i64 = 0;
    a.users = segments, a.hq = g, a.hkv = 1, a.bs = block_size, a.w = kept_blocks, a.nb = num_blocks * kv_heads;
    a.scale_log2e = scale * 1.4426950408889634f;
    a.ws_slots = reinterpret_cast<float *>(ws);
    if (const int rc = attend(a, k_scales, v_scales, head_size, s.arrived, st)) return rc;
  }
  return TTPA_OK;
}
