// Decode attention over the 8-bit cache: entry points, and the choice of blocks for its sparse form.
//
// Sparse form.  For every (user, KV head) the blocks of the context are scored by what their key bounds allow,
//   score(block) = max over the group's heads of  sum_d  max(q_d, 0) high_d + min(q_d, 0) low_d,
// an upper bound of q . k over the block's keys; the block that holds the newest token, the first block and the best of the others are
// attended, `kept` in all, of equal scores the lower column.  A choice flips with the last bit of a score, so scores
// are sums in 64 bits: products of bfloat16 values are exact there and a sum of 256 of them keeps 30 bits to spare, so that
// neither the order of the sum nor its split matters in practice.
//   block_scores_kernel   a block's bounds are 4 D consecutive bytes, D / 4 lanes of 16 bytes: half of them hold lows and the negative
//                         parts of the queries, half highs and the positive parts.  Memory bound: each bound is read once for up to
//                         eight heads, whose parts a lane keeps in registers as doubles.
//   choose_blocks_kernel  one workgroup per (user, KV head): a histogram over the scores' range finds the bin the last kept block
//                         lies in, ranks inside that bin (or histograms of it, while it is crowded) find the block; the columns come out in
//                         order, as a page table of their own.
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
struct ScoreArgs {
  const uint16_t *q;
  int64_t q_us, q_hs;
  const uint16_t *bounds;
  const int32_t *pt;
  int64_t pt_rs;
  const void *cur;
  int cur_i64;
  int users, hkv, g, bs, w, nb, kept;
  uint64_t *keys;  // [users * hkv][w]
  int32_t *table;  // [users * hkv][kept]
  int32_t *pos;    // [users * hkv]
  int32_t *columns;  // [users, hkv, kept], the caller's
};

// Blocks of a user's context; 0 for a padded row.
__device__ __forceinline__ int blocks_of(const ScoreArgs &a, int u, int64_t &pos) {
  pos = load_index(a.cur, a.cur_i64, u);
  const int64_t cap = (int64_t)a.w * a.bs;
  if (pos >= cap) pos = cap - 1;
  return pos < 0 ? 0 : (int)(pos / a.bs) + 1;
}

constexpr uint64_t kAlways = ~0ull, kUnbounded = ~0ull - 1;
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
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_max_u64(uint64_t b) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
  const uint64_t o = (uint64_t)hi << 32 | lo;
  return b > o ? b : o;
}
constexpr int kDppRor1 = 0x121, kDppRor2 = 0x122, kDppRor4 = 0x124, kDppRor8 = 0x128;

// One level of the exchange that leaves each lane the sums of half of its heads: lanes with `bit` keep the upper half.
template <int CTRL, int N>
__device__ __forceinline__ void halve(double (&v)[N], int count, bool bit) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    if (i < count / 2) {
      const double keep = bit ? v[i + count / 2] : v[i], send = bit ? v[i] : v[i + count / 2];
      v[i] = keep + dpp_move_f64<CTRL>(send);
    }
}

constexpr int kScoreBlocks = 64;  // context blocks per workgroup: enough of them for eight users of 8 heads and 512 blocks to fill the chip

template <int D, int GH>
__global__ __launch_bounds__(256) void block_scores_kernel(ScoreArgs a) {
  constexpr int LPB = D / 4, BPW = 64 / LPB;  // lanes per block, blocks per wavefront and load
  constexpr int UNROLL = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int seg = blockIdx.y, u = seg / a.hkv, h = seg - u * a.hkv;
  int64_t pos;
  const int nblk = blocks_of(a, u, pos);
  if (nblk <= a.kept) return;  // all are attended
  const int from = blockIdx.x * kScoreBlocks, to = min(nblk, from + kScoreBlocks);
  const int in_block = lane % LPB, which = lane / LPB;
  const bool high = in_block >= LPB / 2;
  const int f = 8 * (in_block % (LPB / 2));
  const int32_t *pt = a.pt + u * a.pt_rs;
  for (int g0 = 0; g0 < a.g; g0 += GH) {
    double q[GH][8];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      fp8::u32x4 t = {0, 0, 0, 0};
      if (g0 + g < a.g) t = *reinterpret_cast<const fp8::u32x4 *>(a.q + u * a.q_us + (int64_t)(h * a.g + g0 + g) * a.q_hs + f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v0 = bf16_lo(t[i]), v1 = bf16_hi(t[i]);
        // (a NaN stays one in both parts)
        q[g][2 * i] = high ? (v0 < 0.f ? 0.f : v0) : (v0 > 0.f ? 0.f : v0);
        q[g][2 * i + 1] = high ? (v1 < 0.f ? 0.f : v1) : (v1 > 0.f ? 0.f : v1);
      }
    }
    for (int c0 = from + wave * BPW * UNROLL; c0 < to; c0 += 4 * BPW * UNROLL) {
      fp8::u32x4 raw[UNROLL];
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) {
        const int c = min(c0 + j * BPW + which, to - 1);
        const int id = pt[c];
        const int64_t slab = (int64_t)((unsigned)id < (unsigned)a.nb ? id : 0) * a.hkv + h;
        raw[j] = __builtin_nontemporal_load(reinterpret_cast<const fp8::u32x4 *>(a.bounds + slab * (2 * D) + (high ? D : 0) + f));
      }
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) {
        double s[GH];
#pragma unroll
        for (int g = 0; g < GH; ++g) s[g] = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double b0 = bf16_lo(raw[j][i]), b1 = bf16_hi(raw[j][i]);
#pragma unroll
          for (int g = 0; g < GH; ++g) s[g] = __builtin_fma(q[g][2 * i], b0, s[g]);
#pragma unroll
          for (int g = 0; g < GH; ++g) s[g] = __builtin_fma(q[g][2 * i + 1], b1, s[g]);
        }
        int count = GH;
        if constexpr (GH >= 8) halve<kDppHalfMirror>(s, count, lane & 4), count /= 2;
        if constexpr (GH >= 4) halve<kDppXor2>(s, count, lane & 2), count /= 2;
        if constexpr (GH >= 2) halve<kDppXor1>(s, count, lane & 1), count /= 2;
        double t = s[0];
        t += dpp_move_f64<kDppRor8>(t);
        if constexpr (GH < 8) t += dpp_move_f64<kDppRor4>(t);
        if constexpr (GH < 4) t += dpp_move_f64<kDppRor2>(t);
        if constexpr (GH < 2) t += dpp_move_f64<kDppRor1>(t);
        if constexpr (LPB >= 32) t += __shfl_xor(t, 16);
        if constexpr (LPB >= 64) t += __shfl_xor(t, 32);
        uint64_t key = g0 + (lane & (GH - 1)) < a.g ? score_key(t) : 0;
        if constexpr (GH >= 2) key = dpp_max_u64<kDppXor1>(key);
        if constexpr (GH >= 4) key = dpp_max_u64<kDppXor2>(key);
        if constexpr (GH >= 8) key = dpp_max_u64<kDppHalfMirror>(key);
        const int c = c0 + j * BPW + which;
        if (in_block == 0 && c < to) {
          uint64_t *dst = a.keys + (int64_t)seg * a.w + c;
          if (g0 > 0) key = max(key, *dst);
          if (c == 0 || c == nblk - 1) key = kAlways;
          *dst = key;
        }
      }
    }
  }
}

// ---- choice ----------------------------------------------------------------------------------------
constexpr int kBins = 1024, kHeld = 4096, kRanked = 256;

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, m);
    v = v > o ? v : o;
  }
  return v;
}

__global__ __launch_bounds__(256) void choose_blocks_kernel(ScoreArgs a) {
  __shared__ uint64_t s_keys[kHeld];
  __shared__ uint32_t s_bins[kBins];
  __shared__ uint64_t s_cand[kRanked];
  __shared__ uint64_t s_red[8];
  __shared__ int s_int[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int seg = blockIdx.x, u = seg / a.hkv, h = seg - u * a.hkv;
  int64_t pos;
  const int nblk = blocks_of(a, u, pos);
  const int32_t *pt = a.pt + u * a.pt_rs;
  int32_t *table = a.table + (int64_t)seg * a.kept, *columns = a.columns + (int64_t)seg * a.kept;
  const int chosen = min(nblk, a.kept);
  const auto emit = [&](int at, int c) {
    const int id = pt[c];
    table[at] = ((unsigned)id < (unsigned)a.nb ? id : 0) * a.hkv + h;
    columns[at] = c;
  };
  for (int i = chosen + tid; i < a.kept; i += 256) table[i] = h, columns[i] = -1;
  if (tid == 0) a.pos[seg] = nblk ? (int)((int64_t)(chosen - 1) * a.bs + (pos - (int64_t)(nblk - 1) * a.bs)) : -1;
  if (nblk <= a.kept) {
    for (int c = tid; c < nblk; c += 256) emit(c, c);
    return;
  }
  const uint64_t *keys = a.keys + (int64_t)seg * a.w;
  const bool held = nblk <= kHeld;
  const auto key_at = [&](int c) { return held ? s_keys[c] : keys[c]; };
  // The range of the keys that are not always kept; the first and the last block are.
  uint64_t hi = 0, lo = ~0ull;
  for (int c = tid; c < nblk; c += 256) {
    const uint64_t k = keys[c];
    if (held) s_keys[c] = k;
    if (k != kAlways) hi = max(hi, k), lo = min(lo, k);
  }
  hi = wave_max_u64(hi), lo = ~wave_max_u64(~lo);
  if (lane == 0) s_red[wave] = hi, s_red[4 + wave] = lo;
  __syncthreads();
  hi = max(max(s_red[0], s_red[1]), max(s_red[2], s_red[3]));
  lo = min(min(s_red[4], s_red[5]), min(s_red[6], s_red[7]));
  // `need` blocks with keys in [lo, hi] are kept besides those with larger keys: narrow the range until few are in question.
  int need = a.kept - 2;
  uint64_t threshold = 0;  // keys above it are kept, and of those equal to it the first `ties` columns
  int ties = 0;
  for (;;) {
    if (need == 0) {
      threshold = hi;
      break;
    }
    if (lo == hi) {
      threshold = lo, ties = need;
      break;
    }
    const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 10);  // (hi - lo) >> shift < 1024
    for (int i = tid; i < kBins; i += 256) s_bins[i] = 0;
    __syncthreads();
    for (int c = tid; c < nblk; c += 256) {
      const uint64_t k = key_at(c);
      if (k >= lo && k <= hi) atomicAdd(&s_bins[(k - lo) >> shift], 1u);
    }
    __syncthreads();
    // the bin, from the top, where the count reaches `need`: thread t owns bins 4 (255 - t) .. + 3
    const int base = 4 * (255 - tid);
    uint32_t mine[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[j] = s_bins[base + j], sum += mine[j];
    const int incl = wave_prefix_sum((int)sum);
    if (lane == 63) s_int[wave] = incl;
    __syncthreads();
    int above = incl - (int)sum;
    for (int w = 0; w < wave; ++w) above += s_int[w];
    if (above < need && above + (int)sum >= need) {  // one thread
      int b = 3;
      while (above + (int)mine[b] < need) above += mine[b], --b;
      s_int[4] = base + b, s_int[5] = above, s_int[6] = (int)mine[b];
    }
    __syncthreads();
    const int bin = s_int[4], over = s_int[5], count = s_int[6];
    need -= over;
    const uint64_t span = ((uint64_t)1 << shift) - 1;
    lo += (uint64_t)bin << shift;
    hi = hi - lo < span ? hi : lo + span;  // (the last bin may reach past the largest number)
    if (shift == 0 || count == need) {
      // all keys of the bin are alike, or all are kept
      if (count == need) threshold = lo - 1;
      else threshold = lo, ties = need;
      break;
    }
    if (count <= kRanked) {
      if (tid == 0) s_int[7] = 0;
      __syncthreads();
      for (int c = tid; c < nblk; c += 256) {
        const uint64_t k = key_at(c);
        if (k >= lo && k <= hi) s_cand[atomicAdd(&s_int[7], 1)] = k;
      }
      __syncthreads();
      if (tid < count) {
        // the need-th largest: fewer than `need` keys are larger, and with its equals there are enough
        const uint64_t k = s_cand[tid];
        int larger = 0, equal = 0;
        for (int i = 0; i < count; ++i) larger += s_cand[i] > k, equal += s_cand[i] == k;
        if (larger < need && larger + equal >= need) s_red[0] = k, s_int[4] = need - larger;  // (equal keys write the same)
      }
      __syncthreads();
      threshold = s_red[0], ties = s_int[4];
      break;
    }
    __syncthreads();
  }
  // the columns in order: a run of `per` neighbouring columns per thread would serialise; 256 at a time with running counts
  int at = 0, tied = 0;
  for (int c0 = 0; c0 < nblk; c0 += 256) {
    const int c = c0 + tid;
    const uint64_t k = c < nblk ? key_at(c) : 0;
    const bool is = c < nblk, tie = is && k == threshold && ties > 0, above = is && k > threshold;
    const uint64_t tie_lanes = __builtin_amdgcn_ballot_w64(tie);
    __syncthreads();  // (the counts of the pass before are read)
    if (lane == 0) s_int[wave] = __builtin_popcountll(tie_lanes);
    __syncthreads();
    int rank = tied + __builtin_amdgcn_mbcnt_hi((uint32_t)(tie_lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)tie_lanes, 0));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) rank += s_int[w];
      tied += s_int[w];
    }
    const bool take = above || (tie && rank < ties);
    const uint64_t take_lanes = __builtin_amdgcn_ballot_w64(take);
    if (lane == 0) s_int[4 + wave] = __builtin_popcountll(take_lanes);
    __syncthreads();
    int to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(take_lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)take_lanes, 0));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) to += s_int[4 + w];
      at += s_int[4 + w];
    }
    if (take && to < a.kept) emit(to, c);
  }
}

template <int D>
void launch_scores(const ScoreArgs &a, hipStream_t st) {
  const dim3 grid((a.w + kScoreBlocks - 1) / kScoreBlocks, a.users * a.hkv);
  if (a.g <= 1) block_scores_kernel<D, 1><<<grid, dim3(256), 0, st>>>(a);
  else if (a.g <= 2) block_scores_kernel<D, 2><<<grid, dim3(256), 0, st>>>(a);
  else if (a.g <= 4) block_scores_kernel<D, 4><<<grid, dim3(256), 0, st>>>(a);
  else block_scores_kernel<D, 8><<<grid, dim3(256), 0, st>>>(a);
}

// ---- the attention's launch ----------------------------------------------------------------------------
// Wavefronts of the workgroup that reads a whole segment, or 0 (see direct_waves in decode.hip).
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

int attend(DecodeArgs a, const float *k_scales, const float *v_scales, int head_size, hipStream_t st) {
  const int g = a.hq / a.hkv;
  int64_t tokens = (int64_t)a.w * a.bs;
  a.bs_magic = block_magic(tokens, a.bs);
  if (a.window > 0) tokens = std::min<int64_t>(tokens, a.window);
  a.slot_floats = slot_floats_for(g, head_size);
  a.kv_format = -1;
  a.direct = fp8_direct_waves(a.users, a.hkv, head_size, tokens);
  a.n_waves = waves_for_device(4.0);
  a.seg_units = segment_units(1);
  if (!segment_units_forced()) a.seg_free_tiles = a.n_waves;
  if (!a.direct && (int64_t)a.users * a.hkv > (int64_t)a.n_waves * kWave)
    return fail(TTPA_ERR_UNSUPPORTED, "fp8 decode: %d x %d segments need a grid of more than %d wavefronts", a.users, a.hkv, a.n_waves);
  const uint32_t runs = (uint32_t)a.bs / (head_size <= 128 ? 16 : 8);
  const uint32_t negate = a.scale_log2e < 0.f ? 0x80008000u : 0u;
  a.scale_log2e = fabsf(a.scale_log2e);
  const Fp8Args fa = {a, k_scales, v_scales, negate, runs, 0xffffffffu / runs};
  const bool ok = head_size == 64 ? launch_fp8_d64(&fa, st) : head_size == 128 ? launch_fp8_d128(&fa, st) : launch_fp8_d256(&fa, st);
  hipEvent_t ev0, ev1;
  take_profile_events(ev0, ev1);  // still armed only if the launch did not happen
  if (!ok) return fail(TTPA_ERR_LAUNCH, "fp8 decode: cannot configure the kernel");
  if (!a.direct) launch_combine(a, a.users * a.hkv, g, head_size, st);
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
  size_t decode, keys, table, total;
};
SparseLayout sparse_layout(int users, int q_heads, int kv_heads, int head_size, int table_width, int kept) {
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t segments = (size_t)users * kv_heads;
  SparseLayout l;
  l.decode = up(ttpa_paged_decode_workspace_bytes((int32_t)segments, q_heads / kv_heads, 1, head_size));
  l.keys = up(segments * (size_t)table_width * 8);
  l.table = up(segments * (size_t)kept * 4);
  l.total = l.decode + l.keys + l.table + up(segments * 4);
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
  return attend(a, k_scales, v_scales, head_size, static_cast<hipStream_t>(stream));
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
    s.keys = reinterpret_cast<uint64_t *>(ws + l.decode);
    s.table = reinterpret_cast<int32_t *>(ws + l.decode + l.keys);
    s.pos = reinterpret_cast<int32_t *>(ws + l.decode + l.keys + l.table);
    s.columns = columns + (int64_t)u0 * kv_heads * kept_blocks;
    if (table_width > kept_blocks) {
      if (head_size == 64) launch_scores<64>(s, st);
      else if (head_size == 128) launch_scores<128>(s, st);
      else launch_scores<256>(s, st);
      if (const int rc = check_launch("fp8 sparse decode (scores)")) return rc;
    }
    choose_blocks_kernel<<<dim3(segments), dim3(256), 0, st>>>(s);
    if (const int rc = check_launch("fp8 sparse decode (choice)")) return rc;
    DecodeArgs a = {};
    a.out = static_cast<uint16_t *>(out) + (int64_t)u0 * q_heads * out_head_stride, a.out_us = g * out_head_stride, a.out_hs = out_head_stride;
    a.q = s.q, a.q_us = g * q_head_stride, a.q_hs = q_head_stride;
    a.k = static_cast<const uint8_t *>(k_cache), a.v = static_cast<const uint8_t *>(v_cache);
    a.pt = s.table, a.pt_rs = kept_blocks, a.cur = s.pos, a.cur_i64 = 0;
    a.users = segments, a.hq = g, a.hkv = 1, a.bs = block_size, a.w = kept_blocks, a.nb = num_blocks * kv_heads;
    a.scale_log2e = scale * 1.4426950408889634f;
    a.ws_seg = reinterpret_cast<int *>(ws);
    a.ws_slots = reinterpret_cast<float *>(ws + header_bytes(segments, 1));
    if (const int rc = attend(a, k_scales, v_scales, head_size, st)) return rc;
  }
  return TTPA_OK;
}
