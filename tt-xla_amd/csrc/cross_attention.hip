// Attention of tokens to an encoder's states in a paged cache, of bfloat16 values or of one byte per element: a length per user, no causal limit.
//
//   out[u, h, t] = sum_j softmax_j(scale q[u, h, t] . k[u, j]) v[u, j],   j < len[u];   zeros where len[u] is 0
//
// This file holds the forms for few rows (a token per user, drafted ones, short texts) and the choice; many rows are the streaming prefill loop's
// (prefill_stream_kernel.h, kEnds).  All tokens of a user see the same keys, so the rows of a KV head are its G query heads times the tokens.  Up to 32 rows, a workgroup's four
// wavefronts have tiles of their own of a part of the keys and all of the rows; else, and at head size 256, they share the tiles and have 16 rows each.
// Bound by memory: K and V are read once for each block of rows.  32 users of 32 / 8 heads of 128 over 256 ... 4096 keys (170 MB) 34 us, of which the merge is four:
// 5.7 TB/s in the kernel; 64 users of 8 / 8 of 64 over 1500 (197 MB) 33.4, 5.9 TB/s; 96 of 64 / 8 of 128 over 512 ... 2048 (436 MB) 74, 5.9; shared, 96 of 64 / 8, 5 tokens, over
// 1500 (590 MB) 102, 5.8; 64 of 16 / 8 of 256 over 800 (419 MB) 68, 6.1.  Between, the chains of tiles do, 1.1 us a tile of 32 keys, or of 64 that are shared:
// 8 users of 32 / 8 over 1500 (49 MB) 13.2, 5 tokens of 64 / 8 16.0.  Tiles of TILE keys (64 at head size 64, else 32; shared 64, 32 at head size 256):
//   memory -> registers -> LDS    whole lines, a tile ahead of its use (shared: two); what lies behind the last key becomes zeros on the way (V) or is masked (K).  One
//                                 buffer takes K, then V: two workgroups share a CU.  (Three, with fewer registers, came to 5.0 TB/s: four wavefronts per SIMD ask for
//                                 more than the memory takes well.)
//   S^T = K . Q^T                 16x16x32 bfloat16; the tile is four runs of TILE / 4 keys, one per quad of lanes: row 4 j + r of block b is
//                                 key (TILE / 4) j + 4 b + r, so lane (row, quad) ends up with its quad's run in order, which is
//   O^T += V^T . P^T              the order in which the second product wants its weights: no moves between the two
// 8-bit caches: the same, an element becoming its bfloat16 value on its way into LDS; 32 users of 32 / 8 heads over 256 ... 4096 keys 23 us (34 with bfloat16), 96 of 64 / 8 over
// 512 ... 2048 51 (75), 64 of 16 / 8 of 256 over 800 42 (67), 96 of 64 / 8, 5 tokens, over 1500 70 (102), 8, 5 tokens, over 512 ... 5469 21 (23).  A piece of 16 elements goes to two chunks of LDS: banks
// that wait for each other are 25 ... 37 % of LDS's cycles, 0 with bfloat16.
// Statistics and accumulators are floats; weights are rounded once to bfloat16 for the matrix instruction, and the same rounded weights are summed.
// Wavefronts' results of their own tiles meet in LDS, the parts' in memory, merged by a kernel of its own.  How many parts there are goes by an estimate of the time, the host's of the longest
// user, or, where that is long enough to pay for it, the device's of all of them (cross_work).
#include "decode_mfma16_kernel.h"
#include "fp8.h"
#include "prefill_common.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

namespace ttpa {
namespace fp8 {
int expand_entries(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, void *k_copy, void *v_copy, int32_t *table,
                   const int32_t *page_table, int64_t page_table_row_stride, const void *lens, int lens_i64, int batch, int width, int kv_heads,
                   int block_size, int head_size, int num_blocks, hipStream_t st);
}

namespace decode {
namespace {

constexpr int kMostCrossParts = 64;  // of a segment's keys

struct CrossArgs {
  const uint16_t *q;
  uint16_t *out;
  int64_t q_bs, q_hs, q_ts, o_bs, o_hs, o_ts;
  const void *k, *v;
  const float *k_scales, *v_scales;  // of 8-bit caches: [num_blocks][hkv]
  const int32_t *pt;
  int64_t pt_rs;
  const void *lens;
  int lens_i64;
  int batch, hkv, g, s, bs, w, nb;
  float scale_log2e;
  uint32_t runs, runs_inv;  // runs of keys per block, and floor((2^32 - 1) / runs)
  int row_blocks, parts, share;  // share: keys of a part at least
  float *slots;  // [batch * hkv * row_blocks][parts]: ROWS * D values, ROWS maxima, ROWS sums
  // Several users: the parts go by their lengths, of which each workgroup makes the same plan (cross_work).  Slots are then [unit][row_blocks], and
  // firsts[u] = a user's first unit over hkv, and its parts.
  int2 *firsts;
  int units;             // most of them: (user, KV head, part)
  float slots_of_cus;    // workgroups of one round, one per CU, over row_blocks
  float step_us, two, merge_us;  // the estimate of cross_cut: a step of a workgroup, two on a CU, a unit's part of the merge
};

template <int D>
constexpr int cross_tile() {
  return D == 64 ? 64 : 32;
}
// LDS of a wavefront: a tile of K, then of V
template <int D>
constexpr int cross_lds_bytes() {
  return cross_tile<D>() * D * 2;
}
// Where a row's 16-byte chunks lie: chunk c at c ^ key(row).  K is read by 16 lanes of 16 rows (four of each run) at one chunk, V by 32 lanes of eight rows (four of
// each of two runs) at 32 bytes: rows of 256 bytes or more are every bank once or twice, two rows of 128 share that.
template <int D, int TILE>
__device__ __forceinline__ int cross_kkey(int row) {
  constexpr int RUN = TILE / 4;
  const int run = row / RUN & 3, r = row & 3;
  return D == 64 ? 2 * run + (r >> 1) : 4 * run + r;
}
template <int D, int TILE>
__device__ __forceinline__ int cross_vkey(int row) {
  constexpr int RUN = TILE / 4;
  const int run = row / RUN & 1, r = row & 3;
  return D == 64 ? 2 * ((r >> 1) + 2 * run) : 2 * (r + 4 * run);
}
// Parts of a user's keys, of a.share keys or more each.
__device__ __forceinline__ int cross_parts(const CrossArgs &a, int keys) { return max(1, min(a.parts, (keys + a.share - 1) / a.share)); }
template <int D, int ROWS>
constexpr int cross_slot_floats() {
  return ROWS * (D + 2);
}
// Keys of a user, of those that the table has room for.
__device__ __forceinline__ int cross_keys(const CrossArgs &a, int64_t length) { return (int)max(min(length, (int64_t)a.w * a.bs), (int64_t)0); }

// What a workgroup does: part `part` of `parts` of a user's keys for a KV head (part >= parts: nothing); the user's first unit over hkv.
struct CrossWork {
  int u, h, part, parts, keys, first;
};
// Steps of a part, of `total` steps of all users' keys per KV head, the longest user's `longest`: as many workgroups as CUs, twice as many, or one per user and KV head, by
// the least estimate.  At least total * hkv / (2 slots_of_cus), so that there are never more than 2 slots_of_cus + batch * hkv units.
__device__ __forceinline__ int cross_share(const CrossArgs &a, int total, int longest) {
  const float all = (float)total * (float)a.hkv, segments = (float)(a.batch * a.hkv), one = a.slots_of_cus;
  const auto cost = [&](float share, float units) {
    const float rounds = units / one;
    return share * a.step_us * (rounds <= 1.f ? 1.f : a.two * ceilf(0.5f * rounds));
  };
  float best = (float)longest, least = cost(best, segments);
#pragma unroll
  for (int k = 1; k <= 2; ++k) {
    const float room = (float)k * one, share = fmaxf(ceilf(all / fmaxf(room - 0.5f * segments, 0.5f * room)), 1.f);
    const float units = fminf(all / share + 0.5f * segments, room), c = cost(share, units) + units * a.merge_us + 1.f;
    if (share < best && c < least) best = share, least = c;
  }
  return max((int)best, (longest + kMostCrossParts - 1) / kMostCrossParts);
}
// The n-th unit by the users' lengths: user after user, a user's parts one after the other, KV heads fastest.  STEP keys are what a workgroup takes at a time.
template <int STEP>
__device__ __forceinline__ CrossWork cross_work(const CrossArgs &a, int n) {
  const int lane = (int)threadIdx.x & 63, x = n / a.hkv;
  const auto keys_of = [&](int u) { return u < a.batch ? cross_keys(a, load_index(a.lens, a.lens_i64, u)) : 0; };
  int keys = keys_of(lane), steps = (keys + STEP - 1) / STEP, total = steps, longest = steps;
  for (int u0 = 64; u0 < a.batch; u0 += 64) {
    const int more = (keys_of(u0 + lane) + STEP - 1) / STEP;
    total += more, longest = max(longest, more);
  }
  total = __builtin_amdgcn_readlane(wave_prefix_sum(total), 63), longest = (int)wave_max_u32((uint32_t)longest);
  const int share = max(cross_share(a, total, longest), 1);
  CrossWork w = {0, n - x * a.hkv, 0, 0, 0, 0};
  for (int u0 = 0, before = 0; u0 < a.batch; u0 += 64) {
    if (u0 > 0) keys = keys_of(u0 + lane), steps = (keys + STEP - 1) / STEP;
    const int mine = u0 + lane < a.batch ? max((steps + share - 1) / share, 1) : 0, upto = before + wave_prefix_sum(mine);
    const uint64_t behind = __builtin_amdgcn_ballot_w64(upto > x);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      w.u = u0 + l, w.parts = __builtin_amdgcn_readlane(mine, l), w.keys = __builtin_amdgcn_readlane(keys, l);
      w.first = __builtin_amdgcn_readlane(upto, l) - w.parts, w.part = x - w.first;
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return w;
}
// The plan for the merge, by one workgroup of a user (behind its loads: the compiler reads page tables by scalar loads only where no store comes before them.  By vector loads, which
// are waited for behind the tiles on their way, cross_shared_kernel took 4 of 26 us more).
__device__ __forceinline__ void cross_note(const CrossArgs &a, const CrossWork &w, int rb) {
  if (a.firsts && rb == 0 && w.part == 0 && w.h == 0 && threadIdx.x == 0) a.firsts[w.u] = make_int2(w.first, w.parts);
}
// The slot of a segment's first part.
__device__ __forceinline__ int64_t cross_slot(const CrossArgs &a, int u, int h, int rb, int first) {
  return a.firsts ? ((int64_t)first * a.hkv + h) * a.row_blocks + rb : ((int64_t)(u * a.hkv + h) * a.row_blocks + rb) * a.parts;
}

// Where a run of keys lies: its first byte, and its block and head.
struct CrossSpot {
  uint64_t at;
  uint32_t slab;
};
// A 16-byte piece of a row -> LDS: eight bfloat16 values as they are, or sixteen elements of an 8-bit cache as bfloat16 values, exactly (their block's scale is a power
// of two).  `key` swizzles the row's chunks.
template <bool FP8>
__device__ __forceinline__ void cross_put(uint8_t *row, int piece, int key, const u32x4 &x, float scale) {
  if constexpr (FP8) {
    *reinterpret_cast<u32x4 *>(row + ((2 * piece ^ key) << 4)) = __builtin_bit_cast(u32x4, fp8::decode8(x.x, x.y, scale));
    *reinterpret_cast<u32x4 *>(row + (((2 * piece + 1) ^ key) << 4)) = __builtin_bit_cast(u32x4, fp8::decode8(x.z, x.w, scale));
  } else {
    *reinterpret_cast<u32x4 *>(row + ((piece ^ key) << 4)) = x;
  }
}

// A wavefront's rows and what it has of the result; what it does with a tile of TILE keys that lies in LDS.
template <int D, int RG, int KEYS>
struct CrossRows {
  static constexpr int TILE = KEYS, RUN = TILE / 4, ROWS = 16 * RG;
  static constexpr int KBLK = TILE / 16, KSTEPS = D / 32, DBLK = D / 16, PSTEPS = TILE / 32;
  static constexpr int RB = 2 * D, CPR = D / 8;  // row bytes, 16-byte chunks of a row

  const CrossArgs &a;
  const int n, quad;
  int k_row, k_key, v_row, v_key;
  u32x4 qf[RG][KSTEPS];  // B operand of k-step i: lane (row n, quad) holds features 32 i + 8 quad + 0 .. 7
  floatx4 acc[RG][DBLK], l_acc[RG];
  float m_run[RG];

  __device__ __forceinline__ CrossRows(const CrossArgs &args) : a(args), n((int)(threadIdx.x & 15)), quad((int)(threadIdx.x & 63) >> 4) {
    // K operand: row RUN (n / 4) + 4 b + n % 4, chunk 4 i + quad (the key is that of every block's row: blocks are four rows apart)
    k_row = RUN * (n >> 2) + (n & 3), k_key = cross_kkey<D, TILE>(k_row);
    // V operand, transposed by the load: four rows x 16 features per quad; of step s and half t, row RUN quad + 8 s + 4 t + n / 4
    v_row = RUN * quad + (n >> 2), v_key = cross_vkey<D, TILE>(v_row);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
      for (int i = 0; i < DBLK; ++i) acc[rg][i] = floatx4{0.f, 0.f, 0.f, 0.f};
      l_acc[rg] = floatx4{0.f, 0.f, 0.f, 0.f}, m_run[rg] = -INFINITY;
    }
  }
  // The rows: row m is token m / g, head m % g of the group.
  __device__ __forceinline__ void load_q(int u, int h, int row0) {
    const int rows = a.g * a.s;
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      const int m = min(row0 + 16 * rg + n, rows - 1), token = m / a.g, head = m - token * a.g;  // (rows past the last: that one again, and not stored)
      const uint16_t *qp = a.q + u * a.q_bs + (int64_t)(h * a.g + head) * a.q_hs + token * a.q_ts + 8 * quad;
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) qf[rg][i] = *reinterpret_cast<const u32x4 *>(qp + 32 * i);
    }
  }
  // Where run x of the keys lies: a run is in one block.  (Ids out of range read block 0; tiles behind the table's room are not asked for.)
  template <bool FP8>
  __device__ __forceinline__ CrossSpot place(int u, int h, uint32_t x) const {
    constexpr int BYTES = FP8 ? D : RB;
    uint32_t col = __umulhi(x, a.runs_inv), r = x - col * a.runs;  // one too few at most
    if (r >= a.runs) ++col, r -= a.runs;
    const int page = (int)col < a.w ? a.pt[(int64_t)u * a.pt_rs + (int)col] : 0;
    const uint32_t slab = ((unsigned)page < (unsigned)a.nb ? (uint32_t)page : 0u) * (uint32_t)a.hkv + (uint32_t)h;  // (fewer than 2^32)
    return {slab * (uint64_t)(a.bs * BYTES) + r * (uint32_t)(RUN * BYTES), slab};
  }
  // (non-temporal also where several blocks of rows read the same keys: 96 users of 64 / 8 heads of 128 over 2033 keys 91 -> 74 us, and three blocks of 8 users
  // over 1500 20.8 -> 19.5)
  __device__ static __forceinline__ u32x4 load(const uint8_t *p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)); }
  // S^T = K . Q^T and the weights, rounded; of the lane's run, `nvalid` keys are attended.
  __device__ __forceinline__ void weigh(const uint8_t *tile, int nvalid, bool partial, u32x4 (&pf)[RG][PSTEPS]) {
    floatx4 st[RG][KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) st[rg][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(tile + (k_row + 4 * b) * RB + (((4 * i + quad) ^ k_key) << 4));
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) st[rg][b] = mma16<false>(w, qf[rg][i], st[rg][b]);
      }
    }
    // The weights' reference follows the maximum only where a score is more than 2^8 ahead of it: they stay below 2^8 with all their bits, and the accumulators are
    // rescaled in the first tile and hardly ever again.
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      float sc[4 * KBLK];
#pragma unroll
      for (int b = 0; b < KBLK; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[4 * b + r] = st[rg][b][r];
      if (partial) {
#pragma unroll
        for (int i = 0; i < 4 * KBLK; ++i) sc[i] = i >= nvalid ? -INFINITY : sc[i];
      }
      float mloc = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) mloc = fmaxf(mloc, sc[i]);
      mloc = max_over_quads(mloc * a.scale_log2e);
      if (__builtin_amdgcn_ballot_w64(mloc > m_run[rg] + 8.f) != 0) {
        const float m_new = fmaxf(m_run[rg], mloc);
        const float alpha = __builtin_amdgcn_exp2f(m_run[rg] - (m_new == -INFINITY ? 0.f : m_new));
        m_run[rg] = m_new;
#pragma unroll
        for (int i = 0; i < DBLK; ++i) acc[rg][i] *= alpha;
        l_acc[rg] *= alpha;
      }
      const float minus_m = m_run[rg] == -INFINITY ? 0.f : -m_run[rg];
#pragma unroll
      for (int i = 0; i < 4 * KBLK; i += 2)
        pf[rg][i >> 3][(i >> 1) & 3] = pack_bf16x2(__builtin_amdgcn_exp2f(fmaf(sc[i], a.scale_log2e, minus_m)), __builtin_amdgcn_exp2f(fmaf(sc[i + 1], a.scale_log2e, minus_m)));
    }
  }
  // O^T += V^T . P^T
  __device__ __forceinline__ void add(const uint8_t *tile, const u32x4 (&pf)[RG][PSTEPS]) {
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) shortx4 *lds_v4;
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) l_acc[rg] = mma16<false>(ones, pf[rg][s], l_acc[rg]);  // (the normaliser sums the weights that multiply V)
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const uint8_t *vp = tile + (v_row + 8 * s) * RB + (((2 * db + ((n & 3) >> 1)) ^ v_key) << 4) + 8 * (n & 1);
        const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vp)));
        const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vp + 4 * RB)));
        const u32x4 v = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) acc[rg][db] = mma16<false>(v, pf[rg][s], acc[rg][db]);
      }
    }
  }
};

// A wavefront with tiles of its own: on their way in registers, then in its share of LDS, K first and V over it.  A quad of lanes has a run of the keys.
template <int D, int RG, bool FP8>
struct CrossTile : CrossRows<D, RG, cross_tile<D>()> {
  using Rows = CrossRows<D, RG, cross_tile<D>()>;
  using Rows::TILE, Rows::RUN, Rows::RB, Rows::PSTEPS, Rows::a, Rows::n, Rows::quad, Rows::load;
  static constexpr int PPR = (FP8 ? D : 2 * D) / 16, NL = RUN * PPR / 16;  // 16-byte pieces of a row, loads of a tile and tensor
  uint8_t *const tile;
  u32x4 kraw[NL], vraw[NL];
  float k_scale, v_scale;  // of the tile on its way

  __device__ __forceinline__ CrossTile(const CrossArgs &args, uint8_t *lds) : Rows(args), tile(lds), k_scale(1.f), v_scale(1.f) {}
  __device__ __forceinline__ CrossSpot look_up(int u, int h, int t) const {
    CrossSpot s = this->template place<FP8>(u, h, (uint32_t)(t * 4 + quad));
    s.at += 16 * n;
    return s;
  }
  __device__ __forceinline__ void request_k(const CrossSpot &s) {
    const uint8_t *const kp = static_cast<const uint8_t *>(a.k) + s.at;
#pragma unroll
    for (int i = 0; i < NL; ++i) kraw[i] = load(kp + 256 * i);
    if constexpr (FP8) k_scale = a.k_scales[s.slab];
  }
  __device__ __forceinline__ void request_v(const CrossSpot &s) {
    const uint8_t *const vp = static_cast<const uint8_t *>(a.v) + s.at;
#pragma unroll
    for (int i = 0; i < NL; ++i) vraw[i] = load(vp + 256 * i);
    if constexpr (FP8) v_scale = a.v_scales[s.slab];
  }
  // Load i of a lane is piece 16 i + n of its run.
  __device__ __forceinline__ int run_row(int i) const { return (16 * i + n) / PPR; }
  // Registers -> LDS (an LDS works through a wavefront's instructions in order: V overwrites K behind the last read of K); of the lane's run, `nvalid` keys
  // are attended.
  __device__ __forceinline__ void stage_k() {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = RUN * quad + run_row(i);
      cross_put<FP8>(tile + row * RB, (16 * i + n) % PPR, cross_kkey<D, TILE>(row), kraw[i], k_scale);
    }
  }
  __device__ __forceinline__ void stage_v(int nvalid, bool partial) {
    if (partial) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const uint32_t keep = run_row(i) < nvalid ? 0xffffffffu : 0u;
        vraw[i] = u32x4{vraw[i].x & keep, vraw[i].y & keep, vraw[i].z & keep, vraw[i].w & keep};
      }
      v_scale = nvalid > 0 ? v_scale : 1.f;  // (of a block that holds nothing: anything)
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = RUN * quad + run_row(i);
      cross_put<FP8>(tile + row * RB, (16 * i + n) % PPR, cross_vkey<D, TILE>(row), vraw[i], v_scale);
    }
  }
  template <bool MORE>
  __device__ __forceinline__ void attend(int nvalid, bool partial, const CrossSpot &next) {
    u32x4 pf[RG][PSTEPS];
    stage_k();
    if constexpr (MORE) request_k(next);
    this->weigh(tile, nvalid, partial, pf);
    stage_v(nvalid, partial);
    if constexpr (MORE) request_v(next);
    this->add(tile, pf);
  }
};

// A workgroup per (user, KV head, block of rows): its wavefronts take the tiles in turn, and their results meet in LDS.
template <int D, int RG, bool FP8>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void cross_rows_kernel(CrossArgs a) {
  using T = CrossTile<D, RG, FP8>;
  constexpr int TILE = T::TILE, ROWS = T::ROWS, DBLK = T::DBLK, CPR = T::CPR;
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
  __shared__ float2 s_ml[4][ROWS];
  // workgroup -> (user, KV head) and block of rows, the blocks of one eight workgroups apart: on one XCD, which reads its keys once
  const uint32_t span = 8u * a.row_blocks, set = blockIdx.x / span, in_set = blockIdx.x - set * span;
  const int rb = (int)(in_set >> 3), unit = (int)(set * 8 + (in_set & 7)), segments = a.batch * a.hkv;
  if (unit >= (a.firsts ? a.units : segments * a.parts)) return;
  const int lane = threadIdx.x & 63, wib = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  CrossWork w;
  if (a.firsts) {
    w = cross_work<4 * TILE>(a, unit);
    if (w.part >= w.parts) return;
  } else {
    w.part = unit / segments, w.u = (unit - w.part * segments) / a.hkv, w.h = unit - w.part * segments - w.u * a.hkv;
  }
  const int u = __builtin_amdgcn_readfirstlane(w.u), h = __builtin_amdgcn_readfirstlane(w.h), part = __builtin_amdgcn_readfirstlane(w.part), rows = a.g * a.s, row0 = rb * ROWS;
  // (the first page and the rows are asked for beside the length)
  T x(a, tiles + wib * cross_lds_bytes<D>());
  int t = part * 4 + wib;
  const int64_t length = a.firsts ? w.keys : load_index(a.lens, a.lens_i64, u);
  const CrossSpot at0 = x.look_up(u, h, t);
  x.load_q(u, h, row0);
  const int keys = __builtin_amdgcn_readfirstlane(cross_keys(a, length)), n_tiles = (keys + TILE - 1) / TILE;
  const int parts = __builtin_amdgcn_readfirstlane(a.firsts ? w.parts : cross_parts(a, keys)), step = 4 * parts;
  if (part >= parts) return;
  if (keys == 0) {  // nothing to attend
    cross_note(a, w, rb);
#pragma unroll 1
    for (int i = threadIdx.x; i < min(ROWS, rows - row0) * CPR; i += 256) {
      const int m = row0 + i / CPR, token = m / a.g, head = m - token * a.g;
      uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 8 * (i % CPR);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(0u, 0u), *reinterpret_cast<uint2 *>(dst + 4) = make_uint2(0u, 0u);
    }
    return;
  }
  CrossSpot next = {0, 0};
  const auto process_tile = [&](auto more_tag) {
    constexpr bool more = decltype(more_tag)::value;
    const int nvalid = keys - (t * TILE + T::RUN * x.quad);
    const bool partial = (t + 1) * TILE > keys;
    const CrossSpot at = next;
    if constexpr (more) next = x.look_up(u, h, t + 2 * step);
    x.template attend<more>(nvalid, partial, at);
    t += step;
  };
  if (t < n_tiles) {
    next = x.look_up(u, h, t + step);
    x.request_k(at0), x.request_v(at0);
    while (t + step < n_tiles) process_tile(std::true_type{});
    process_tile(std::false_type{});
  }

  cross_note(a, w, rb);
  // ---- the wavefronts' results, a share of the features at a time (a wavefront's tiles hold that many) ------
  constexpr int FIT = cross_lds_bytes<D>() / (RG * 64 * 16);  // blocks of 16 features: 16 bytes per lane and group
  constexpr int BLOCKS = FIT >= 8 ? 8 : FIT >= 4 ? 4 : FIT >= 2 ? 2 : FIT;
  constexpr int SHARE = BLOCKS < DBLK ? BLOCKS : DBLK;
  static_assert(SHARE >= 1 && DBLK % SHARE == 0, "shares of whole blocks");
  if (lane < 16) {
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) s_ml[wib][16 * rg + lane] = make_float2(x.m_run[rg], x.l_acc[rg][0]);
  }
#pragma unroll
  for (int share = 0; share < DBLK / SHARE; ++share) {
    __syncthreads();  // (the tiles, or the share before, are done with)
#pragma unroll
    for (int b = 0; b < SHARE; ++b)
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const floatx4 &v = x.acc[rg][share * SHARE + b];
        *reinterpret_cast<float4 *>(x.tile + ((b * RG + rg) * 64 + lane) * 16) = make_float4(v[0], v[1], v[2], v[3]);
      }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < SHARE * RG * 64; i += 256) {
      const int b = i / (RG * 64), rg = i / 64 % RG, l = i & 63, row = 16 * rg + (l & 15), feature = 16 * (share * SHARE + b) + 4 * (l >> 4);
      const int m = row0 + row;
      if (m >= rows) continue;
      float mall = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mall = fmaxf(mall, s_ml[w][row].x);
      const float ref = merge_reference(mall);
      float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float wgt = __builtin_amdgcn_exp2f(s_ml[w][row].x - ref);
        const float4 v = *reinterpret_cast<const float4 *>(tiles + w * cross_lds_bytes<D>() + i * 16);
        num[0] = fmaf(wgt, v.x, num[0]), num[1] = fmaf(wgt, v.y, num[1]), num[2] = fmaf(wgt, v.z, num[2]), num[3] = fmaf(wgt, v.w, num[3]);
        den = fmaf(wgt, s_ml[w][row].y, den);
      }
      if (parts > 1) {
        float *const slot = a.slots + (a.firsts ? (int64_t)unit * a.row_blocks + rb : cross_slot(a, u, h, rb, 0) + part) * cross_slot_floats<D, ROWS>();
        *reinterpret_cast<float4 *>(slot + row * D + feature) = make_float4(num[0], num[1], num[2], num[3]);
        if (feature == 0) slot[ROWS * D + row] = mall, slot[ROWS * (D + 1) + row] = den;
        continue;
      }
      const int token = m / a.g, head = m - token * a.g;
      const float inv = 1.f / den;
      *reinterpret_cast<uint2 *>(a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + feature) =
          make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
    }
  }
}

// More rows: the four wavefronts have 16 rows each and share the tiles, of which each loads a run of the keys: two tiles on their way in registers, one in LDS,
// the next one written beside it, a barrier per tile.  (Two groups of rows per wavefront: 16 users of 32 / 8 heads over 1500 keys, 32 tokens, longer for every number of
// parts, as are 40 and 64 rows: a tile's time is the products' and the reads of LDS.)
template <int D>
constexpr int shared_tile() {
  return D == 256 ? 32 : 64;
}
template <int D, bool FP8>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void cross_shared_kernel(CrossArgs a) {
  using T = CrossRows<D, 1, shared_tile<D>()>;
  constexpr int TILE = T::TILE, RUN = T::RUN, RB = T::RB, CPR = T::CPR, ROWS = 64, DBLK = T::DBLK, BYTES = TILE * RB;
  constexpr int PPR = FP8 ? CPR / 2 : CPR, NL = RUN * PPR / 64;  // 16-byte pieces of a row, loads of a tile, wavefront and tensor
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];  // two of K and V
  const uint32_t span = 8u * a.row_blocks, set = blockIdx.x / span, in_set = blockIdx.x - set * span;
  const int rb = (int)(in_set >> 3), unit = (int)(set * 8 + (in_set & 7)), segments = a.batch * a.hkv;
  if (unit >= (a.firsts ? a.units : segments * a.parts)) return;
  const int lane = threadIdx.x & 63, wib = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  CrossWork w;
  if (a.firsts) {
    w = cross_work<TILE>(a, unit);
    if (w.part >= w.parts) return;
  } else {
    w.part = unit / segments, w.u = (unit - w.part * segments) / a.hkv, w.h = unit - w.part * segments - w.u * a.hkv;
  }
  const int u = __builtin_amdgcn_readfirstlane(w.u), h = __builtin_amdgcn_readfirstlane(w.h), part = __builtin_amdgcn_readfirstlane(w.part), rows = a.g * a.s, row0 = rb * ROWS + 16 * wib;
  const bool mine = row0 < rows;  // (a wavefront without rows loads its share of the keys)
  T x(a);
  int t = part;
  const auto look_up = [&](int tile) { return x.template place<FP8>(u, h, (uint32_t)(tile * 4 + wib)); };
  const int64_t length = a.firsts ? w.keys : load_index(a.lens, a.lens_i64, u);
  const CrossSpot at0 = look_up(t);
  if (mine) x.load_q(u, h, row0);
  const int keys = __builtin_amdgcn_readfirstlane(cross_keys(a, length)), n_tiles = (keys + TILE - 1) / TILE;
  const int parts = __builtin_amdgcn_readfirstlane(a.firsts ? w.parts : cross_parts(a, keys)), step = parts;
  if (part >= parts) return;
  if (keys == 0) {  // nothing to attend
    cross_note(a, w, rb);
#pragma unroll 1
    for (int i = threadIdx.x; i < min(ROWS, rows - rb * ROWS) * CPR; i += 256) {
      const int m = rb * ROWS + i / CPR, token = m / a.g, head = m - token * a.g;
      uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 8 * (i % CPR);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(0u, 0u), *reinterpret_cast<uint2 *>(dst + 4) = make_uint2(0u, 0u);
    }
    return;
  }
  struct Flight {  // a tile on its way
    u32x4 k[NL], v[NL];
    float k_scale, v_scale;
  };
  Flight flights[2];
  const auto request = [&](const CrossSpot &s, Flight &f) {
    const uint8_t *const kp = static_cast<const uint8_t *>(a.k) + s.at + 16 * lane, *const vp = static_cast<const uint8_t *>(a.v) + s.at + 16 * lane;
#pragma unroll
    for (int i = 0; i < NL; ++i) f.k[i] = T::load(kp + 1024 * i);
#pragma unroll
    for (int i = 0; i < NL; ++i) f.v[i] = T::load(vp + 1024 * i);
    f.k_scale = FP8 ? a.k_scales[s.slab] : 1.f, f.v_scale = FP8 ? a.v_scales[s.slab] : 1.f;
  };
  CrossSpot at2 = {0, 0};  // of the tile two steps ahead
  const auto process = [&](int buffer, Flight &f) {
    uint8_t *const kt = tiles + buffer * 2 * BYTES, *const vt = kt + BYTES;
    const bool partial = (t + 1) * TILE > keys;
    const CrossSpot at = at2;
    if (t + 3 * step < n_tiles) at2 = look_up(t + 3 * step);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = 64 * i + lane, row = RUN * wib + c / PPR;
      cross_put<FP8>(kt + row * RB, c % PPR, cross_kkey<D, TILE>(row), f.k[i], f.k_scale);
    }
    if (partial) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const uint32_t keep = t * TILE + RUN * wib + (64 * i + lane) / PPR < keys ? 0xffffffffu : 0u;
        f.v[i] = u32x4{f.v[i].x & keep, f.v[i].y & keep, f.v[i].z & keep, f.v[i].w & keep};
      }
      f.v_scale = t * TILE + RUN * wib < keys ? f.v_scale : 1.f;  // (of a block that holds nothing: anything)
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = 64 * i + lane, row = RUN * wib + c / PPR;
      cross_put<FP8>(vt + row * RB, c % PPR, cross_vkey<D, TILE>(row), f.v[i], f.v_scale);
    }
    if (t + 2 * step < n_tiles) request(at, f);
    __syncthreads();  // the tile is there; whoever is ahead writes the other buffer, whose tile everybody is done with
    if (mine) {
      u32x4 pf[1][T::PSTEPS];
      x.weigh(kt, keys - (t * TILE + RUN * x.quad), partial, pf);
      x.add(vt, pf);
    }
    t += step;
  };
  if (t < n_tiles) {
    CrossSpot at1 = {0, 0};
    if (t + step < n_tiles) at1 = look_up(t + step);
    if (t + 2 * step < n_tiles) at2 = look_up(t + 2 * step);
    request(at0, flights[0]);
    if (t + step < n_tiles) request(at1, flights[1]);
    while (t < n_tiles) {
      process(0, flights[0]);
      if (t < n_tiles) process(1, flights[1]);
    }
  }
  cross_note(a, w, rb);
  const int m = row0 + x.n, token = m / a.g, head = m - token * a.g;
  if (m >= rows) return;
  if (parts > 1) {
    float *const slot = a.slots + (a.firsts ? (int64_t)unit * a.row_blocks + rb : cross_slot(a, u, h, rb, 0) + part) * cross_slot_floats<D, ROWS>();
    const int row = m - rb * ROWS;
#pragma unroll
    for (int db = 0; db < DBLK; ++db) {
      const floatx4 &v = x.acc[0][db];
      *reinterpret_cast<float4 *>(slot + row * D + 16 * db + 4 * x.quad) = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (x.quad == 0) slot[ROWS * D + row] = x.m_run[0], slot[ROWS * (D + 1) + row] = x.l_acc[0][0];
    return;
  }
  const float inv = 1.f / x.l_acc[0][0];
  uint16_t *const dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 4 * x.quad;
#pragma unroll
  for (int db = 0; db < DBLK; ++db) {
    const floatx4 &v = x.acc[0][db];
    *reinterpret_cast<uint2 *>(dst + 16 * db) = make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
  }
}

// The parts of a segment's rows, four features per thread: a workgroup per row, 1024 / D slices of the parts (16, 8 and 4 at head sizes 64, 128 and 256) that meet in
// LDS, or several rows and all of a row's parts a thread's own (SLICES 1), where they are few.
template <int D, int ROWS, int SLICES>
__global__ __launch_bounds__(256) void cross_merge_kernel(CrossArgs a) {
  constexpr int SLOT = cross_slot_floats<D, ROWS>(), PER = D / 4, BATCH = SLICES > 1 ? 4 : 8, THREADS = SLICES > 1 ? SLICES * PER : 256;
  constexpr int AT_ONCE = THREADS / (PER * SLICES);  // rows of a workgroup
  const int slice = SLICES > 1 ? (int)threadIdx.x / PER : 0, f = threadIdx.x % PER;
  const int seg = blockIdx.x, m = blockIdx.y * AT_ONCE + (SLICES > 1 ? 0 : (int)threadIdx.x / PER), rb = m / ROWS, row = m - rb * ROWS;
  const int u = seg / a.hkv, h = seg - u * a.hkv, token = m / a.g, head = m - token * a.g;
  if (m >= a.g * a.s) return;
  uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 4 * f;
  const int64_t length = load_index(a.lens, a.lens_i64, u);
  int first = 0, count = a.parts;
  if (a.firsts) first = a.firsts[u].x, count = a.firsts[u].y;
  const float *slot = a.slots + cross_slot(a, u, h, rb, first) * SLOT;
  const int64_t behind = a.firsts ? (int64_t)a.hkv * a.row_blocks * SLOT : SLOT;
  float mv[BATCH], lv[BATCH];
  float4 v[BATCH];
  const auto fetch = [&](int p0) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (p0 + j * SLICES >= count) continue;
      const float *p = slot + (p0 + j * SLICES) * behind;
      v[j] = *reinterpret_cast<const float4 *>(p + row * D + 4 * f);
      mv[j] = p[ROWS * D + row], lv[j] = p[ROWS * (D + 1) + row];
    }
  };
  fetch(slice);  // (where they do not go by the plan, beside the length; parts that the user does not have hold anything, and are not used)
  if (!a.firsts) count = cross_parts(a, cross_keys(a, length));
  if (count == 1) return;  // (the one workgroup has written the output)
  float mall = -INFINITY, num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  for (int p0 = slice; p0 < count; p0 += SLICES * BATCH) {
    if (p0 != slice) fetch(p0);
    float m_new = mall;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) m_new = p0 + j * SLICES < count ? fmaxf(m_new, mv[j]) : m_new;
    const float ref = merge_reference(m_new), resc = __builtin_amdgcn_exp2f(mall - ref);
#pragma unroll
    for (int r = 0; r < 4; ++r) num[r] *= resc;
    den *= resc, mall = m_new;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (p0 + j * SLICES >= count) continue;
      const float wgt = __builtin_amdgcn_exp2f(mv[j] - ref);
      num[0] = fmaf(wgt, v[j].x, num[0]), num[1] = fmaf(wgt, v[j].y, num[1]), num[2] = fmaf(wgt, v[j].z, num[2]), num[3] = fmaf(wgt, v[j].w, num[3]);
      den = fmaf(wgt, lv[j], den);
    }
  }
  if constexpr (SLICES > 1) {
    __shared__ float4 s_num[SLICES][PER];
    __shared__ float2 s_md[SLICES];
    s_num[slice][f] = make_float4(num[0], num[1], num[2], num[3]);
    if (f == 0) s_md[slice] = make_float2(mall, den);
    __syncthreads();
    if (slice != 0) return;
    mall = -INFINITY, den = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) num[r] = 0.f;
    const int used = min(count, SLICES);
    for (int s = 0; s < used; ++s) mall = fmaxf(mall, s_md[s].x);
    const float ref = merge_reference(mall);
    for (int s = 0; s < used; ++s) {
      const float wgt = __builtin_amdgcn_exp2f(s_md[s].x - ref);
      const float4 v = s_num[s][f];
      num[0] = fmaf(wgt, v.x, num[0]), num[1] = fmaf(wgt, v.y, num[1]), num[2] = fmaf(wgt, v.z, num[2]), num[3] = fmaf(wgt, v.w, num[3]);
      den = fmaf(wgt, s_md[s].y, den);
    }
  }
  const float inv = 1.f / den;
  *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
}

// TTPA_CROSS_FORM=rows|planned|stream, read on every call.
bool form_is(const char *name) {
  const char *e = getenv("TTPA_CROSS_FORM");
  return e && !strcmp(e, name);
}

// How a call is cut: blocks of rows, and the groups of 16 that a wavefront has of one; parts of the keys and keys of a part.
// Wavefronts share their tiles from 33 rows on, where blocks of 32 would read the keys more than once, and at head size 256, where 32 rows are too many for a wavefront
// and tiles of its own leave room for one workgroup on a CU.  us per call, own tiles / shared, the best parts of each: 128, 8 users of 64 / 8 heads over 512 ... 5469 keys,
// 5 tokens 28.3 / 23.6; 96 over 1500 152 / 115; 32 of 32 / 8 over 800, 16 tokens 27.7 / 24.0; 16 over 1500, 32 tokens 37.7 / 33.9; one user over 1500, 7 tokens 9.8 / 9.4; 8, 16 tokens
// 17.0 / 17.6; 256, 16 / 8 heads, 8 over 1500, 48 tokens 62 / 38; 2 over 6404, 20 tokens 39.9 / 26.5, one 26.0 / 23.9; 64 over 800, one 71 / 71.  Up to 32 rows: 128, 32 users over
// 256 ... 4096, 4 rows 34.6 / 36.0; 96 over 512 ... 2048, 8 rows 74.8 / 83.5; 64 over 300, 32 rows 20.4 / 19.7; 64, 64 over 2015, 32 rows 25.5 / 31.2.
struct CrossCut {
  bool shared;
  int groups, row_blocks, parts, share, tile;
  int units;  // planned on the device: most of them; else 0
  double step_us, two, merge_us;
  int rows() const { return (shared ? 64 : 16) * groups; }
};

// The rule for the parts: the least of an estimate of the time, us behind what every launch needs, of a chain of tiles one after the other (a wavefront's, or a workgroup's
// that shares them).  Of full tables: rounds of workgroups, one per CU, or two that share its ways to memory; of ragged ones, of which three or four tenths are there:
// the longest chain, or all of them.  The two are weighed 7 : 3; with tiles of their own, chains of more than eight count more while the launch does not fill the chip; a
// split costs the merge.  Chosen / best of all: within 1 % over 28 shapes from 1 x 8 heads of 250 keys to 96 x 8 of 2033, 10 % at worst (8 x 8 of 512 ... 3597, 32
// rows); shared, 3 % over 31 from 1 x 8 of 100 to 96 x 8 of 1500, 14 % at worst (one user of 1500, 56 rows).
// Parts by the users' lengths: the host sees the longest alone, and a launch cut for tables as long as that leaves CUs to a few users' parts.  So where the estimate is 12 us or more, the
// device plans (cross_work), which costs each workgroup a round trip, 0.5 ... 0.7 us a call.  us per call, by the longest / planned: 64 / 8 heads of 128, 5 tokens, 8 users over 512 ... 5469 keys
// 26.5 / 22.0, seven over 200 and one over 6404 27.4 / 16.8, 32 over 256 ... 1983 35.1 / 31.0, 48 over 512 ... 6238 104 / 96, 8 over 1500 each (less than 12) 15.9 / 16.6; 32 / 8, 16
// over 100 ... 6976 40.4 / 25.7, 32 over 256 ... 3911 35.2 / 33.9; of 64, 16 over 512 ... 5918, 5 tokens 24.0 / 19.9; of 256, 64 / 8, 8 over 512 ... 3597, 8 tokens 39.6 / 32.8.
CrossCut cross_cut(int batch, int kv_heads, int64_t rows, int head_size, int64_t keys) {
  CrossCut c = {};
  c.shared = head_size == 256 || rows > 32;
  c.groups = c.shared || rows <= 16 ? 1 : 2;
  c.row_blocks = (int)((rows + c.rows() - 1) / c.rows());
  c.tile = c.shared ? (head_size == 256 ? shared_tile<256>() : shared_tile<128>()) : head_size == 64 ? cross_tile<64>() : cross_tile<128>();
  const double segments = (double)batch * kv_heads * c.row_blocks, cus = std::max(device_cus(), 1);
  const int tiles = (int)((keys + c.tile - 1) / c.tile), chains = c.shared ? 1 : 4;  // chains of a workgroup
  const double tile_us = c.shared ? (head_size == 64 ? 0.7 : head_size == 128 ? 1.05 : 0.95) : (head_size == 64 ? 1.2 : 1.1) * (c.groups == 2 ? 1.2 : 1.0);
  const double two = c.shared ? 1.7 : 1.9, there = c.shared ? 0.4 : 0.3;
  const double merged = c.shared ? segments * std::min<int64_t>(rows, 64) * 0.2e-3 : segments * 6.25e-3;
  double best = 0;
  for (int parts = 1; parts <= kMostCrossParts && (parts == 1 || chains * (parts - 1) < tiles); ++parts) {
    const int longest = (tiles + chains * parts - 1) / (chains * parts);
    if (parts > 1 && (tiles + chains * longest - 1) / (chains * longest) < parts) continue;  // (fewer parts are as short)
    const double all = segments * parts / cus, one = longest * tile_us, full = all <= 1 ? one : two * std::ceil(all / 2) * one;
    const double cost = 0.7 * full + 0.3 * std::max(one, there * all * one) + (!c.shared && segments < 2 * cus ? 0.2 * std::max(0, longest - 8) : 0.0) +
                        (parts > 1 ? 3.0 + parts * (merged + 0.02) : 0.0);
    if (c.parts == 0 || cost < best) best = cost, c.parts = parts;
  }
  c.parts = std::max(c.parts, 1);
  c.share = std::max((tiles + c.parts - 1) / c.parts, chains) * c.tile;
  // (the plan counts a user's steps in floats: up to 2^24 they are exact, and the room for units holds)
  if (c.parts > 1 && (best >= 12.0 || form_is("planned")) && batch > 1 && batch <= 1024 && tiles < (1 << 24) && (int64_t)batch * tiles < (1 << 30)) {
    c.units = (int)(2 * cus / c.row_blocks) + 1 + batch * kv_heads;
    c.step_us = tile_us, c.two = two, c.merge_us = (c.shared ? 1.75 * head_size / 128 : 1.0) * merged / (batch * kv_heads);
  }
  return c;
}
int64_t firsts_bytes(int batch) { return ((int64_t)batch * 8 + 255) & ~int64_t(255); }
int64_t cross_bytes(const CrossCut &c, int batch, int kv_heads, int head_size) {
  const int64_t slot = c.rows() * (int64_t)(head_size + 2) * 4;
  if (c.units) return firsts_bytes(batch) + (int64_t)c.units * c.row_blocks * slot;
  return c.parts == 1 ? 0 : (int64_t)batch * kv_heads * c.row_blocks * c.parts * slot;
}

template <int D, int RG, bool SHARED, bool FP8>
int launch_cross(const CrossArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> lds_ready{0};
  constexpr auto kernel = [] {
    if constexpr (SHARED) return &cross_shared_kernel<D, FP8>;
    else return &cross_rows_kernel<D, RG, FP8>;
  }();
  const size_t lds = SHARED ? 4 * shared_tile<D>() * D * 2 : 4 * cross_lds_bytes<D>();
  if (!ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds, lds_ready))
    return fail(TTPA_ERR_LAUNCH, "cross attention: cannot reserve %d bytes of LDS", (int)lds);
  const int64_t units = a.firsts ? a.units : (int64_t)a.batch * a.hkv * a.parts;
  launch_dominant(kernel, dim3((unsigned)((units + 7) / 8 * 8 * a.row_blocks)), dim3(256), lds, st, a);
  if (const int rc = check_launch("cross attention")) return rc;
  if (a.parts == 1) return TTPA_OK;
  // slices only for many parts: 2 / 3 / 4 parts of 64 rows, 8 users of 32 / 8 heads over 1500 keys 19.8 / 23.5 / 22.3 us with them, 17.0 / 20.5 / 19.5 without; 16 the same
  constexpr int ROWS = (SHARED ? 64 : 16) * RG, AT_ONCE = 1024 / D;
  if (a.firsts ? 2 * a.slots_of_cus > 16 * a.batch * a.hkv : a.parts > 16)
    cross_merge_kernel<D, ROWS, 1024 / D><<<dim3(a.batch * a.hkv, a.g * a.s), dim3(256), 0, st>>>(a);
  else
    cross_merge_kernel<D, ROWS, 1><<<dim3(a.batch * a.hkv, (a.g * a.s + AT_ONCE - 1) / AT_ONCE), dim3(256), 0, st>>>(a);
  return check_launch("cross attention (merge)");
}

template <int D, bool FP8>
int launch_cross_d(const CrossArgs &a, const CrossCut &c, hipStream_t st) {
  if constexpr (D < 256)
    if (!c.shared) return c.groups == 2 ? launch_cross<D, 2, false, FP8>(a, st) : launch_cross<D, 1, false, FP8>(a, st);
  return launch_cross<D, 1, true, FP8>(a, st);
}
template <bool FP8>
int launch_cross_any(const CrossArgs &a, int head_size, const CrossCut &c, hipStream_t st) {
  switch (head_size) {
    case 64: return launch_cross_d<64, FP8>(a, c, st);
    case 128: return launch_cross_d<128, FP8>(a, c, st);
    default: return launch_cross_d<256, FP8>(a, c, st);
  }
}

// The streaming loop's arguments.  It steps through rows by unsigned 32-bit numbers of bytes and through blocks by a 32-bit inverse; what does not fit those is
// the few rows' form's.
bool stream_args(const CrossArgs &c, int head_size, bool keys_known, int64_t keys, PrefillArgs &a) {
  for (const int64_t rows : {c.q_ts, c.o_ts})
    if (rows < 0 || rows >= (int64_t)1 << 31) return false;
  if ((int64_t)c.w * c.bs * c.bs >= (1ll << 32)) return false;
  a = {};
  a.out = c.out, a.out_bs = c.o_bs, a.out_hs = c.o_hs, a.out_ts = c.o_ts;
  a.q = c.q, a.q_bs = c.q_bs, a.q_hs = c.q_hs, a.q_ts = c.q_ts;
  a.k = static_cast<const uint16_t *>(c.k), a.v = static_cast<const uint16_t *>(c.v), a.pt = c.pt, a.pt_rs = c.pt_rs, a.lens = c.lens, a.lens_i64 = c.lens_i64;
  a.batch = c.batch, a.hq = c.hkv * c.g, a.hkv = c.hkv, a.sq = c.s, a.skv = c.w * c.bs, a.bs = c.bs, a.w = c.w, a.nb = c.nb;
  a.bs_magic = (uint32_t)((1ull << 32) / (uint32_t)c.bs) + 1u;
  a.scale_log2e = c.scale_log2e, a.parts = 1, a.stream = 1;
  a.cus = std::max(device_cus(), 1), a.keys_known = keys_known, a.keys_bound = keys;
  return true;
}

// Which form takes a call: the rows' where it reads the keys no more often than the streaming loop, which reads a key once for 128 rows, 32 tokens of four heads, whether
// there are as many or not; and while its workgroups have no more than 28 shared tiles per CU to go through (14 at head size 128, 10 at 256).  us per call, rows / stream (row
// blocks / groups of the loop per KV head, tiles per CU): 128, 32 / 8 heads, 8 users over 1500 keys, 16 tokens 18.4 / 22.8 (1 / 1), 32 (2 / 1, 12) 24.0 / 24.5, 48 (3 / 2, 18)
// 32.0 / 29.5, 128 46.7 / 34.3; 32 over 800, 16 tokens 24.2 / 29.4, 24 (2 / 1, 26) 31.8 / 26.0; 64 / 8 heads, 8 over 512 ... 5469, 16 tokens (2 / 2, 43) 32.3 / 45.3, 32 (4 / 2) 49.6 / 45.3;
// 64, 16 / 16 heads, 32 over 800, 64 tokens 23.0 / 27.9, 128 (2 / 1, 52) 37.0 / 31.1; 256, 16 / 8 heads, 2 over 6404, 32 tokens 29.6 / 37.2, 48 (2 / 1, 13) 42.5 / 39.5,
// 96 57 / 44.  Of 525 such pairs the rule takes the slower one, by more than 3 %, of 47: by 13 ... 18 % at most where all users are as long as the longest, which is what the host
// knows, and by 35 % where they are not and parts by their lengths would have paid (40 / 8 heads, 8 over 512 ... 5469, 48 tokens 49 / 66).
// 8-bit caches become bfloat16 copies for the streaming loop, so there both are estimated, us: 0.47 / 0.85 / 0.8 per 256 shared tiles behind 10, and the loop's products at 0.55 / 1.0 /
// 0.8 PFLOP/s, six bytes of copies per value at 6 TB/s and 17.  us per call, rows / copies (chosen so, but for *): 128, 32 / 8 heads, 8 users over 1500 keys, 48 tokens 32.7 / 50.3, 128
// 44.8 / 51.8, 256 82 / 72; 32 over 800, 64 53 / 65, 128 96 / 92 (*); 2 over 6404, 128 52 / 59, 512 157 / 131; of 64, 16 / 16, 4 over 1500, 447 29.6 / 46.0; of 256, 16 / 8, 8 over 1500, 96
// 63 / 73, 256 79 / 90; 2 over 1601 ... 4528, 2048 tokens 324 / 223.
// TTPA_CROSS_FORM overrides.
bool streams(const CrossArgs &c, const CrossCut &cut, int head_size, int64_t keys, bool fp8) {
  if (form_is("rows") || form_is("planned")) return false;
  if (form_is("stream")) return true;
  const int64_t tiles = (keys + cut.tile - 1) / cut.tile, row_blocks = (c.s + kRowsPerWave - 1) / kRowsPerWave;
  const int64_t groups = c.g % 4 == 0 ? c.g / 4 * row_blocks : (row_blocks * c.g + 3) / 4;  // workgroups of the streaming loop per KV head
  if (cut.row_blocks <= groups) return false;
  if (fp8) {
    const double segments = (double)c.batch * c.hkv, flops = 4.0 * segments * groups * 128 * keys * head_size;
    const double rows_us = 10 + (head_size == 64 ? 0.47 : head_size == 128 ? 0.85 : 0.8) * segments * cut.row_blocks * tiles / std::max(device_cus(), 1);
    return 17 + 6 * segments * keys * head_size / 6e6 + flops / (head_size == 64 ? 0.55e9 : head_size == 128 ? 1.0e9 : 0.8e9) < rows_us;
  }
  return (int64_t)c.batch * c.hkv * cut.row_blocks * tiles > (head_size == 64 ? 28 : head_size == 128 ? 14 : 10) * (int64_t)std::max(device_cus(), 1);
}

// Keys that the call is laid out for.
int64_t room_of(int block_size, int table_width, int64_t most_keys) {
  const int64_t room = (int64_t)block_size * table_width;
  return most_keys > 0 ? std::min(room, most_keys) : room;
}

// An 8-bit cache in the streaming loop: bfloat16 copies of the keys (exact), their table and the parts, in the workspace.
constexpr int64_t kMostCopies = int64_t(4) << 30;  // bytes of them: beyond, the rows' forms, which read the cache as it is
struct CrossCopies {
  int64_t copy, table;
  CrossCopies(const CrossArgs &c, int head_size)
      : copy(((int64_t)c.batch * c.w + 1) * c.hkv * c.bs * head_size * 2), table(((int64_t)c.batch * c.w * 4 + 255) & ~int64_t(255)) {}
  bool fit(const CrossArgs &c) const { return 2 * copy <= kMostCopies && c.hkv < 32768; }
  int64_t bytes() const { return 2 * copy + table; }
};

int64_t workspace_bytes(bool fp8, int batch, int q_heads, int kv_heads, int q_len, int head_size, int block_size, int table_width, int64_t most_keys) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_len <= 0 || head_size <= 0 || block_size <= 0 || table_width <= 0 || q_heads % kv_heads) return 0;
  const int64_t keys = room_of(block_size, table_width, most_keys);
  const CrossCut c = cross_cut(batch, kv_heads, (int64_t)(q_heads / kv_heads) * q_len, head_size, keys);
  int64_t bytes = cross_bytes(c, batch, kv_heads, head_size);
  // (strides are not known here: what either form may want)
  CrossArgs a = {};
  a.batch = batch, a.hkv = kv_heads, a.g = q_heads / kv_heads, a.s = q_len, a.bs = block_size, a.w = (int)((keys + block_size - 1) / block_size);
  PrefillArgs p;
  const CrossCopies copies(a, head_size);
  if ((head_size == 64 || head_size == 128 || head_size == 256) && streams(a, c, head_size, keys, fp8) && stream_args(a, head_size, most_keys > 0, keys, p) &&
      (!fp8 || copies.fit(a)))
    bytes = std::max(bytes, stream_ends_part_bytes(p, head_size) + (fp8 ? copies.bytes() : 0));
  return bytes;
}

int attend(CrossArgs &a, bool fp8, int head_size, int64_t table_width, float scale, int64_t most_keys, void *workspace, int64_t workspace_bytes, hipStream_t st) {
  const int batch = a.batch, kv_heads = a.hkv, block_size = a.bs;
  TTPA_REQUIRE(a.out && a.q && a.k && a.v && a.pt && a.lens && (!fp8 || (a.k_scales && a.v_scales)), "cross attention: null pointer argument");
  TTPA_REQUIRE(batch >= 0 && a.s >= 0 && a.g >= 0 && kv_heads > 0 && block_size > 0 && table_width > 0 && a.nb > 0, "cross attention: non-positive dimension");
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return fail(TTPA_ERR_UNSUPPORTED, "cross attention: head_size %d; supported 64, 128, 256", head_size);
  if (block_size % 32 || block_size > 4096)
    return fail(TTPA_ERR_UNSUPPORTED, "cross attention: block_size %d must be a multiple of 32 up to 4096", block_size);
  TTPA_REQUIRE(scale > 0.f, "cross attention: scale %g must be positive", (double)scale);
  TTPA_REQUIRE(most_keys >= 0, "cross attention: most_keys must not be negative");
  TTPA_REQUIRE(table_width * block_size < (1ll << 31) - 8192, "cross attention: a page-table row holds too many keys");
  TTPA_REQUIRE((int64_t)a.g * a.s < (1ll << 30) && (int64_t)a.nb * kv_heads < (1ll << 32), "cross attention: too many rows or blocks");
  TTPA_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out), "cross attention: operands must be 16-byte aligned");
  TTPA_REQUIRE(a.q_bs % 8 == 0 && a.q_hs % 8 == 0 && a.q_ts % 8 == 0 && a.o_bs % 4 == 0 && a.o_hs % 4 == 0 && a.o_ts % 4 == 0,
               "cross attention: strides must be multiples of 8 elements (out: 4)");
  if (batch == 0 || a.s == 0) return TTPA_OK;
  // (what a caller's bound excludes is not there)
  const int64_t keys = room_of(block_size, (int)table_width, most_keys);
  a.w = (int)((keys + block_size - 1) / block_size);
  a.scale_log2e = scale * 1.4426950408889634f;
  PrefillArgs p;
  const CrossCut c = cross_cut(batch, kv_heads, (int64_t)a.g * a.s, head_size, keys);
  const CrossCopies copies(a, head_size);
  if (streams(a, c, head_size, keys, fp8) && stream_args(a, head_size, most_keys > 0, keys, p) && (!fp8 || copies.fit(a))) {
    TTPA_REQUIRE((int64_t)batch * kv_heads * a.g * ((a.s + 31) / 32) < (1ll << 26), "cross attention: too many rows for one launch");
    char *ws = workspace && aligned16(workspace) ? static_cast<char *>(workspace) : nullptr;
    if (fp8) {
      if (!ws || workspace_bytes < copies.bytes())
        return fail(TTPA_ERR_WORKSPACE, "cross attention: needs %lld bytes of workspace, 16-byte aligned", (long long)copies.bytes());
      int32_t *const table = reinterpret_cast<int32_t *>(ws + 2 * copies.copy);
      if (const int rc = fp8::expand_entries(a.k, a.v, a.k_scales, a.v_scales, ws, ws + copies.copy, table, a.pt, a.pt_rs, a.lens, a.lens_i64, batch, a.w,
                                             kv_heads, block_size, head_size, a.nb, st))
        return rc;
      p.k = reinterpret_cast<uint16_t *>(ws), p.v = reinterpret_cast<uint16_t *>(ws + copies.copy), p.pt = table, p.pt_rs = a.w, p.nb = batch * a.w + 1;
      ws += copies.bytes(), workspace_bytes -= copies.bytes();
    }
    if (ws) p.part_acc = reinterpret_cast<float *>(ws), p.part_bytes = workspace_bytes;
    return launch_stream_ends(p, head_size, st);
  }
  a.row_blocks = c.row_blocks, a.parts = c.parts, a.share = c.share;
  a.runs = (uint32_t)block_size / (c.tile / 4), a.runs_inv = 0xffffffffu / a.runs;
  TTPA_REQUIRE(((int64_t)std::max(c.units, batch * kv_heads * c.parts) + 8) * c.row_blocks < (1ll << 24) && (c.parts == 1 || (int64_t)a.g * a.s < 65536),
               "cross attention: too many rows for one launch");
  const int64_t need = cross_bytes(c, batch, kv_heads, head_size);
  if (a.parts > 1 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(TTPA_ERR_WORKSPACE, "cross attention: needs %lld bytes of workspace, 16-byte aligned", (long long)need);
  a.slots = static_cast<float *>(workspace);
  if (c.units) {
    a.firsts = static_cast<int2 *>(workspace), a.slots = reinterpret_cast<float *>(static_cast<char *>(workspace) + firsts_bytes(batch));
    a.units = c.units, a.slots_of_cus = (float)std::max(device_cus(), 1) / (float)c.row_blocks;
    a.step_us = (float)c.step_us, a.two = (float)c.two, a.merge_us = (float)c.merge_us;
  }
  return fp8 ? launch_cross_any<true>(a, head_size, c, st) : launch_cross_any<false>(a, head_size, c, st);
}

}  // namespace
}  // namespace decode
}  // namespace ttpa

using namespace ttpa;

extern "C" int64_t ttpa_paged_cross_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                                              int32_t block_size, int32_t table_width, int64_t most_keys) {
  return decode::workspace_bytes(false, batch, q_heads, kv_heads, q_len, head_size, block_size, table_width, most_keys);
}

extern "C" int64_t ttpa_paged_fp8_cross_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                                                  int32_t block_size, int32_t table_width, int64_t most_keys) {
  return decode::workspace_bytes(true, batch, q_heads, kv_heads, q_len, head_size, block_size, table_width, most_keys);
}

#define TTPA_CROSS_ARGS                                                                                                                                  \
  TTPA_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, "cross attention: q_heads %d is not divisible by kv_heads %d", q_heads, kv_heads); \
  decode::CrossArgs a = {};                                                                                                                              \
  a.q = static_cast<const uint16_t *>(q), a.q_bs = q_batch_stride, a.q_hs = q_head_stride, a.q_ts = q_token_stride;                                      \
  a.out = static_cast<uint16_t *>(out), a.o_bs = out_batch_stride, a.o_hs = out_head_stride, a.o_ts = out_token_stride;                                  \
  a.k = k_cache, a.v = v_cache, a.pt = page_table, a.pt_rs = page_table_row_stride, a.lens = encoder_lens, a.lens_i64 = lens_is_i64;                     \
  a.batch = batch, a.hkv = kv_heads, a.g = q_heads / kv_heads, a.s = q_len, a.bs = block_size, a.nb = num_blocks

extern "C" int ttpa_paged_cross_attention(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q,
                                          int64_t q_batch_stride, int64_t q_head_stride, int64_t q_token_stride, const void *k_cache,
                                          const void *v_cache, const int32_t *page_table, int64_t page_table_row_stride, const void *encoder_lens,
                                          int lens_is_i64, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                          int32_t block_size, int32_t table_width, int32_t num_blocks, float scale, int64_t most_keys,
                                          void *workspace, int64_t workspace_bytes, void *stream) {
  TTPA_CROSS_ARGS;
  return decode::attend(a, false, head_size, table_width, scale, most_keys, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int ttpa_paged_fp8_cross_attention(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q,
                                              int64_t q_batch_stride, int64_t q_head_stride, int64_t q_token_stride, const void *k_cache,
                                              const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table,
                                              int64_t page_table_row_stride, const void *encoder_lens, int lens_is_i64, int32_t batch, int32_t q_heads,
                                              int32_t kv_heads, int32_t q_len, int32_t head_size, int32_t block_size, int32_t table_width,
                                              int32_t num_blocks, float scale, int64_t most_keys, void *workspace, int64_t workspace_bytes,
                                              void *stream) {
  TTPA_CROSS_ARGS;
  a.k_scales = k_scales, a.v_scales = v_scales;
  return decode::attend(a, true, head_size, table_width, scale, most_keys, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
