// Attention of tokens to an encoder's states in a paged bfloat16 cache: a length per user, no causal limit.
//
//   out[u, h, t] = sum_j softmax_j(scale q[u, h, t] . k[u, j]) v[u, j],   j < len[u];   zeros where len[u] is 0
//
// This file holds the form for few rows (a token per user, a few drafted ones) and the choice; many rows are the streaming prefill loop's
// (prefill_stream_kernel.h, kEnds).  All tokens of a user see the same keys, so the rows of a KV head are its G query heads times the tokens, and a workgroup takes
// 16 RG of them (RG 1 or 2) over a part of the keys.
// Bound by memory: K and V are read once for each block of rows.  32 users of 32 / 8 heads of 128 over 256 ... 4096 keys (170 MB) 35 us, of which the merge is four:
// 5.7 TB/s in the kernel; 64 users of 8 / 8 of 64 over 1500 (197 MB) 33.4, 5.9 TB/s; 96 of 64 / 8 of 128 over 512 ... 2048 (436 MB) 74, 5.9.  Between, the wavefronts' chains
// of tiles do, 1.1 us a tile: 8 users of 32 / 8 over 1500 (49 MB) 13.4.  A wavefront takes every 4 parts-th tile of TILE keys (64 at head size 64, else 32):
//   memory -> registers -> LDS    whole lines, a tile ahead of its use; what lies behind the last key becomes zeros on the way (V) or is masked (K).  One buffer
//                                 takes K, then V: two workgroups share a CU.  (Three, with fewer registers, came to 5.0 TB/s: four wavefronts per SIMD ask for more than
//                                 the memory takes well.)
//   S^T = K . Q^T                 16x16x32 bfloat16; the tile is four runs of TILE / 4 keys, one per quad of lanes: row 4 j + r of block b is
//                                 key (TILE / 4) j + 4 b + r, so lane (row, quad) ends up with its quad's run in order, which is
//   O^T += V^T . P^T              the order in which the second product wants its weights: no moves between the two
// Statistics and accumulators are floats; weights are rounded once to bfloat16 for the matrix instruction, and the same rounded weights are summed.
// The four wavefronts' results meet in LDS, the parts' in memory, merged by a kernel of its own.
#include "decode_mfma16_kernel.h"
#include "prefill_common.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

namespace ttpa {
namespace decode {
namespace {

constexpr int kMostCrossParts = 64;  // of a segment's keys

struct CrossArgs {
  const uint16_t *q;
  uint16_t *out;
  int64_t q_bs, q_hs, q_ts, o_bs, o_hs, o_ts;
  const uint16_t *k, *v;
  const int32_t *pt;
  int64_t pt_rs;
  const void *lens;
  int lens_i64;
  int batch, hkv, g, s, bs, w, nb;
  float scale_log2e;
  uint32_t runs, runs_inv;  // runs of keys per block, and floor((2^32 - 1) / runs)
  int row_blocks, parts, share;  // share: tiles of a part at least
  float *slots;  // [batch * hkv * row_blocks][parts]: ROWS * D values, ROWS maxima, ROWS sums
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
template <int D>
__device__ __forceinline__ int cross_kkey(int row) {
  constexpr int RUN = cross_tile<D>() / 4;
  const int run = row / RUN & 3, r = row & 3;
  return D == 64 ? 2 * run + (r >> 1) : 4 * run + r;
}
template <int D>
__device__ __forceinline__ int cross_vkey(int row) {
  constexpr int RUN = cross_tile<D>() / 4;
  const int run = row / RUN & 1, r = row & 3;
  return D == 64 ? 2 * ((r >> 1) + 2 * run) : 2 * (r + 4 * run);
}
// Parts of a user's keys, of a.share tiles or more each.
template <int D>
__device__ __forceinline__ int cross_parts(const CrossArgs &a, int keys) {
  constexpr int TILE = cross_tile<D>();
  return max(1, min(a.parts, ((keys + TILE - 1) / TILE + a.share - 1) / a.share));
}
template <int D, int RG>
constexpr int cross_slot_floats() {
  return 16 * RG * (D + 2);
}
// Workgroups of a CU, by the registers of one (and the LDS at head size 256).
template <int D, int RG>
constexpr int cross_per_cu() {
  return D == 256 ? 1 : 2;
}
// Keys of a user, of those that the table has room for.
__device__ __forceinline__ int cross_keys(const CrossArgs &a, int64_t length) { return (int)max(min(length, (int64_t)a.w * a.bs), (int64_t)0); }

// A wavefront's rows, its tile of keys and what it has of the result.
template <int D, int RG>
struct CrossTile {
  static constexpr int TILE = cross_tile<D>(), RUN = TILE / 4, ROWS = 16 * RG;
  static constexpr int KBLK = TILE / 16, KSTEPS = D / 32, DBLK = D / 16, PSTEPS = TILE / 32;
  static constexpr int RB = 2 * D, CPR = D / 8, NL = RUN * CPR / 16;  // row bytes, 16-byte chunks of a row, loads of a tile and tensor

  const CrossArgs &a;
  uint8_t *const tile;
  const int n, quad;
  int k_row, k_key, v_row, v_key;
  u32x4 qf[RG][KSTEPS];  // B operand of k-step i: lane (row n, quad) holds features 32 i + 8 quad + 0 .. 7
  u32x4 kraw[NL], vraw[NL];
  floatx4 acc[RG][DBLK], l_acc[RG];
  float m_run[RG];

  __device__ __forceinline__ CrossTile(const CrossArgs &args, uint8_t *lds)
      : a(args), tile(lds), n((int)(threadIdx.x & 15)), quad((int)(threadIdx.x & 63) >> 4) {
    // K operand: row RUN (n / 4) + 4 b + n % 4, chunk 4 i + quad (the key is that of every block's row: blocks are four rows apart)
    k_row = RUN * (n >> 2) + (n & 3), k_key = cross_kkey<D>(k_row);
    // V operand, transposed by the load: four rows x 16 features per quad; of step s and half t, row RUN quad + 8 s + 4 t + n / 4
    v_row = RUN * quad + (n >> 2), v_key = cross_vkey<D>(v_row);
    clear();
  }
  __device__ __forceinline__ void clear() {
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
  // Where the lane's run of tile t lies.  A run is in one block; its quad of lanes looks up its page and loads its rows.  (Ids out of range read block 0;
  // tiles behind the table's room are not asked for.)
  __device__ __forceinline__ uint64_t look_up(int u, int h, int t) const {
    const uint32_t x = (uint32_t)(t * 4 + quad);
    uint32_t col = __umulhi(x, a.runs_inv), r = x - col * a.runs;  // one too few at most
    if (r >= a.runs) ++col, r -= a.runs;
    const int page = (int)col < a.w ? a.pt[(int64_t)u * a.pt_rs + (int)col] : 0;
    const uint64_t slab = (uint64_t)((unsigned)page < (unsigned)a.nb ? page : 0) * (uint32_t)a.hkv + (uint32_t)h;
    return slab * (uint64_t)(a.bs * RB) + r * (uint32_t)(RUN * RB) + 16 * n;
  }
  // (non-temporal also where several blocks of rows read the same keys: 96 users of 64 / 8 heads of 128 over 2033 keys 91 -> 74 us, and three blocks of 8 users
  // over 1500 20.8 -> 19.5)
  __device__ static __forceinline__ u32x4 load(const uint8_t *p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)); }
  __device__ __forceinline__ void request_k(uint64_t at) {
    const uint8_t *const kp = reinterpret_cast<const uint8_t *>(a.k) + at;
#pragma unroll
    for (int i = 0; i < NL; ++i) kraw[i] = load(kp + 256 * i);
  }
  __device__ __forceinline__ void request_v(uint64_t at) {
    const uint8_t *const vp = reinterpret_cast<const uint8_t *>(a.v) + at;
#pragma unroll
    for (int i = 0; i < NL; ++i) vraw[i] = load(vp + 256 * i);
  }
  // Load i of a lane is chunk 16 i + n of its run.
  __device__ __forceinline__ int run_row(int i) const { return (16 * i + n) / CPR; }
  // Registers -> LDS (an LDS works through a wavefront's instructions in order: V overwrites K behind the last read of K); of the lane's run, `nvalid` keys
  // are attended.
  __device__ __forceinline__ void stage_k() {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = RUN * quad + run_row(i), chunk = (16 * i + n) % CPR;
      *reinterpret_cast<u32x4 *>(tile + row * RB + ((chunk ^ cross_kkey<D>(row)) << 4)) = kraw[i];
    }
  }
  __device__ __forceinline__ void stage_v(int nvalid, bool partial) {
    if (partial) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const uint32_t keep = run_row(i) < nvalid ? 0xffffffffu : 0u;
        vraw[i] = u32x4{vraw[i].x & keep, vraw[i].y & keep, vraw[i].z & keep, vraw[i].w & keep};
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = RUN * quad + run_row(i), chunk = (16 * i + n) % CPR;
      *reinterpret_cast<u32x4 *>(tile + row * RB + ((chunk ^ cross_vkey<D>(row)) << 4)) = vraw[i];
    }
  }
  template <bool MORE>
  __device__ __forceinline__ void attend(int nvalid, bool partial, uint64_t next) {
    stage_k();
    if constexpr (MORE) request_k(next);
    // ---- S^T = K . Q^T ----
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
    // ---- online softmax.  The weights' reference follows the maximum only where a score is more than 2^8 ahead of it: they stay below 2^8 with
    // all their bits, and the accumulators are rescaled in the first tile and hardly ever again. ----
    u32x4 pf[RG][PSTEPS];
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
    stage_v(nvalid, partial);
    if constexpr (MORE) request_v(next);
    // ---- O^T += V^T . P^T ----
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

// A workgroup per (user, KV head, block of rows): its wavefronts take the tiles in turn, and their results meet in LDS.
template <int D, int RG>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(cross_per_cu<D, RG>(), cross_per_cu<D, RG>()))) void cross_rows_kernel(CrossArgs a) {
  using T = CrossTile<D, RG>;
  constexpr int TILE = T::TILE, ROWS = T::ROWS, DBLK = T::DBLK, CPR = T::CPR;
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
  __shared__ float2 s_ml[4][ROWS];
  // workgroup -> (user, KV head) and block of rows, the blocks of one eight workgroups apart: on one XCD, which reads its keys once
  const uint32_t span = 8u * a.row_blocks, set = blockIdx.x / span, in_set = blockIdx.x - set * span;
  const int rb = (int)(in_set >> 3), unit = (int)(set * 8 + (in_set & 7)), segments = a.batch * a.hkv;
  if (unit >= segments * a.parts) return;
  const int part = unit / segments, uh = unit - part * segments, u = uh / a.hkv, h = uh - u * a.hkv;
  const int lane = threadIdx.x & 63, wib = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int rows = a.g * a.s, row0 = rb * ROWS;
  // (the first page and the rows are asked for beside the length)
  T x(a, tiles + wib * cross_lds_bytes<D>());
  int t = part * 4 + wib;
  const int64_t length = load_index(a.lens, a.lens_i64, u);
  const uint64_t at0 = x.look_up(u, h, t);
  x.load_q(u, h, row0);
  const int keys = __builtin_amdgcn_readfirstlane(cross_keys(a, length)), n_tiles = (keys + TILE - 1) / TILE;
  const int parts = cross_parts<D>(a, keys), step = 4 * parts;
  if (part >= parts) return;
  if (keys == 0) {  // nothing to attend
#pragma unroll 1
    for (int i = threadIdx.x; i < min(ROWS, rows - row0) * CPR; i += 256) {
      const int m = row0 + i / CPR, token = m / a.g, head = m - token * a.g;
      uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 8 * (i % CPR);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(0u, 0u), *reinterpret_cast<uint2 *>(dst + 4) = make_uint2(0u, 0u);
    }
    return;
  }
  uint64_t next = 0;
  const auto process_tile = [&](auto more_tag) {
    constexpr bool more = decltype(more_tag)::value;
    const int nvalid = keys - (t * TILE + T::RUN * x.quad);
    const bool partial = (t + 1) * TILE > keys;
    const uint64_t at = next;
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
        float *const slot = a.slots + ((int64_t)(uh * a.row_blocks + rb) * a.parts + part) * cross_slot_floats<D, RG>();
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

// The wavefronts' shares of a segment: a workgroup per row, eight slices of the shares that meet in LDS; four features per thread.
template <int D, int RG>
__global__ __launch_bounds__(2 * D) void cross_merge_kernel(CrossArgs a) {
  constexpr int ROWS = 16 * RG, SLOT = cross_slot_floats<D, RG>(), PER = D / 4, SLICES = 8, BATCH = 4;
  __shared__ float4 s_num[SLICES][PER];
  __shared__ float2 s_md[SLICES];
  const int seg = blockIdx.x, m = blockIdx.y, rb = m / ROWS, row = m - rb * ROWS;
  const int slice = threadIdx.x / PER, f = threadIdx.x - slice * PER;
  const int u = seg / a.hkv, h = seg - u * a.hkv, token = m / a.g, head = m - token * a.g;
  const int count = cross_parts<D>(a, cross_keys(a, load_index(a.lens, a.lens_i64, u)));
  if (count == 1) return;  // (the one workgroup has written the output)
  uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 4 * f;
  const float *slot = a.slots + (int64_t)(seg * a.row_blocks + rb) * a.parts * SLOT;
  float mall = -INFINITY, num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  for (int p0 = slice; p0 < count; p0 += SLICES * BATCH) {
    float mv[BATCH], lv[BATCH];
    float4 v[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const float *p = slot + (int64_t)min(p0 + j * SLICES, count - 1) * SLOT;
      v[j] = *reinterpret_cast<const float4 *>(p + row * D + 4 * f);
      mv[j] = p[ROWS * D + row], lv[j] = p[ROWS * (D + 1) + row];
    }
    // (shares past the last, the last one again, do not count)
    float m_new = mall;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) m_new = fmaxf(m_new, mv[j]);
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
  const float inv = 1.f / den;
  *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
}

// How the rows form cuts a call: groups of 16 rows per wavefront, blocks of rows, parts of the keys and tiles of a part.
struct CrossCut {
  int groups, row_blocks, parts, share;
};
int tile_of(int head_size) { return head_size == 64 ? 64 : 32; }

// The rule for the parts: the least of an estimate of the time, us behind what every launch needs, of a wavefront's tiles one after the other.  Of full tables: rounds of
// workgroups, one per CU, or two that share its ways to memory (1.9 times as long for both); of ragged ones, of which three tenths are there: the longest
// wavefront, or all of them.  The two are weighed 7 : 3; chains of more than eight tiles count more while the launch does not fill the chip; a split costs the merge.
// Chosen / best of all: within 1 % over 28 shapes from 1 x 8 heads of 250 keys to 96 x 8 of 2033, 16 % at worst (8 users of 512 ... 6404 keys, 40 rows).
CrossCut cross_cut(int batch, int kv_heads, int64_t rows, int head_size, int64_t keys) {
  CrossCut c;
  c.groups = rows <= 16 || head_size == 256 ? 1 : 2;  // (two at head size 256 spill)
  c.row_blocks = (int)((rows + 16 * c.groups - 1) / (16 * c.groups));
  const double segments = (double)batch * kv_heads * c.row_blocks, cus = std::max(device_cus(), 1);
  const int tiles = (int)((keys + tile_of(head_size) - 1) / tile_of(head_size));
  const double tile_us = (head_size == 64 ? 1.2 : head_size == 128 ? 1.1 : 2.3) * (c.groups == 2 ? 1.2 : 1.0);
  double best = 0;
  c.parts = 0;
  for (int chain = (tiles + 3) / 4; chain >= 1; --chain) {
    const int parts = std::max(1, (tiles + 4 * chain - 1) / (4 * chain));
    if (parts == c.parts) continue;  // (as many parts of fewer tiles: the same)
    if (parts > kMostCrossParts) break;
    const int longest = (tiles + 4 * parts - 1) / (4 * parts);
    const double groups = segments * parts, one = longest * tile_us, all = groups / cus;
    const double full = head_size == 256 ? std::ceil(all) * one : all <= 1 ? one : 1.9 * std::ceil(all / 2) * one;
    const double cost = 0.7 * full + 0.3 * std::max(one, 0.3 * all * one) + (segments < 2 * cus ? 0.2 * std::max(0, longest - 8) : 0.0) +
                        (parts > 1 ? 3.0 + parts * (0.4 * segments / 64 + 0.02) : 0.0);
    if (c.parts == 0 || cost < best) best = cost, c.parts = parts;
  }
  c.parts = std::max(c.parts, 1);
  c.share = std::max((tiles + c.parts - 1) / c.parts, 4);
  return c;
}
int64_t cross_bytes(const CrossCut &c, int batch, int kv_heads, int head_size) {
  return c.parts == 1 ? 256 : (int64_t)batch * kv_heads * c.row_blocks * c.parts * (16 * c.groups * (int64_t)(head_size + 2) * 4);
}

template <int D, int RG>
int launch_cross(const CrossArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> lds_ready{0};
  const size_t lds = 4 * cross_lds_bytes<D>();
  if (!ensure_dynamic_lds(reinterpret_cast<const void *>(&cross_rows_kernel<D, RG>), lds, lds_ready))
    return fail(TTPA_ERR_LAUNCH, "cross attention: cannot reserve %d bytes of LDS", (int)lds);
  const int64_t units = (int64_t)a.batch * a.hkv * a.parts;
  launch_dominant(&cross_rows_kernel<D, RG>, dim3((unsigned)((units + 7) / 8 * 8 * a.row_blocks)), dim3(256), lds, st, a);
  if (const int rc = check_launch("cross attention")) return rc;
  if (a.parts == 1) return TTPA_OK;
  cross_merge_kernel<D, RG><<<dim3(a.batch * a.hkv, a.g * a.s), dim3(2 * D), 0, st>>>(a);
  return check_launch("cross attention (merge)");
}

template <int D>
int launch_cross_d(const CrossArgs &a, int groups, hipStream_t st) {
  if constexpr (D < 256)
    if (groups == 2) return launch_cross<D, 2>(a, st);
  return launch_cross<D, 1>(a, st);
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
  a.k = c.k, a.v = c.v, a.pt = c.pt, a.pt_rs = c.pt_rs, a.lens = c.lens, a.lens_i64 = c.lens_i64;
  a.batch = c.batch, a.hq = c.hkv * c.g, a.hkv = c.hkv, a.sq = c.s, a.skv = c.w * c.bs, a.bs = c.bs, a.w = c.w, a.nb = c.nb;
  a.bs_magic = (uint32_t)((1ull << 32) / (uint32_t)c.bs) + 1u;
  a.scale_log2e = c.scale_log2e, a.parts = 1, a.stream = 1;
  a.cus = std::max(device_cus(), 1), a.keys_known = keys_known, a.keys_bound = keys;
  return true;
}

// Which form takes a call: the rows' where it reads every key once; while its blocks of rows have no more than 50 tiles of keys per CU to go through (25 of twice the
// bytes at head size 256); or no more than one and a half for each that the streaming loop has.  That reads a key once for 128 rows, 32 tokens of four heads, whether there
// are as many or not, and takes the rest.  us per call, rows / stream: 32 / 8 heads of 128, 8 users over 1500 keys, 1 token 13.4 / 22.2,
// 16 (24 tiles per CU) 19.4 / 22.6, 32 (47) 21.0 / 22.7, 48 (70) 33.2 / 29.4, 256 105 / 51; 2 users over 6404, 24 (38) 25.5 / 23.5, 48 (75) 35.3 / 28.1; 32 over 800, 8 (25)
// 21.6 / 25.1, 16 (50) 27.2 / 25.3, 32 (100) 44 / 26; 16 / 16 of 64, 8 over 1500, 96 (36) 20.7 / 21.8, 256 (96) 34 / 25; 16 / 8 of 256, 8 over 1500, 8 (12) 24.6 / 32.7,
// 16 (24) 37.6 / 33.0, 64 (94) 63 / 37; tokens that leave most of the streaming loop's rows empty: 64 / 8 of 128, 8 over 512 ... 5469, 5 (86) 31 / 45, 32 over 800, 8 (50)
// 27 / 38, 16 (100) 44 / 39.  TTPA_CROSS_FORM=rows|stream, read on every call, overrides.
bool streams(const CrossArgs &c, int head_size, int64_t keys) {
  const char *e = getenv("TTPA_CROSS_FORM");
  if (e && (!strcmp(e, "rows") || !strcmp(e, "stream"))) return !strcmp(e, "stream");
  const CrossCut cut = cross_cut(c.batch, c.hkv, (int64_t)c.g * c.s, head_size, keys);
  const int64_t tiles = (keys + tile_of(head_size) - 1) / tile_of(head_size), row_blocks = (c.s + kRowsPerWave - 1) / kRowsPerWave;
  const int64_t groups = c.g % 4 == 0 ? c.g / 4 * row_blocks : (row_blocks * c.g + 3) / 4;  // workgroups of the streaming loop per KV head
  if (cut.row_blocks == 1 || 2 * cut.row_blocks <= 3 * groups) return false;
  return (int64_t)c.batch * c.hkv * cut.row_blocks * tiles > (head_size == 256 ? 25 : 50) * (int64_t)std::max(device_cus(), 1);
}

// Keys that the call is laid out for.
int64_t room_of(int block_size, int table_width, int64_t most_keys) {
  const int64_t room = (int64_t)block_size * table_width;
  return most_keys > 0 ? std::min(room, most_keys) : room;
}

}  // namespace
}  // namespace decode
}  // namespace ttpa

using namespace ttpa;

extern "C" int64_t ttpa_paged_cross_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                                              int32_t block_size, int32_t table_width, int64_t most_keys) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_len <= 0 || head_size <= 0 || block_size <= 0 || table_width <= 0 || q_heads % kv_heads) return 0;
  const int64_t keys = decode::room_of(block_size, table_width, most_keys);
  const decode::CrossCut c = decode::cross_cut(batch, kv_heads, (int64_t)(q_heads / kv_heads) * q_len, head_size, keys);
  int64_t bytes = decode::cross_bytes(c, batch, kv_heads, head_size);
  // (strides are not known here: what either form may want)
  decode::CrossArgs a = {};
  a.batch = batch, a.hkv = kv_heads, a.g = q_heads / kv_heads, a.s = q_len, a.bs = block_size, a.w = (int)((keys + block_size - 1) / block_size);
  PrefillArgs p;
  if ((head_size == 64 || head_size == 128 || head_size == 256) && decode::stream_args(a, head_size, most_keys > 0, keys, p) && decode::streams(a, head_size, keys))
    bytes = std::max(bytes, stream_ends_part_bytes(p, head_size));
  return bytes;
}

extern "C" int ttpa_paged_cross_attention(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q,
                                          int64_t q_batch_stride, int64_t q_head_stride, int64_t q_token_stride, const void *k_cache,
                                          const void *v_cache, const int32_t *page_table, int64_t page_table_row_stride, const void *encoder_lens,
                                          int lens_is_i64, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                          int32_t block_size, int32_t table_width, int32_t num_blocks, float scale, int64_t most_keys,
                                          void *workspace, int64_t workspace_bytes, void *stream) {
  TTPA_REQUIRE(out && q && k_cache && v_cache && page_table && encoder_lens, "cross attention: null pointer argument");
  TTPA_REQUIRE(batch >= 0 && q_len >= 0 && q_heads > 0 && kv_heads > 0 && block_size > 0 && table_width > 0 && num_blocks > 0,
               "cross attention: non-positive dimension");
  TTPA_REQUIRE(q_heads % kv_heads == 0, "cross attention: q_heads %d is not divisible by kv_heads %d", q_heads, kv_heads);
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return fail(TTPA_ERR_UNSUPPORTED, "cross attention: head_size %d; supported 64, 128, 256", head_size);
  if (block_size % 32 || block_size > 4096)
    return fail(TTPA_ERR_UNSUPPORTED, "cross attention: block_size %d must be a multiple of 32 up to 4096", block_size);
  TTPA_REQUIRE(scale > 0.f, "cross attention: scale %g must be positive", (double)scale);
  TTPA_REQUIRE(most_keys >= 0, "cross attention: most_keys must not be negative");
  TTPA_REQUIRE((int64_t)table_width * block_size < (1ll << 31) - 8192, "cross attention: a page-table row holds too many keys");
  TTPA_REQUIRE((int64_t)q_heads / kv_heads * q_len < (1ll << 30), "cross attention: too many rows");
  TTPA_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out), "cross attention: operands must be 16-byte aligned");
  TTPA_REQUIRE(q_batch_stride % 8 == 0 && q_head_stride % 8 == 0 && q_token_stride % 8 == 0 && out_batch_stride % 4 == 0 && out_head_stride % 4 == 0 &&
                   out_token_stride % 4 == 0,
               "cross attention: strides must be multiples of 8 elements (out: 4)");
  if (batch == 0 || q_len == 0) return TTPA_OK;
  decode::CrossArgs a = {};
  a.q = static_cast<const uint16_t *>(q), a.q_bs = q_batch_stride, a.q_hs = q_head_stride, a.q_ts = q_token_stride;
  a.out = static_cast<uint16_t *>(out), a.o_bs = out_batch_stride, a.o_hs = out_head_stride, a.o_ts = out_token_stride;
  a.k = static_cast<const uint16_t *>(k_cache), a.v = static_cast<const uint16_t *>(v_cache);
  a.pt = page_table, a.pt_rs = page_table_row_stride, a.lens = encoder_lens, a.lens_i64 = lens_is_i64;
  a.batch = batch, a.hkv = kv_heads, a.g = q_heads / kv_heads, a.s = q_len, a.bs = block_size, a.nb = num_blocks;
  // (what a caller's bound excludes is not there)
  const int64_t keys = decode::room_of(block_size, table_width, most_keys);
  a.w = (int)((keys + block_size - 1) / block_size);
  a.scale_log2e = scale * 1.4426950408889634f;
  a.runs = (uint32_t)block_size / (decode::tile_of(head_size) / 4), a.runs_inv = 0xffffffffu / a.runs;
  hipStream_t st = static_cast<hipStream_t>(stream);
  PrefillArgs p;
  if (decode::stream_args(a, head_size, most_keys > 0, keys, p) && decode::streams(a, head_size, keys)) {
    TTPA_REQUIRE((int64_t)batch * q_heads * ((q_len + 31) / 32) < (1ll << 26), "cross attention: too many rows for one launch");
    if (workspace && aligned16(workspace)) p.part_acc = static_cast<float *>(workspace), p.part_bytes = workspace_bytes;
    return launch_stream_ends(p, head_size, st);
  }
  const decode::CrossCut c = decode::cross_cut(batch, kv_heads, (int64_t)a.g * q_len, head_size, keys);
  a.row_blocks = c.row_blocks, a.parts = c.parts, a.share = c.share;
  TTPA_REQUIRE(((int64_t)batch * kv_heads * c.parts + 8) * c.row_blocks < (1ll << 24) && (c.parts == 1 || (int64_t)a.g * q_len < 65536),
               "cross attention: too many rows for one launch");
  const int64_t need = decode::cross_bytes(c, batch, kv_heads, head_size);
  if (a.parts > 1 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(TTPA_ERR_WORKSPACE, "cross attention: needs %lld bytes of workspace, 16-byte aligned", (long long)need);
  a.slots = static_cast<float *>(workspace);
  switch (head_size) {
    case 64: return decode::launch_cross_d<64>(a, c.groups, st);
    case 128: return decode::launch_cross_d<128>(a, c.groups, st);
    default: return decode::launch_cross_d<256>(a, c.groups, st);
  }
}
