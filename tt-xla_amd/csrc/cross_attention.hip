// Attention of tokens to an encoder's states in a paged bfloat16 cache: a length per user, no causal limit.
//
//   out[u, h, t] = sum_j softmax_j(scale q[u, h, t] . k[u, j]) v[u, j],   j < len[u];   zeros where len[u] is 0
//
// This file holds the form for few rows (a token per user, a few drafted ones) and the choice; many rows are the streaming prefill loop's
// (prefill_stream_kernel.h, kEnds).  All tokens of a user see the same keys, so the rows of a KV
// head are its G query heads times the tokens, and a workgroup takes 16 RG of them over a part of the keys.
// Bound by memory: K and V are read once for each block of rows.  A wavefront takes every 4 parts-th tile of TILE keys (64 at head size 64, else 32):
//   memory -> registers -> LDS    whole lines, a tile ahead of its use; what lies behind the last key becomes zeros on the way (V) or is masked (K)
//   S^T = K . Q^T                 16x16x32 bfloat16; the tile is four runs of TILE / 4 keys, one per quad of lanes: row 4 j + r of block b is
//                                 key (TILE / 4) j + 4 b + r, so lane (row, quad) ends up with its quad's run in order, which is
//   O^T += V^T . P^T              the order in which the second product wants its weights: no moves between the two
// Statistics and accumulators are floats; weights are rounded once to bfloat16 for the matrix instruction, and the same rounded weights are summed.
// The four wavefronts' results meet in LDS, the parts' in memory, merged by a kernel of its own.
#include "decode_mfma16_kernel.h"
#include "prefill_common.h"

#include <algorithm>
#include <cstdlib>
#include <cstring>

namespace ttpa {
namespace decode {
namespace {

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
  int row_blocks, parts;
  float *slots;  // [batch * hkv * row_blocks][parts]: ROWS * D values, ROWS maxima, ROWS sums
};

template <int D>
constexpr int cross_tile() {
  return D == 64 ? 64 : 32;
}
// LDS of a wavefront: a tile of K and one of V
template <int D>
constexpr int cross_lds_bytes() {
  return cross_tile<D>() * D * 4;
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
template <int D, int RG>
constexpr int cross_slot_floats() {
  return 16 * RG * (D + 2);
}
// Workgroups of a CU, by the registers of one (and the LDS at head size 256).
template <int D, int RG>
constexpr int cross_per_cu() {
  return D == 64 || (D == 128 && RG <= 2) ? 2 : 1;
}
// Keys of a user, of those that the table has room for.
__device__ __forceinline__ int cross_keys(const CrossArgs &a, int u) {
  return (int)max(min(load_index(a.lens, a.lens_i64, u), (int64_t)a.w * a.bs), (int64_t)0);
}
// Parts of a user's keys: no more than there are tiles for their wavefronts.
template <int D>
__device__ __forceinline__ int cross_parts(const CrossArgs &a, int keys) {
  constexpr int TILE = cross_tile<D>();
  return max(1, min(a.parts, ((keys + TILE - 1) / TILE + 3) / 4));
}

template <int D, int RG>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(cross_per_cu<D, RG>(), 2))) void cross_rows_kernel(CrossArgs a) {
  constexpr int TILE = cross_tile<D>(), RUN = TILE / 4, ROWS = 16 * RG;
  constexpr int KBLK = TILE / 16, KSTEPS = D / 32, DBLK = D / 16, PSTEPS = TILE / 32;
  constexpr int RB = 2 * D, CPR = D / 8, NL = RUN * CPR / 16;  // row bytes, 16-byte chunks of a row, loads of a tile and tensor
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
  __shared__ float2 s_ml[4][ROWS];
  // workgroup -> (user, KV head, part) and block of rows, the blocks of one unit eight workgroups apart: on one XCD, which reads its keys once
  const uint32_t span = 8u * a.row_blocks, set = blockIdx.x / span, in_set = blockIdx.x - set * span;
  const int rb = (int)(in_set >> 3), unit = (int)(set * 8 + (in_set & 7));
  if (unit >= a.batch * a.hkv * a.parts) return;
  const int uh = unit / a.parts, part = unit - uh * a.parts, u = uh / a.hkv, h = uh - u * a.hkv;
  const int keys = __builtin_amdgcn_readfirstlane(cross_keys(a, u));
  const int n_tiles = (keys + TILE - 1) / TILE, parts = cross_parts<D>(a, keys);
  if (part >= parts) return;
  const int lane = threadIdx.x & 63, wib = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int rows = a.g * a.s, row0 = rb * ROWS;
  if (keys == 0) {  // nothing to attend
#pragma unroll 1
    for (int i = threadIdx.x; i < min(ROWS, rows - row0) * CPR; i += 256) {
      const int m = row0 + i / CPR, token = m / a.g, head = m - token * a.g;
      uint16_t *dst = a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + 8 * (i % CPR);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(0u, 0u), *reinterpret_cast<uint2 *>(dst + 4) = make_uint2(0u, 0u);
    }
    return;
  }

  // ---- the rows: row m is token m / g, head m % g of the group -----------------------------------------
  u32x4 qf[RG][KSTEPS];  // B operand of k-step i: lane (row n, quad) holds features 32 i + 8 quad + 0 .. 7
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    const int m = min(row0 + 16 * rg + n, rows - 1), token = m / a.g, head = m - token * a.g;  // (rows past the last: that one again, and not stored)
    const uint16_t *qp = a.q + u * a.q_bs + (int64_t)(h * a.g + head) * a.q_hs + token * a.q_ts + 8 * quad;
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) qf[rg][i] = *reinterpret_cast<const u32x4 *>(qp + 32 * i);
  }

  // ---- addresses ---------------------------------------------------------------------------------------
  // A run lies in one block; its quad of lanes looks up its page and loads its rows.  (Ids out of range read block 0; tiles behind the table's room are not
  // asked for.)
  auto look_up = [&](int t) {
    const uint32_t x = (uint32_t)(t * 4 + quad);
    uint32_t col = __umulhi(x, a.runs_inv), r = x - col * a.runs;  // one too few at most
    if (r >= a.runs) ++col, r -= a.runs;
    const int page = (int)col < a.w ? a.pt[(int64_t)u * a.pt_rs + (int)col] : 0;
    const uint64_t slab = (uint64_t)((unsigned)page < (unsigned)a.nb ? page : 0) * (uint32_t)a.hkv + (uint32_t)h;
    return slab * (uint64_t)(a.bs * RB) + r * (uint32_t)(RUN * RB) + 16 * n;
  };
  u32x4 kraw[NL], vraw[NL];
  auto request = [&](uint64_t at) {
    const uint8_t *const kp = reinterpret_cast<const uint8_t *>(a.k) + at, *const vp = reinterpret_cast<const uint8_t *>(a.v) + at;
#pragma unroll
    for (int i = 0; i < NL; ++i) kraw[i] = *reinterpret_cast<const u32x4 *>(kp + 256 * i);
#pragma unroll
    for (int i = 0; i < NL; ++i) vraw[i] = *reinterpret_cast<const u32x4 *>(vp + 256 * i);
  };
  uint8_t *const k_tile = tiles + wib * cross_lds_bytes<D>(), *const v_tile = k_tile + TILE * RB;
  // load i of a lane: chunk 16 i + n of its run
  const auto run_row = [&](int i) { return (16 * i + n) / CPR; };
  uint32_t kw[NL], vw[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = RUN * quad + run_row(i), chunk = (16 * i + n) % CPR;
    kw[i] = (uint32_t)(row * RB + ((chunk ^ cross_kkey<D>(row)) << 4));
    vw[i] = (uint32_t)(row * RB + ((chunk ^ cross_vkey<D>(row)) << 4));
  }
  // K operand: row RUN (n / 4) + 4 b + n % 4, chunk 4 i + quad (the key is that of every block's row: blocks are four rows apart)
  const int k_row = RUN * (n >> 2) + (n & 3), k_key = cross_kkey<D>(k_row);
  // V operand, transposed by the load: four rows x 16 features per quad; of step s and half t, row RUN quad + 8 s + 4 t + n / 4
  const int v_row = RUN * quad + (n >> 2), v_key = cross_vkey<D>(v_row);

  floatx4 acc[RG][DBLK], l_acc[RG];
  float m_run[RG];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
    for (int i = 0; i < DBLK; ++i) acc[rg][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    l_acc[rg] = floatx4{0.f, 0.f, 0.f, 0.f}, m_run[rg] = -INFINITY;
  }
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  // Tile t of the wavefront's, every 4 * parts-th from part * 4 + wib on; `next`: where the following one lies.
  int t = part * 4 + wib;
  const int step = 4 * parts;
  uint64_t next = 0;
  auto process_tile = [&](auto more_tag) {
    constexpr bool more = decltype(more_tag)::value;
    const int nvalid = keys - (t * TILE + RUN * quad);  // of the lane's run
    const bool partial = (t + 1) * TILE > keys;
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(k_tile + kw[i]) = kraw[i];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const uint32_t keep = !partial || run_row(i) < nvalid ? 0xffffffffu : 0u;
      *reinterpret_cast<u32x4 *>(v_tile + vw[i]) = u32x4{vraw[i].x & keep, vraw[i].y & keep, vraw[i].z & keep, vraw[i].w & keep};
    }
    if constexpr (more) {
      request(next);
      next = look_up(min(t + 2 * step, n_tiles - 1));
    }
    // ---- S^T = K . Q^T ----
    floatx4 st[RG][KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) st[rg][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(k_tile + (k_row + 4 * b) * RB + (((4 * i + quad) ^ k_key) << 4));
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
        for (int r = 0; r < 4; ++r) sc[4 * b + r] = st[rg][b][r] * a.scale_log2e;
      if (partial) {
#pragma unroll
        for (int i = 0; i < 4 * KBLK; ++i) sc[i] = i >= nvalid ? -INFINITY : sc[i];
      }
      float mloc = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) mloc = fmaxf(mloc, sc[i]);
      mloc = max_over_quads(mloc);
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
        pf[rg][i >> 3][(i >> 1) & 3] = pack_bf16x2(__builtin_amdgcn_exp2f(sc[i] + minus_m), __builtin_amdgcn_exp2f(sc[i + 1] + minus_m));
    }
    // ---- O^T += V^T . P^T ----
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) shortx4 *lds_v4;
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) l_acc[rg] = mma16<false>(ones, pf[rg][s], l_acc[rg]);
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const uint8_t *vp = v_tile + (v_row + 8 * s) * RB + (((2 * db + ((n & 3) >> 1)) ^ v_key) << 4) + 8 * (n & 1);
        const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vp)));
        const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vp + 4 * RB)));
        const u32x4 v = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) acc[rg][db] = mma16<false>(v, pf[rg][s], acc[rg][db]);
      }
    }
    t += step;
  };
  if (t < n_tiles) {
    request(look_up(t));
    next = look_up(min(t + step, n_tiles - 1));
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
    for (int rg = 0; rg < RG; ++rg) s_ml[wib][16 * rg + n] = make_float2(m_run[rg], l_acc[rg][0]);
  }
  float *const slot = a.slots + ((int64_t)(uh * a.row_blocks + rb) * a.parts + part) * cross_slot_floats<D, RG>();
#pragma unroll
  for (int share = 0; share < DBLK / SHARE; ++share) {
    __syncthreads();  // (the tiles, or the share before, are done with)
#pragma unroll
    for (int b = 0; b < SHARE; ++b)
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const floatx4 &x = acc[rg][share * SHARE + b];
        *reinterpret_cast<float4 *>(k_tile + ((b * RG + rg) * 64 + lane) * 16) = make_float4(x[0], x[1], x[2], x[3]);
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
        const float4 x = *reinterpret_cast<const float4 *>(tiles + w * cross_lds_bytes<D>() + i * 16);
        num[0] = fmaf(wgt, x.x, num[0]), num[1] = fmaf(wgt, x.y, num[1]), num[2] = fmaf(wgt, x.z, num[2]), num[3] = fmaf(wgt, x.w, num[3]);
        den = fmaf(wgt, s_ml[w][row].y, den);
      }
      if (parts == 1) {
        const int token = m / a.g, head = m - token * a.g;
        const float inv = 1.f / den;
        *reinterpret_cast<uint2 *>(a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + feature) =
            make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
      } else {
        *reinterpret_cast<float4 *>(slot + row * D + feature) = make_float4(num[0], num[1], num[2], num[3]);
        if (feature == 0) slot[ROWS * D + row] = mall, slot[ROWS * (D + 1) + row] = den;
      }
    }
  }
}

// The parts' results: a thread per four features of a row.
template <int D, int RG>
__global__ __launch_bounds__(256) void cross_merge_kernel(CrossArgs a) {
  constexpr int ROWS = 16 * RG, PER = D / 4, SLOT = cross_slot_floats<D, RG>();
  const int seg = blockIdx.x, uh = seg / a.row_blocks, rb = seg - uh * a.row_blocks, u = uh / a.hkv, h = uh - u * a.hkv;
  const int i = blockIdx.y * 256 + threadIdx.x, row = i / PER, feature = 4 * (i - row * PER);
  const int rows = a.g * a.s, m = rb * ROWS + row;
  if (row >= ROWS || m >= rows) return;
  const int parts = cross_parts<D>(a, cross_keys(a, u));
  if (parts == 1) return;  // (the one workgroup has written the output)
  const float *slot = a.slots + (int64_t)seg * a.parts * SLOT;
  float mall = -INFINITY, num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  constexpr int kBatch = 4;
  for (int p0 = 0; p0 < parts; p0 += kBatch) {
    float mv[kBatch], lv[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float *p = slot + (int64_t)min(p0 + j, parts - 1) * SLOT;
      x[j] = *reinterpret_cast<const float4 *>(p + row * D + feature);
      mv[j] = p[ROWS * D + row], lv[j] = p[ROWS * (D + 1) + row];
    }
    // (parts past the last, the last one again, have no share)
    float m_new = mall;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m_new = fmaxf(m_new, mv[j]);
    const float ref = merge_reference(m_new), resc = __builtin_amdgcn_exp2f(mall - ref);
#pragma unroll
    for (int r = 0; r < 4; ++r) num[r] *= resc;
    den *= resc, mall = m_new;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (p0 + j >= parts) continue;
      const float wgt = __builtin_amdgcn_exp2f(mv[j] - ref);
      num[0] = fmaf(wgt, x[j].x, num[0]), num[1] = fmaf(wgt, x[j].y, num[1]), num[2] = fmaf(wgt, x[j].z, num[2]), num[3] = fmaf(wgt, x[j].w, num[3]);
      den = fmaf(wgt, lv[j], den);
    }
  }
  const int token = m / a.g, head = m - token * a.g;
  const float inv = 1.f / den;
  *reinterpret_cast<uint2 *>(a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + feature) =
      make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
}

// What a call is cut into: groups of 16 rows per workgroup, blocks of rows, parts of the keys.
struct CrossCut {
  int groups, row_blocks, parts;
};
int tile_of(int head_size) { return head_size == 64 ? 64 : 32; }

CrossCut cross_cut(int batch, int kv_heads, int64_t rows, int head_size, int64_t keys) {
  CrossCut c;
  c.groups = rows <= 16 || head_size == 256 ? 1 : 2;  // (two at head size 256 spill)
  c.row_blocks = (int)((rows + 16 * c.groups - 1) / (16 * c.groups));
  // What counts is rounds of workgroups, each as long as a wavefront's tiles and about three more for its beginning and end.
  const int64_t segments = (int64_t)batch * kv_heads * c.row_blocks, tiles = (keys + tile_of(head_size) - 1) / tile_of(head_size);
  const int64_t at_once = (int64_t)std::max(device_cus(), 1) * (head_size == 256 ? 1 : 2);
  int64_t best = INT64_MAX;
  c.parts = 1;
  for (int64_t p = 1; p <= std::min<int64_t>(32, (tiles + 3) / 4); ++p) {
    const int64_t cost = (segments * p + at_once - 1) / at_once * ((tiles + 4 * p - 1) / (4 * p) + 3);
    if (cost < best) best = cost, c.parts = (int)p;
  }
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
  const int units = a.batch * a.hkv * a.parts;
  launch_dominant(&cross_rows_kernel<D, RG>, dim3((unsigned)((units + 7) / 8 * 8 * a.row_blocks)), dim3(256), lds, st, a);
  if (const int rc = check_launch("cross attention")) return rc;
  if (a.parts == 1) return TTPA_OK;
  cross_merge_kernel<D, RG><<<dim3(a.batch * a.hkv * a.row_blocks, (16 * RG * D / 4 + 255) / 256), dim3(256), 0, st>>>(a);
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

// Which form takes a call.  TTPA_CROSS_FORM=rows|stream, read on every call, overrides.
bool streams(const CrossArgs &c, int head_size, const PrefillArgs &a) {
  const char *e = getenv("TTPA_CROSS_FORM");
  if (e && (!strcmp(e, "rows") || !strcmp(e, "stream"))) return !strcmp(e, "stream");
  return c.s >= 32;
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
  if ((head_size == 64 || head_size == 128 || head_size == 256) && decode::stream_args(a, head_size, most_keys > 0, keys, p) && decode::streams(a, head_size, p))
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
  if (decode::stream_args(a, head_size, most_keys > 0, keys, p) && decode::streams(a, head_size, p)) {
    TTPA_REQUIRE((int64_t)batch * q_heads * ((q_len + 31) / 32) < (1ll << 26), "cross attention: too many rows for one launch");
    if (workspace && aligned16(workspace)) p.part_acc = static_cast<float *>(workspace), p.part_bytes = workspace_bytes;
    return launch_stream_ends(p, head_size, st);
  }
  const decode::CrossCut c = decode::cross_cut(batch, kv_heads, (int64_t)a.g * q_len, head_size, keys);
  a.row_blocks = c.row_blocks, a.parts = c.parts;
  TTPA_REQUIRE(((int64_t)batch * kv_heads * a.parts + 8) * a.row_blocks < (1ll << 24), "cross attention: too many rows for one launch");
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
