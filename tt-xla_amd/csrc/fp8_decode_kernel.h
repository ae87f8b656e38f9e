// Decode attention over the 8-bit cache (fp8.h) on the 16x16x32 bfloat16 matrix-core shape: one query token per user, up to 16 query heads per
// KV head, head sizes 64, 128 and 256.
//
// Bound by memory: an element is a byte, read once.  The work is cut as in the other decode kernels (decode_common.h: a flat list
// of tiles in equal ranges per wavefront, partial results, the merge kernel; or a workgroup per segment, DIRECT).
//
// Inside a wavefront a tile of TILE tokens (64; 32 at head size 256) is four runs of TILE / 4 consecutive tokens, one for
// each quad of lanes of a matrix-core operand, and a run lies in one block: its lanes look up its page and its two scales themselves, which takes no
// scalar registers and no loop over runs, and every block size that is a multiple of a run is the same code.
//   S^T block b (16 keys):  A = K rows, row 4 j + r is token (TILE / 4) j + 4 b + r; straight from global memory: the 16 bytes of a lane
//                           are 16 features, the operands of two k-steps, so lane (n, quad) holds features 64 i + 16 quad + 0 .. 15
//                           and Q's operand is laid out alike.  C: lane (head, quad) holds tokens (TILE / 4) quad + 4 b + r,
//                           a run in order: one scale per lane takes its keys to their values
//   O^T block db (16 d):    the 32 k slots of a step are the eight tokens of each quad's run in order, the probabilities the lane has
//                           already; A = V^T by the transposing LDS load of bytes (eight rows of a quad x 16 features)
// e4m3 elements become bfloat16 in registers, on their way into the matrix instructions: exactly, V's times its lane's scale in the same
// instruction (v_cvt_scalef32_pk_bf16_fp8), at two elements per instruction.
//
// V tile in LDS: rows of D bytes, 16-byte chunks at chunk ^ vkey(row), so that the 16 rows x 16 bytes that half a wavefront reads at once
// (8 rows of each of two quads) lie in different banks: 256 bytes are every bank once, so for D = 128 the eight rows of either
// parity need eight keys, for D = 64 the four rows of either residue four, for D = 256 sixteen.
//
// Pipeline per tile: V registers -> LDS | S^T (K's registers free) | request the next tile's V, K and scales, by pages requested one tile
// earlier | softmax | O^T.  A tile's data has a whole iteration to arrive, its pages another.
#pragma once
#include "decode_mfma16_kernel.h"
#include "fp8.h"

namespace ttpa {
namespace decode {
namespace {

struct Fp8Args {
  DecodeArgs d;
  const float *k_scales, *v_scales;
};

template <int D>
constexpr int fp8_tile() {
  return D <= 128 ? 64 : 32;
}
// LDS of a wavefront: the V tile, or the results it hands to the merge of a whole segment (merge_waves: 64 bytes per feature)
template <int D>
constexpr int fp8_lds_bytes() {
  return D * 64;
}
static_assert(fp8_tile<64>() * 64 <= fp8_lds_bytes<64>() && fp8_tile<128>() * 128 <= fp8_lds_bytes<128>() &&
                  fp8_tile<256>() * 256 <= fp8_lds_bytes<256>(), "the V tile fits");

template <int D>
__device__ __forceinline__ int fp8_vkey(int row) {
  if (D == 64) return ((row >> 2) & 1) | (((row >> 4) & 1) << 1);
  if (D == 128) return ((row >> 1) & 3) | (((row >> 4) & 1) << 2);
  return row & 15;
}

template <int D, int DIRECT>
__global__ __launch_bounds__(DIRECT ? kWave *DIRECT : 256) __attribute__((amdgpu_waves_per_eu(2, 8)))
void paged_decode_fp8_kernel(Fp8Args fa, const int32_t *__restrict__ page_table, const void *__restrict__ cur_pos) {
  const DecodeArgs &a = fa.d;
  constexpr int TILE = fp8_tile<D>(), RUN = TILE / 4;
  constexpr int KBLK = TILE / 16, KP = D / 64;  // score blocks; 16-byte pieces of a K row per lane
  constexpr int DBLK = D / 16, PSTEPS = TILE / 32;
  constexpr int CPR = D / 16;                   // 16-byte chunks of a row
  constexpr int RPL = 16 / CPR, NV = RUN / RPL;  // V: rows per load and quad of lanes, loads per tile
  __shared__ int s_pref[DIRECT ? 1 : kMaxUsers + 1];
  __shared__ int s_len[DIRECT ? 1 : kMaxUsers];
  __shared__ int s_wsum[kWavesPerBlock];
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];

  int seg_units = 0, n_ranges = a.n_waves;
  if constexpr (DIRECT == 0) seg_units = build_prefix_units<TILE, true>(a, cur_pos, s_pref, s_len, s_wsum, n_ranges);
  const int lane = threadIdx.x & 63;
  const int wib = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int wave = blockIdx.x * kWavesPerBlock + wib;
  int64_t total = 0, x = 0, x_hi = 0;
  int n_eff = 0, n_tiles = 0;
  Cursor cur;
  if constexpr (DIRECT > 0) {
    cur.u = (int)blockIdx.x / a.hkv;
    cur.h = (int)blockIdx.x - cur.u * a.hkv;
    n_tiles = tiles_of_user<TILE>(a, cur_pos, cur.u, cur.len);
    if (n_tiles == 0) {  // a padded row: NaN, like softmax over nothing
      const int g_all = a.hq / a.hkv;
      for (int i = threadIdx.x; i < g_all * D; i += kWave * DIRECT)
        a.out[cur.u * a.out_us + (int64_t)(cur.h * g_all + i / D) * a.out_hs + i % D] = 0x7fc0;
      return;
    }
    cur.lo = window_lo(a, cur.len);
    cur.t = cur.lo / TILE + wib;
    cur.tiles_left = n_tiles - wib;
  } else {
    const int total_units = __builtin_amdgcn_readfirstlane(s_pref[a.users]);
    const Share share = share_of(total_units, a.hkv, n_ranges, seg_units, wave);
    total = share.total, n_eff = share.n_eff;
    if (total == 0 || wave >= n_eff) {
      publish_segment_row(a, s_pref, total, n_eff, seg_units);
      return;
    }
    x_hi = share.hi;
    cur = locate_unit<TILE>(a, s_pref, s_len, share.lo, seg_units, &x);
  }
  uint8_t *tile = tiles + wib * fp8_lds_bytes<D>();
  const int G = a.hq / a.hkv;

  // ---- addresses -------------------------------------------------------------------------------
  // The block of the run that the lane's K rows lie in (run n / 4) or its V rows, scores and scales (run quad); ids out of
  // range read block 0.
  auto page_of = [&](const Cursor &cu, int run) {
    const int col = block_of(a, cu.t * TILE + run * RUN);
    return col < a.w ? page_table[(int64_t)cu.u * a.pt_rs + col] : 0;
  };
  auto row_of = [&](const Cursor &cu, int run) {
    const int tok = cu.t * TILE + run * RUN;
    return tok - block_of(a, tok) * a.bs;
  };
  auto slab_of = [&](int id, int h) { return (int64_t)((unsigned)id < (unsigned)a.nb ? id : 0) * a.hkv + h; };
  const int k_lane = n & 3, v_row = n / CPR, v_chunk = n % CPR;
  struct Pages {
    int k, v;
  };
  auto request_pages = [&](const Cursor &cu) { return Pages{page_of(cu, n >> 2), page_of(cu, quad)}; };

  u32x4 kraw[KBLK][KP], vraw[NV];
  float ks, vs;
  auto request = [&](const Cursor &cu, const Pages &pg) {
    const int64_t vslab = slab_of(pg.v, cu.h);
    const uint8_t *vp = a.v + (vslab * a.bs + row_of(cu, quad) + v_row) * D + 16 * v_chunk;
    const uint8_t *kp = a.k + (slab_of(pg.k, cu.h) * a.bs + row_of(cu, n >> 2) + k_lane) * D + 16 * quad;
#pragma unroll
    for (int i = 0; i < NV; ++i) vraw[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vp + i * RPL * D));
#pragma unroll
    for (int b = 0; b < KBLK; ++b)
#pragma unroll
      for (int i = 0; i < KP; ++i) kraw[b][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kp + 4 * b * D + 64 * i));
    ks = fa.k_scales[vslab], vs = fa.v_scales[vslab];
  };

  // Q: B operand of k-step 2 i + t: lane (head n, quad) holds features 64 i + 16 quad + 8 t + 0 .. 7 (zeros beyond G)
  u32x4 qf[2 * KP];
  auto load_q = [&](const Cursor &cu) {
    const uint16_t *qp = a.q + cu.u * a.q_us + (int64_t)(cu.h * G + min(n, G - 1)) * a.q_hs + 16 * quad;
    const uint32_t qmask = n < G ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i < KP; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint4 w = *reinterpret_cast<const uint4 *>(qp + 64 * i + 8 * t);
        qf[2 * i + t] = u32x4{w.x & qmask, w.y & qmask, w.z & qmask, w.w & qmask};
      }
  };
  // staging and transposing addresses of the V tile
  uint32_t vw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int row = RUN * quad + i * RPL + v_row;
    vw[i] = (uint32_t)(row * D + ((v_chunk ^ fp8_vkey<D>(row)) << 4));
  }
  uint32_t vr[PSTEPS];  // of chunk 0, and the key that goes with it
  int vkey[PSTEPS];
#pragma unroll
  for (int s = 0; s < PSTEPS; ++s) {
    const int row = RUN * quad + 8 * s + (n >> 1);
    vr[s] = (uint32_t)(row * D + 8 * (n & 1));
    vkey[s] = fp8_vkey<D>(row);
  }

  // ---- the walk over the list ------------------------------------------------------------------
  // The unit and cursor of the tile behind (cu, at); false: the range (or the wavefront's part of a segment) ends there.
  auto behind = [&](const Cursor &cu, int64_t at, Cursor &nx, int64_t &nx_at) {
    nx = cu;
    if constexpr (DIRECT > 0) {
      nx.t += DIRECT, nx.tiles_left -= DIRECT;
      return nx.tiles_left > 0;
    }
    const bool same = cu.tiles_left > 1;
    nx_at = at + (same ? 1 : 1 + seg_units);
    if (nx_at >= x_hi) return false;
    if (same) ++nx.t, --nx.tiles_left;
    else nx = locate_unit<TILE>(a, s_pref, s_len, at + 1, seg_units);
    return true;
  };

  const bool works = DIRECT == 0 || cur.tiles_left > 0;  // (a short segment leaves wavefronts without a tile)
  Cursor nxt = cur;
  int64_t x_nxt = x;
  bool more = false;
  Pages pages = {0, 0};
  if (works) {
    pages = request_pages(cur);
    load_q(cur);
    request(cur, pages);
    more = behind(cur, x, nxt, x_nxt);
    if (more) pages = request_pages(nxt);
  }
  if constexpr (DIRECT == 0) publish_segment_row(a, s_pref, total, n_eff, seg_units);

  floatx4 acc[DBLK];
#pragma unroll
  for (int i = 0; i < DBLK; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  while (works) {
    const int first = cur.t * TILE + RUN * quad;           // the lane's first position (scores, scales, V rows)
    const int nvalid = cur.len - first, nbelow = cur.lo - first;
    const bool partial = cur.len - cur.t * TILE < TILE || cur.lo > cur.t * TILE;
    // ---- V: registers -> LDS; rows that nobody attends (behind the last token, below a window) become zeros --------
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = i * RPL + v_row;
      const bool keep = !partial || (row < nvalid && row >= nbelow);
      *reinterpret_cast<u32x4 *>(tile + vw[i]) = keep ? vraw[i] : u32x4{0, 0, 0, 0};
    }
    const float kscale = ks * a.scale_log2e;
    const float vscale = !partial || (nvalid > 0 && nbelow < RUN) ? vs : 1.f;  // (of a run without a token: anything may stand there)
    // ---- S^T = K . Q^T ------------------------------------------------------------------------
    floatx4 st[KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b) {
      st[b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        st[b] = mma16<false>(fp8::decode8(kraw[b][i].x, kraw[b][i].y, 1.f), qf[2 * i], st[b]);
        st[b] = mma16<false>(fp8::decode8(kraw[b][i].z, kraw[b][i].w, 1.f), qf[2 * i + 1], st[b]);
      }
    }
    const Cursor done = cur;
    const bool last = !more, closes = DIRECT == 0 && (last || done.tiles_left <= 1);
    if (more) {
      cur = nxt, x = x_nxt;
      request(cur, pages);
      more = behind(cur, x, nxt, x_nxt);
      if (more) pages = request_pages(nxt);
    }
    // ---- online softmax -----------------------------------------------------------------------
    // (plain floats: with elements of the matrix results changed inside a branch the compiler wrote others of them, too, at head size 256)
    float sc[4 * KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[4 * b + r] = st[b][r] * kscale;
    if (partial) {
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) sc[i] = (i >= nvalid) | (i < nbelow) ? -INFINITY : sc[i];
    }
    float mloc = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * KBLK; ++i) mloc = fmaxf(mloc, sc[i]);
    mloc = max_over_quads(mloc);
    const float m_new = fmaxf(m_run, mloc);
    const float m_safe = (m_new == -INFINITY) ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_safe);
    m_run = m_new;
    float lsum = 0.f;
    u32x4 pf[PSTEPS];
#pragma unroll
    for (int b = 0; b < KBLK; ++b)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(sc[4 * b + r] - m_safe);
        const float p1 = __builtin_amdgcn_exp2f(sc[4 * b + r + 1] - m_safe);
        const uint32_t w = pack_bf16x2(p0, p1);
        lsum += bf16_lo(w) + bf16_hi(w);  // the normaliser sums the weights that multiply V
        pf[b >> 1][2 * (b & 1) + (r >> 1)] = w;
      }
    l_run = l_run * alpha + lsum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int i = 0; i < DBLK; ++i) acc[i] *= alpha;
    }
    // ---- O^T += V^T . P^T ---------------------------------------------------------------------
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s)
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        typedef int intx2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) intx2 *lds_v2;
        const intx2 t = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2)(tile + vr[s] + (uint32_t)((db ^ vkey[s]) << 4)));
        acc[db] = mma16<false>(fp8::decode8((uint32_t)t.x, (uint32_t)t.y, vscale), pf[s], acc[db]);
      }
    // ---- close the segment --------------------------------------------------------------------
    if (closes) {
      float *slot = a.ws_slots + ((int64_t)wave + (int64_t)done.u * a.hkv + done.h) * a.slot_floats;
      const float l_tot = sum_over_quads(l_run);
      if (n < G) {
        float *dst = slot + n * D + 4 * quad;
#pragma unroll
        for (int db = 0; db < DBLK; ++db) *reinterpret_cast<float4 *>(dst + 16 * db) = make_float4(acc[db][0], acc[db][1], acc[db][2], acc[db][3]);
        if (quad == 0) slot[G * D + n] = m_run, slot[G * D + G + n] = l_tot;
      }
      if (!last) {
#pragma unroll
        for (int i = 0; i < DBLK; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
        m_run = -INFINITY, l_run = 0.f;
        load_q(cur);
      }
    }
    if (last) break;
  }
  if constexpr (DIRECT > 0)
    merge_waves<D, DIRECT>(a, (int)blockIdx.x / a.hkv, (int)blockIdx.x % a.hkv, G, std::min(n_tiles, DIRECT), tile, tiles, fp8_lds_bytes<D>(), acc, 1.f,
                           m_run, sum_over_quads(l_run));
}

template <int D, int DIRECT>
bool launch_fp8_form(const Fp8Args &fa, hipStream_t st) {
  const DecodeArgs &a = fa.d;
  constexpr int kWaves = DIRECT ? DIRECT : kWavesPerBlock;
  const int blocks = DIRECT ? a.users * a.hkv : a.n_waves / kWavesPerBlock;
  const size_t lds = (size_t)kWaves * fp8_lds_bytes<D>();
  static std::atomic<uint64_t> lds_ready{0};
  const auto kernel = &paged_decode_fp8_kernel<D, DIRECT>;
  if (!ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds, lds_ready)) return false;
  launch_dominant(kernel, dim3(blocks), dim3(kWave * kWaves), lds, st, fa, a.pt, a.cur);
  return true;
}

template <int D>
bool launch_fp8(const Fp8Args &fa, hipStream_t st) {
  if (fa.d.direct == 4) return launch_fp8_form<D, 4>(fa, st);
  if constexpr (D <= 128)
    if (fa.d.direct == 8) return launch_fp8_form<D, 8>(fa, st);
  return launch_fp8_form<D, 0>(fa, st);
}

}  // namespace
}  // namespace decode
}  // namespace ttpa
