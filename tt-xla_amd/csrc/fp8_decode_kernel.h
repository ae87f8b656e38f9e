// Decode attention over the 8-bit cache (fp8.h) on the 16x16x32 bfloat16 matrix-core shape: one query token per user, up to 16 query heads per
// KV head, head sizes 64, 128 and 256.
//
// Bound by memory: an element is a byte, read once.  The work is cut as in the other decode kernels (decode_common.h: a flat list
// of tiles in equal ranges per wavefront, partial results, the merge kernel; or a workgroup per segment, DIRECT).
//
// Inside a wavefront a tile of TILE tokens (64; 32 at head size 256) is four runs of TILE / 4 consecutive tokens, one for
// each quad of lanes of a matrix-core operand, and a run lies in one block: its lanes look up its page and its two scales themselves, which takes no
// scalar registers and no loop over runs, and every block size that is a multiple of a run is the same code.
//   S^T block b (16 keys):  A = K rows, row 4 j + r is token (TILE / 4) j + 4 b + r; the 16 bytes that a lane reads are 16 features, the
//                           operands of two k-steps, so lane (n, quad) holds features 64 i + 16 quad + 0 .. 15 and Q's operand
//                           is laid out alike.  C: lane (head, quad) holds tokens (TILE / 4) quad + 4 b + r, a run in order: one scale
//                           per lane takes its keys to their values
//   O^T block db (16 d):    the 32 k slots of a step are the eight tokens of each quad's run in order, the probabilities the lane has
//                           already; A = V^T by the transposing LDS load of bytes (eight rows of a quad x 16 features)
// e4m3 elements become bfloat16 in registers, on their way into the matrix instructions: exactly, V's times its lane's scale in the same
// instruction (v_cvt_scalef32_pk_bf16_fp8), at two elements per instruction.
//
// K and V reach the matrix instructions through LDS, as bytes, for the sake of the loads: a non-temporal load that asks for half of a
// 128-byte line at a time streams 5.0 ... 6.1 TB/s on this card, whole lines 6.8 ... 7.1 (720 MB, three and four wavefronts per CU), and an operand of
// K straight from memory is half lines.  In LDS a row is D bytes, its 16-byte chunks at chunk ^ key(row): 256 bytes are every bank once, and the
// 16 rows that a read takes a chunk of at a time (K: four of each run; V: eight of each of two) need keys that differ as far as
// their rows lie in the same banks, eight keys for D = 128, four for 64, sixteen for 256.
//
// Pipeline per tile: registers -> LDS | request the next tile, by pages requested one tile earlier | S^T | softmax | O^T.  A tile's data
// has a whole iteration to arrive, its pages another.  Four wavefronts per CU, 16 KiB each on its way: 64 users with 1024 ... 16384 tokens of 64 / 8
// heads of 128 (727 MB) 130 us a pass, 5.8 TB/s in this kernel; 32 users with 512 ... 4096 of 32 / 8 (114 MB) 27.7.  (Steps to there: K's operand straight from
// memory and requests under a condition 157 and 32.8; no conditions 142 and 30.2.  Three wavefronts per CU 139 and 28.7, eight 129 and 28.9.)
#pragma once
#include "decode_mfma16_kernel.h"
#include "fp8.h"

namespace ttpa {
namespace decode {
namespace {

constexpr int kMostParts = 32;  // workgroups that share a segment
struct Fp8Args {
  DecodeArgs d;  // scale_log2e: its magnitude
  const float *k_scales, *v_scales;
  uint32_t negate;     // 0x80008000 where the scale is negative: the queries' signs are turned instead
  uint32_t runs, runs_inv;  // runs of tokens per block, and floor((2^32 - 1) / runs)
  // DIRECT: a segment's tiles are shared by `parts` workgroups; `arrived` [segments] counts those that have left their results, from zero
  int parts;
  int *arrived;
};

template <int D>
constexpr int fp8_tile() {
  return D <= 128 ? 64 : 32;
}
// LDS of a wavefront: a tile of K and one of V, or the results it hands to the merge of a whole segment (merge_waves: 64 bytes per feature)
template <int D>
constexpr int fp8_lds_bytes() {
  return fp8_tile<D>() * D * 2;
}
static_assert(fp8_lds_bytes<64>() >= 64 * 64 && fp8_lds_bytes<128>() >= 128 * 64 && fp8_lds_bytes<256>() >= 256 * 64, "the results fit");

template <int D>
__device__ __forceinline__ int fp8_vkey(int row) {
  if (D == 64) return ((row >> 2) & 1) | (((row >> 4) & 1) << 1);
  if (D == 128) return ((row >> 1) & 3) | (((row >> 4) & 1) << 2);
  return row & 15;
}

template <int D>
__device__ __forceinline__ int fp8_kkey(int row) {
  if (D == 64) return (row >> 4) & 3;
  if (D == 128) return 2 * ((row >> 4) & 3) + ((row >> 1) & 1);
  return 4 * ((row >> 3) & 3) + (row & 3);
}

// Stores and loads that pass by the XCD's own L2 copy, of values that a workgroup of another XCD reads or has written in the same launch.  (An
// acquire and release of all memory, which writes back and drops a whole L2 per workgroup, cost 10 us of a launch of 256.)
__device__ __forceinline__ void store_shared(float *p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float load_shared(const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The end of a segment that several workgroups have read: their wavefronts' results meet in LDS as in merge_waves, the workgroups' in memory
// (slots [segment][part]: G * D values, G maxima, G sums), and the workgroup that arrives last merges those of all, in their order.
template <int D, int WAVES>
__device__ __forceinline__ void merge_parts(const DecodeArgs &a, int seg, int G, int active, int part, int parts, int slots, int *arrived, uint8_t *own,
                                            const uint8_t *all, int pitch, const floatx4 (&acc)[D / 16], float m, float l) {
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, wib = threadIdx.x >> 6;
  if (wib < active) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *reinterpret_cast<float4 *>(own + db * 1024 + lane * 16) = make_float4(acc[db][0], acc[db][1], acc[db][2], acc[db][3]);
    if (lane < 16) s_m[wib][lane] = m, s_l[wib][lane] = l;
  }
  __syncthreads();
  float *const first = a.ws_slots + (int64_t)seg * slots * a.slot_floats, *const slot = first + (int64_t)part * a.slot_floats;
  const int gshift = G <= 1 ? 0 : 32 - __builtin_clz(G - 1);
  for (int i = threadIdx.x; i < (D / 4) << gshift; i += kWave * WAVES) {
    const int g = i & ((1 << gshift) - 1), d4 = i >> gshift;
    if (g >= G) continue;
    float mall = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < active) mall = fmaxf(mall, s_m[w][g]);
    const float ref = merge_reference(mall);
    float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < active) {
        const float wgt = __builtin_amdgcn_exp2f(s_m[w][g] - ref);
        const float4 x = *reinterpret_cast<const float4 *>(all + w * pitch + d4 * 256 + g * 16);
        num[0] = fmaf(wgt, x.x, num[0]), num[1] = fmaf(wgt, x.y, num[1]);
        num[2] = fmaf(wgt, x.z, num[2]), num[3] = fmaf(wgt, x.w, num[3]);
        den = fmaf(wgt, s_l[w][g], den);
      }
#pragma unroll
    for (int r = 0; r < 4; ++r) store_shared(slot + g * D + 4 * d4 + r, num[r]);
    if (d4 == 0) store_shared(slot + G * D + g, mall), store_shared(slot + G * D + G + g, den);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the thread's results have arrived where other XCDs see them
  __syncthreads();
  if (threadIdx.x == 0) s_last = __hip_atomic_fetch_add(arrived + seg, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
  __syncthreads();
  if (!s_last) return;
  // two round trips: every part's maxima and sums, then the values, eight parts at a time
  const int u = seg / a.hkv, h = seg - u * a.hkv;
  float *const s_w = reinterpret_cast<float *>(const_cast<uint8_t *>(all)), *const s_den = s_w + kMostParts * 16;  // (the tiles are done with)
  for (int i = threadIdx.x; i < parts * G; i += kWave * WAVES) {
    const int p = i / G, g = i - p * G;
    const float *sl = first + (int64_t)p * a.slot_floats + G * D + g;
    s_w[p * 16 + g] = load_shared(sl), s_den[p * 16 + g] = load_shared(sl + G);
  }
  __syncthreads();
  if (threadIdx.x < G) {
    const int g = threadIdx.x;
    float mall = -INFINITY, den = 0.f;
    for (int p = 0; p < parts; ++p) mall = fmaxf(mall, s_w[p * 16 + g]);
    const float ref = merge_reference(mall);
    for (int p = 0; p < parts; ++p) {
      const float wgt = __builtin_amdgcn_exp2f(s_w[p * 16 + g] - ref);
      s_w[p * 16 + g] = wgt, den = fmaf(wgt, s_den[p * 16 + g], den);
    }
    s_den[g] = den;
  }
  __syncthreads();
  for (int i = 2 * threadIdx.x; i < G * D; i += 2 * kWave * WAVES) {
    const int g = i / D;
    float num[2] = {0.f, 0.f};
    for (int p0 = 0; p0 < parts; p0 += 8) {
      uint64_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = __hip_atomic_load(reinterpret_cast<const uint64_t *>(first + (int64_t)min(p0 + j, parts - 1) * a.slot_floats + i), __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (p0 + j < parts) {
          const float wgt = s_w[(p0 + j) * 16 + g];
          num[0] = fmaf(wgt, __builtin_bit_cast(float, (uint32_t)v[j]), num[0]);
          num[1] = fmaf(wgt, __builtin_bit_cast(float, (uint32_t)(v[j] >> 32)), num[1]);
        }
    }
    uint16_t *dst = a.out + u * a.out_us + (int64_t)(h * G + g) * a.out_hs + (i - g * D);
    dst[0] = (uint16_t)f32_to_bf16_bits(num[0] / s_den[g]), dst[1] = (uint16_t)f32_to_bf16_bits(num[1] / s_den[g]);
  }
}

template <int D, int DIRECT>
__global__ __launch_bounds__(DIRECT ? kWave *DIRECT : 256) __attribute__((amdgpu_waves_per_eu(2, 8)))
void paged_decode_fp8_kernel(Fp8Args fa, const int32_t *__restrict__ page_table, const void *__restrict__ cur_pos) {
  const DecodeArgs &a = fa.d;
  constexpr int TILE = fp8_tile<D>(), RUN = TILE / 4;
  constexpr int KBLK = TILE / 16, KP = D / 64;  // score blocks; 16-byte pieces of a K row per lane
  constexpr int DBLK = D / 16, PSTEPS = TILE / 32;
  constexpr int CPR = D / 16;                   // 16-byte chunks of a row
  constexpr int RPL = 16 / CPR, NL = RUN / RPL;  // rows per load and quad of lanes, loads per tile and tensor
  __shared__ int s_wsum[kWavesPerBlock];
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
  // (the tables are as long as there are users: two workgroups share a CU's LDS)
  int *const s_pref = reinterpret_cast<int *>(tiles + kWavesPerBlock * fp8_lds_bytes<D>()), *const s_len = s_pref + a.users + 1;

  int seg_units = 0, n_ranges = a.n_waves;
  if constexpr (DIRECT == 0) seg_units = build_prefix_units<TILE, true>(a, cur_pos, s_pref, s_len, s_wsum, n_ranges);
  const int lane = threadIdx.x & 63;
  const int wib = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int wave = blockIdx.x * kWavesPerBlock + wib;
  int64_t total = 0, x = 0, x_hi = 0;
  int n_eff = 0, n_tiles = 0, seg = 0, part = 0, parts = 1;
  Cursor cur;
  if constexpr (DIRECT > 0) {
    seg = (int)blockIdx.x / fa.parts, part = (int)blockIdx.x - seg * fa.parts;
    cur.u = seg / a.hkv;
    cur.h = seg - cur.u * a.hkv;
    n_tiles = tiles_of_user<TILE>(a, cur_pos, cur.u, cur.len);
    parts = min(fa.parts, (n_tiles + DIRECT - 1) / DIRECT);
    if (part >= max(parts, 1)) return;
    if (n_tiles == 0) {  // a padded row: NaN, like softmax over nothing
      const int g_all = a.hq / a.hkv;
      for (int i = threadIdx.x; i < g_all * D; i += kWave * DIRECT)
        a.out[cur.u * a.out_us + (int64_t)(cur.h * g_all + i / D) * a.out_hs + i % D] = 0x7fc0;
      return;
    }
    cur.lo = window_lo(a, cur.len);
    cur.t = cur.lo / TILE + part * DIRECT + wib;
    cur.tiles_left = n_tiles - (part * DIRECT + wib);
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
  const int G = a.hq / a.hkv;

  // ---- addresses -------------------------------------------------------------------------------
  // Where the lane's run lies: its block (by the page table; ids out of range read block 0) and its first row there.  A quad of lanes
  // loads the rows of its run, whole rows per instruction, and holds its scores and scales.
  struct Run {
    int page;
    uint32_t row;
  };
  auto look_up = [&](const Cursor &cu) {
    const uint32_t x = (uint32_t)(cu.t * 4 + quad);
    uint32_t col = __umulhi(x, fa.runs_inv), r = x - col * fa.runs;  // one too few at most
    if (r >= fa.runs) ++col, r -= fa.runs;
    return Run{(int)col < a.w ? page_table[(int64_t)cu.u * a.pt_rs + (int)col] : 0, r * RUN};
  };
  auto slab_of = [&](const Run &r, int h) { return (uint32_t)((unsigned)r.page < (unsigned)a.nb ? r.page : 0) * (uint32_t)a.hkv + (uint32_t)h; };
  const int l_row = n / CPR, l_chunk = n % CPR;  // the lane's part of a load: row and 16-byte chunk
  const uint8_t *const k_base = a.k + l_row * D + 16 * l_chunk, *const v_base = a.v + l_row * D + 16 * l_chunk;
  const uint32_t slab_bytes = (uint32_t)(a.bs * D);

  u32x4 kraw[NL], vraw[NL];
  float ks, vs;
  auto request = [&](const Cursor &cu, const Run &run) {
    const uint32_t slab = slab_of(run, cu.h);
    const uint64_t at = (uint64_t)slab * slab_bytes + run.row * D;
#pragma unroll
    for (int i = 0; i < NL; ++i) kraw[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(k_base + at + i * RPL * D));
#pragma unroll
    for (int i = 0; i < NL; ++i) vraw[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(v_base + at + i * RPL * D));
    ks = fa.k_scales[slab], vs = fa.v_scales[slab];
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
        qf[2 * i + t] = u32x4{(w.x ^ fa.negate) & qmask, (w.y ^ fa.negate) & qmask, (w.z ^ fa.negate) & qmask, (w.w ^ fa.negate) & qmask};
      }
  };
  // staging addresses, and those of the operands' reads: K row (TILE / 4) (n / 4) + 4 b + n % 4, chunk 4 i + quad; V as transposed above
  uint8_t *const k_tile = tiles + wib * fp8_lds_bytes<D>(), *const v_tile = k_tile + TILE * D;
  uint32_t kw[NL], vw[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = RUN * quad + i * RPL + l_row;
    kw[i] = (uint32_t)(row * D + ((l_chunk ^ fp8_kkey<D>(row)) << 4));
    vw[i] = (uint32_t)(row * D + ((l_chunk ^ fp8_vkey<D>(row)) << 4));
  }
  uint32_t kr[KP];  // (the key is that of every block's row: blocks are four rows apart)
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    const int row = RUN * (n >> 2) + (n & 3);
    kr[i] = (uint32_t)(row * D + (((4 * i + quad) ^ fp8_kkey<D>(row)) << 4));
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
  // The cursor and unit of the tile behind (cu, at); behind the last one (of the range, or of the wavefront's part of a segment) that itself.
  auto is_last = [&](const Cursor &cu, int64_t at) {
    if constexpr (DIRECT > 0) return cu.tiles_left <= DIRECT * parts;
    return at + (cu.tiles_left > 1 ? 1 : 1 + seg_units) >= x_hi;
  };
  auto advance = [&](Cursor &cu, int64_t &at) {
    if (is_last(cu, at)) return;
    if constexpr (DIRECT > 0) {
      cu.t += DIRECT * parts, cu.tiles_left -= DIRECT * parts;
    } else if (cu.tiles_left > 1) {
      ++cu.t, --cu.tiles_left, ++at;
    } else {
      cu = locate_unit<TILE>(a, s_pref, s_len, at + 1, seg_units);
      at += 1 + seg_units;
    }
  };

  const bool works = DIRECT == 0 || cur.tiles_left > 0;  // (a short segment leaves wavefronts without a tile)
  Cursor nxt = cur;
  int64_t x_nxt = x;
  Run run = {};
  if (works) {
    run = look_up(cur);
    load_q(cur);
    request(cur, run);
    advance(nxt, x_nxt);
    run = look_up(nxt);
  }
  if constexpr (DIRECT == 0) publish_segment_row(a, s_pref, total, n_eff, seg_units);

  floatx4 acc[DBLK];
#pragma unroll
  for (int i = 0; i < DBLK; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  floatx4 l_acc = floatx4{0.f, 0.f, 0.f, 0.f};  // the weights' sum, by the matrix pipe: a row of ones times the probabilities
  float m_run = -INFINITY;                      // what the weights are relative to
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  // The loop holds no request under a condition: where paths with and without one meet, the compiler would wait for all that are out.
  auto process_tile = [&](auto more_tag) {
    constexpr bool more = decltype(more_tag)::value;
    const int first = cur.t * TILE + RUN * quad;           // the lane's first position (scores, scales, V rows)
    const int nvalid = cur.len - first, nbelow = cur.lo - first;
    const bool partial = cur.len - cur.t * TILE < TILE || cur.lo > cur.t * TILE;
    // ---- registers -> LDS; V rows that nobody attends (behind the last token, below a window) become zeros ---------
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(k_tile + kw[i]) = kraw[i];
    if (partial) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = i * RPL + l_row;
        const uint32_t keep = ((row < nvalid) & (row >= nbelow)) ? 0xffffffffu : 0u;
        *reinterpret_cast<u32x4 *>(v_tile + vw[i]) = u32x4{vraw[i].x & keep, vraw[i].y & keep, vraw[i].z & keep, vraw[i].w & keep};
      }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(v_tile + vw[i]) = vraw[i];
    }
    // (not zero, so that masked scores stay -inf)
    // (of a run without a token: anything may stand there)
    const bool some = (nvalid > 0) & (nbelow < RUN);
    const float kscale = some ? fmaxf(ks * a.scale_log2e, 1e-37f) : 1.f, vscale = some ? vs : 1.f;
    const Cursor done = cur;
    const bool closes = DIRECT == 0 && (!more || done.tiles_left <= 1);
    if constexpr (more) {
      cur = nxt, x = x_nxt;
      request(cur, run);
      advance(nxt, x_nxt);
      run = look_up(nxt);
    }
    // ---- S^T = K . Q^T ------------------------------------------------------------------------
    floatx4 st[KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b) {
      st[b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(k_tile + kr[i] + b * (4 * D));
        st[b] = mma16<false>(fp8::decode8(w.x, w.y, 1.f), qf[2 * i], st[b]);
        st[b] = mma16<false>(fp8::decode8(w.z, w.w, 1.f), qf[2 * i + 1], st[b]);
      }
    }
    // ---- V^T from LDS, on its way while the softmax runs ------------------------------------------
    typedef int intx2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) intx2 *lds_v2;
    auto v_block = [&](int s, int db) { return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2)(v_tile + vr[s] + (uint32_t)((db ^ vkey[s]) << 4))); };
    constexpr bool kEarly = D == 64 || (D == 128 && DIRECT == 0);  // (elsewhere there are no registers for it)
    intx2 vt[PSTEPS][kEarly ? DBLK : 1];
    if constexpr (kEarly) {
#pragma unroll
      for (int s = 0; s < PSTEPS; ++s)
#pragma unroll
        for (int db = 0; db < DBLK; ++db) vt[s][db] = v_block(s, db);
    }
    // ---- online softmax -----------------------------------------------------------------------
    // (plain floats: with elements of the matrix results changed inside a branch the compiler wrote others of them, too, at head size 256)
    float sc[4 * KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[4 * b + r] = st[b][r];
    if (partial) {
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) sc[i] = ((i >= nvalid) | (i < nbelow)) ? -INFINITY : sc[i];
    }
    float mloc = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * KBLK; ++i) mloc = fmaxf(mloc, sc[i]);
    mloc = max_over_quads(mloc * kscale);
    // Weights are relative to a maximum that follows only where a score is more than 2^8 ahead of it: they stay below 2^8 with all their
    // bits, and the accumulators are rescaled in the first tile and hardly ever again.
    if (__builtin_amdgcn_ballot_w64(mloc > m_run + 8.f) != 0) {
      const float m_new = fmaxf(m_run, mloc);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      m_run = m_new;
#pragma unroll
      for (int i = 0; i < DBLK; ++i) acc[i] *= alpha;
      l_acc *= alpha;
    }
    const float minus_m = m_run == -INFINITY ? 0.f : -m_run;
    u32x4 pf[PSTEPS];
#pragma unroll
    for (int i = 0; i < 4 * KBLK; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[i], kscale, minus_m));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[i + 1], kscale, minus_m));
      pf[i >> 3][(i >> 1) & 3] = pack_bf16x2(p0, p1);
    }
    // ---- O^T += V^T . P^T ---------------------------------------------------------------------
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
      l_acc = mma16<false>(ones, pf[s], l_acc);  // (the normaliser sums the weights that multiply V)
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const intx2 t = kEarly ? vt[s][kEarly ? db : 0] : v_block(s, db);
        acc[db] = mma16<false>(fp8::decode8((uint32_t)t.x, (uint32_t)t.y, vscale), pf[s], acc[db]);
      }
    }
    // ---- close the segment --------------------------------------------------------------------
    if (closes) {
      float *slot = a.ws_slots + ((int64_t)wave + (int64_t)done.u * a.hkv + done.h) * a.slot_floats;
      if (n < G) {
        float *dst = slot + n * D + 4 * quad;
#pragma unroll
        for (int db = 0; db < DBLK; ++db) *reinterpret_cast<float4 *>(dst + 16 * db) = make_float4(acc[db][0], acc[db][1], acc[db][2], acc[db][3]);
        if (quad == 0) slot[G * D + n] = m_run, slot[G * D + G + n] = l_acc[0];
      }
      if constexpr (more) {
#pragma unroll
        for (int i = 0; i < DBLK; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
        l_acc = floatx4{0.f, 0.f, 0.f, 0.f};
        m_run = -INFINITY;
        load_q(cur);
      }
    }
  };
  if (works) {
    while (!is_last(cur, x)) process_tile(std::true_type{});
    process_tile(std::false_type{});
  }
  if constexpr (DIRECT > 0) {
    const int active = std::min(n_tiles - part * DIRECT, DIRECT);
    if (parts > 1)
      merge_parts<D, DIRECT>(a, seg, G, active, part, parts, fa.parts, fa.arrived, k_tile, tiles, fp8_lds_bytes<D>(), acc, m_run, l_acc[0]);
    else
      merge_waves<D, DIRECT>(a, cur.u, cur.h, G, active, k_tile, tiles, fp8_lds_bytes<D>(), acc, 1.f, m_run, l_acc[0]);
  }
}

template <int D, int DIRECT>
bool launch_fp8_form(const Fp8Args &fa, hipStream_t st) {
  const DecodeArgs &a = fa.d;
  constexpr int kWaves = DIRECT ? DIRECT : kWavesPerBlock;
  const int blocks = DIRECT ? a.users * a.hkv * fa.parts : a.n_waves / kWavesPerBlock;
  const auto lds_for = [](int users) { return (size_t)kWaves * fp8_lds_bytes<D>() + (DIRECT ? 0 : (2 * (size_t)users + 1) * sizeof(int)); };
  static std::atomic<uint64_t> lds_ready{0};
  const auto kernel = &paged_decode_fp8_kernel<D, DIRECT>;
  if (!ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds_for(kMaxUsers), lds_ready)) return false;
  const size_t lds = lds_for(a.users);
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
