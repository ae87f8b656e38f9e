// Attention of a chunk of few rows over the 8-bit cache, read as it is: rows of a KV head are its G query heads times the chunk's tokens, and a
// workgroup takes a block of them (64; 32 at head sizes 128 and 256) over a part of the keys.
//
// Bound by memory with one block of rows per KV head, by the matrix and vector pipes with more: the tiles, their layouts and their way through LDS are
// those of the decode kernel (fp8_decode_kernel.h), a wavefront turns a tile into bfloat16 once and multiplies it with RG groups of 16 rows.
//   S^T, O^T   per group of rows as there: lane (row, quad) holds TILE / 4 tokens in order
//   causal     a row attends chunk_start + its token + 1 keys: a limit per lane and group
// The wavefronts' results meet in LDS, the parts' in memory, merged by a kernel of its own.  Blocks of rows of one KV head and part have
// workgroups on one XCD, which then reads its keys once.  Four groups at head size 128 spill (one token of 32/8 heads behind 8192 28 us, two groups 17.4, three
// 36 with 32 tokens where two take 21.6).  Against copies (fp8_chunk.hip), us a pass copies / this: 8/8 heads of 64, four users, 64 rows behind 10112 tokens
// 49 / 24; 16/16 of 128, four users, 64 behind 4096 66 / 24; 32/8 of 256, one user, 32 behind 8192 55 / 35; 64/8 of 128, 32 behind 6912 34 / 27.
#include "fp8_decode_kernel.h"

#include <algorithm>

namespace ttpa {
namespace decode {
namespace {

struct FewArgs {
  const uint16_t *q;
  uint16_t *out;
  int64_t q_bs, q_hs, q_ts, o_bs, o_hs, o_ts;
  const uint8_t *k, *v;
  const float *k_scales, *v_scales;
  const int32_t *pt;
  int64_t pt_rs;
  const int32_t *chunk_start;
  int batch, hkv, g, s, bs, w, nb;
  float scale_log2e;
  uint32_t runs, runs_inv;  // runs of tokens per block, and floor((2^32 - 1) / runs)
  int row_blocks, parts;
  float *slots;  // [batch * hkv * row_blocks][parts]: ROWS * D values, ROWS maxima, ROWS sums
};

template <int D>
constexpr int few_groups() {
  return D == 64 ? 4 : 2;
}
// Workgroups per CU: two at head size 128, in whose 256 registers two groups fit (five users, 256 rows of a KV head behind 4096 tokens: 53.7 us, 78 with one; 768 rows
// 110, 168); with one each the others need more (64 in 256: 192 rows behind 60000 tokens 64 us as in 366, but 32 rows 43 and not 33).
template <int D>
constexpr int few_per_cu() {
  return D == 128 ? 2 : 1;
}
template <int D>
constexpr int few_slot_floats() {
  return 16 * few_groups<D>() * (D + 2);
}
// Keys that a token of the chunk attends, of those that the table has room for; none in front of the prompt.
__device__ __forceinline__ int keys_of(const FewArgs &a, int start, int token) {
  return (int)max(min((int64_t)start + token + 1, (int64_t)a.w * a.bs), (int64_t)0);
}
// Parts of a block's keys that have any.
template <int D>
__device__ __forceinline__ int few_parts(const FewArgs &a, int keys) {
  constexpr int TILE = fp8_tile<D>();
  return max(1, min(a.parts, ((keys + TILE - 1) / TILE + 3) / 4));
}

template <int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_per_cu<D>(), 2))) void few_rows_kernel(FewArgs a) {
  constexpr int TILE = fp8_tile<D>(), RUN = TILE / 4, RG = few_groups<D>(), ROWS = 16 * RG;
  constexpr int KBLK = TILE / 16, KP = D / 64, DBLK = D / 16, PSTEPS = TILE / 32;
  constexpr int CPR = D / 16, RPL = 16 / CPR, NL = RUN / RPL;
  extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
  __shared__ float2 s_ml[4][ROWS];  // maximum and sum (of two arrays [4][ROWS] the compiler, ROCm 7.2, put two stores into a two-address LDS instruction with a wrong offset for one: the maxima of the first 16 rows went elsewhere)
  // workgroup -> (user, KV head, part) and block of rows, the blocks of one unit eight workgroups apart
  const uint32_t span = 8u * a.row_blocks, set = blockIdx.x / span, in_set = blockIdx.x - set * span;
  const int rb = (int)(in_set >> 3), unit = (int)(set * 8 + (in_set & 7));
  if (unit >= a.batch * a.hkv * a.parts) return;
  const int uh = unit / a.parts, part = unit - uh * a.parts, u = uh / a.hkv, h = uh - u * a.hkv;
  const int lane = threadIdx.x & 63, wib = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int rows = a.g * a.s, row0 = rb * ROWS;
  const int start = a.chunk_start ? *a.chunk_start : 0;
  const int most_keys = keys_of(a, start, (min(row0 + ROWS, rows) - 1) / a.g), least_keys = keys_of(a, start, row0 / a.g);
  const int n_tiles = (most_keys + TILE - 1) / TILE, parts = few_parts<D>(a, most_keys);
  if (part >= parts) return;

  // ---- the rows: row m is token m / g, head m % g of the group -----------------------------------------
  int keys[RG];
  u32x4 qf[RG][2 * KP];  // B operand of k-step 2 i + t: lane (row n, quad) holds features 64 i + 16 quad + 8 t + 0 .. 7
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    const int m = min(row0 + 16 * rg + n, rows - 1), token = m / a.g, head = m - token * a.g;  // (rows past the last: that one again, and not stored)
    keys[rg] = keys_of(a, start, token);
    const uint16_t *qp = a.q + u * a.q_bs + (int64_t)(h * a.g + head) * a.q_hs + token * a.q_ts + 16 * quad;
#pragma unroll
    for (int i = 0; i < KP; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) qf[rg][2 * i + t] = *reinterpret_cast<const u32x4 *>(qp + 64 * i + 8 * t);
  }

  // ---- addresses (fp8_decode_kernel.h) -----------------------------------------------------------------
  struct Run {
    int page;
    uint32_t row;
  };
  auto look_up = [&](int t) {
    const uint32_t x = (uint32_t)(t * 4 + quad);
    uint32_t col = __umulhi(x, a.runs_inv), r = x - col * a.runs;  // one too few at most
    if (r >= a.runs) ++col, r -= a.runs;
    return Run{(int)col < a.w ? a.pt[(int64_t)u * a.pt_rs + (int)col] : 0, r * RUN};
  };
  const int l_row = n / CPR, l_chunk = n % CPR;
  const uint8_t *const k_base = a.k + l_row * D + 16 * l_chunk, *const v_base = a.v + l_row * D + 16 * l_chunk;
  const uint32_t slab_bytes = (uint32_t)(a.bs * D);
  u32x4 kraw[NL], vraw[NL];
  float ks, vs;
  auto request = [&](const Run &run) {
    const uint32_t slab = (uint32_t)((unsigned)run.page < (unsigned)a.nb ? run.page : 0) * (uint32_t)a.hkv + (uint32_t)h;
    const uint64_t at = (uint64_t)slab * slab_bytes + run.row * D;
#pragma unroll
    for (int i = 0; i < NL; ++i) kraw[i] = *reinterpret_cast<const u32x4 *>(k_base + at + i * RPL * D);
#pragma unroll
    for (int i = 0; i < NL; ++i) vraw[i] = *reinterpret_cast<const u32x4 *>(v_base + at + i * RPL * D);
    ks = a.k_scales[slab], vs = a.v_scales[slab];
  };
  uint8_t *const k_tile = tiles + wib * fp8_lds_bytes<D>(), *const v_tile = k_tile + TILE * D;
  uint32_t kw[NL], vw[NL], kr[KP], vr[PSTEPS];
  int vkey[PSTEPS];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = RUN * quad + i * RPL + l_row;
    kw[i] = (uint32_t)(row * D + ((l_chunk ^ fp8_kkey<D>(row)) << 4));
    vw[i] = (uint32_t)(row * D + ((l_chunk ^ fp8_vkey<D>(row)) << 4));
  }
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    const int row = RUN * (n >> 2) + (n & 3);
    kr[i] = (uint32_t)(row * D + (((4 * i + quad) ^ fp8_kkey<D>(row)) << 4));
  }
#pragma unroll
  for (int s = 0; s < PSTEPS; ++s) {
    const int row = RUN * quad + 8 * s + (n >> 1);
    vr[s] = (uint32_t)(row * D + 8 * (n & 1));
    vkey[s] = fp8_vkey<D>(row);
  }

  floatx4 acc[RG][DBLK], l_acc[RG];
  float m_run[RG];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
    for (int i = 0; i < DBLK; ++i) acc[rg][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    l_acc[rg] = floatx4{0.f, 0.f, 0.f, 0.f}, m_run[rg] = -INFINITY;
  }
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  // Tile t of the wavefront's, every 4 * parts-th from part * 4 + wib on; `run`: the next one's.
  int t = part * 4 + wib;
  const int step = 4 * parts;
  Run run = {};
  auto process_tile = [&](auto more_tag) {
    constexpr bool more = decltype(more_tag)::value;
    const int first = t * TILE + RUN * quad;
    const bool partial = (t + 1) * TILE > least_keys;
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(k_tile + kw[i]) = kraw[i];
    const int nvalid = most_keys - first;  // (V rows that nobody of the block attends become zeros)
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const uint32_t keep = !partial || i * RPL + l_row < nvalid ? 0xffffffffu : 0u;
      *reinterpret_cast<u32x4 *>(v_tile + vw[i]) = u32x4{vraw[i].x & keep, vraw[i].y & keep, vraw[i].z & keep, vraw[i].w & keep};
    }
    // (not zero, so that masked scores stay -inf; of a run without a key anything may stand there)
    const float kscale = nvalid > 0 ? fmaxf(ks * a.scale_log2e, 1e-37f) : 1.f, vscale = nvalid > 0 ? vs : 1.f;
    if constexpr (more) {
      request(run);
      run = look_up(min(t + 2 * step, n_tiles - 1));
    }
    // ---- S^T = K . Q^T ----
    floatx4 st[RG][KBLK];
#pragma unroll
    for (int b = 0; b < KBLK; ++b) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) st[rg][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(k_tile + kr[i] + b * (4 * D));
        const u32x4 lo = fp8::decode8(w.x, w.y, 1.f), hi = fp8::decode8(w.z, w.w, 1.f);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) st[rg][b] = mma16<false>(lo, qf[rg][2 * i], st[rg][b]);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) st[rg][b] = mma16<false>(hi, qf[rg][2 * i + 1], st[rg][b]);
      }
    }
    // ---- online softmax, the lazy maximum of the decode kernel ----
    u32x4 pf[RG][PSTEPS];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      float sc[4 * KBLK];
#pragma unroll
      for (int b = 0; b < KBLK; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[4 * b + r] = st[rg][b][r];
      const int valid = partial ? keys[rg] - first : TILE;
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) sc[i] = i >= valid ? -INFINITY : sc[i];
      float mloc = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * KBLK; ++i) mloc = fmaxf(mloc, sc[i]);
      mloc = max_over_quads(mloc * kscale);
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
      for (int i = 0; i < 4 * KBLK; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[i], kscale, minus_m));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[i + 1], kscale, minus_m));
        pf[rg][i >> 3][(i >> 1) & 3] = pack_bf16x2(p0, p1);
      }
      __builtin_amdgcn_sched_barrier(0);  // (interleaved, the groups want more registers than there are)
    }
    // ---- O^T += V^T . P^T ----
    typedef int intx2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) intx2 *lds_v2;
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) l_acc[rg] = mma16<false>(ones, pf[rg][s], l_acc[rg]);
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const intx2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2)(v_tile + vr[s] + (uint32_t)((db ^ vkey[s]) << 4)));
        const u32x4 v = fp8::decode8((uint32_t)w.x, (uint32_t)w.y, vscale);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) acc[rg][db] = mma16<false>(v, pf[rg][s], acc[rg][db]);
      }
    }
    t += step;
  };
  if (t < n_tiles) {
    run = look_up(t);
    request(run);
    run = look_up(min(t + step, n_tiles - 1));
    while (t + step < n_tiles) process_tile(std::true_type{});
    process_tile(std::false_type{});
  }

  // ---- the wavefronts' results, a share of the features at a time (a wavefront's tiles hold that many) ------
  constexpr int FIT = fp8_lds_bytes<D>() / (RG * 64 * 16);  // blocks of 16 features: 16 bytes per lane and group
  constexpr int BLOCKS = FIT >= 8 ? 8 : FIT >= 4 ? 4 : FIT >= 2 ? 2 : FIT;
  static_assert(BLOCKS >= 1 && DBLK % BLOCKS == 0, "shares of whole blocks");
  if (lane < 16) {
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) s_ml[wib][16 * rg + n] = make_float2(m_run[rg], l_acc[rg][0]);
  }
  float *const slot = a.slots + ((int64_t)(uh * a.row_blocks + rb) * a.parts + part) * few_slot_floats<D>();
#pragma unroll
  for (int share = 0; share < DBLK / BLOCKS; ++share) {
    __syncthreads();  // (the tiles, or the share before, are done with)
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const floatx4 &x = acc[rg][share * BLOCKS + b];
        *reinterpret_cast<float4 *>(k_tile + ((b * RG + rg) * 64 + lane) * 16) = make_float4(x[0], x[1], x[2], x[3]);
      }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < BLOCKS * RG * 64; i += 256) {
      const int b = i / (RG * 64), rg = i / 64 % RG, l = i & 63, row = 16 * rg + (l & 15), feature = 16 * (share * BLOCKS + b) + 4 * (l >> 4);
      float mall = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mall = fmaxf(mall, s_ml[w][row].x);
      const float ref = merge_reference(mall);
      float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float wgt = __builtin_amdgcn_exp2f(s_ml[w][row].x - ref);
        const float4 x = *reinterpret_cast<const float4 *>(tiles + w * fp8_lds_bytes<D>() + i * 16);
        num[0] = fmaf(wgt, x.x, num[0]), num[1] = fmaf(wgt, x.y, num[1]), num[2] = fmaf(wgt, x.z, num[2]), num[3] = fmaf(wgt, x.w, num[3]);
        den = fmaf(wgt, s_ml[w][row].y, den);
      }
      if (a.parts == 1) {
        const int m = row0 + row;
        if (m < rows) {
          const int token = m / a.g, head = m - token * a.g;
          const float inv = 1.f / den;
          *reinterpret_cast<uint2 *>(a.out + u * a.o_bs + (int64_t)(h * a.g + head) * a.o_hs + token * a.o_ts + feature) =
              make_uint2(pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv));
        }
      } else {
        *reinterpret_cast<float4 *>(slot + row * D + feature) = make_float4(num[0], num[1], num[2], num[3]);
        if (feature == 0) slot[ROWS * D + row] = mall, slot[ROWS * (D + 1) + row] = den;
      }
    }
  }
}

// The parts' results: a thread per four features of a row.
template <int D>
__global__ __launch_bounds__(256) void few_rows_merge_kernel(FewArgs a) {
  constexpr int ROWS = 16 * few_groups<D>(), PER = D / 4;
  const int seg = blockIdx.x, uh = seg / a.row_blocks, rb = seg - uh * a.row_blocks, u = uh / a.hkv, h = uh - u * a.hkv;
  const int i = blockIdx.y * 256 + threadIdx.x, row = i / PER, feature = 4 * (i - row * PER);
  const int rows = a.g * a.s, m = rb * ROWS + row;
  if (m >= rows) return;
  const int start = a.chunk_start ? *a.chunk_start : 0;
  const int parts = few_parts<D>(a, keys_of(a, start, (min((rb + 1) * ROWS, rows) - 1) / a.g));
  const float *slot = a.slots + (int64_t)seg * a.parts * few_slot_floats<D>();
  float mall = -INFINITY, num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  constexpr int kBatch = 4;
  for (int p0 = 0; p0 < parts; p0 += kBatch) {
    float mv[kBatch], lv[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float *p = slot + (int64_t)min(p0 + j, parts - 1) * few_slot_floats<D>();
      x[j] = *reinterpret_cast<const float4 *>(p + row * D + feature);
      mv[j] = p0 + j < parts ? p[ROWS * D + row] : -INFINITY, lv[j] = p[ROWS * (D + 1) + row];
    }
    float m_new = mall;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m_new = fmaxf(m_new, mv[j]);
    const float ref = merge_reference(m_new), resc = __builtin_amdgcn_exp2f(mall - ref);
#pragma unroll
    for (int r = 0; r < 4; ++r) num[r] *= resc;
    den *= resc, mall = m_new;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
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

template <int D>
int launch_few(FewArgs &a, hipStream_t st) {
  constexpr int ROWS = 16 * few_groups<D>();
  static std::atomic<uint64_t> lds_ready{0};
  const size_t lds = 4 * fp8_lds_bytes<D>();
  if (!ensure_dynamic_lds(reinterpret_cast<const void *>(&few_rows_kernel<D>), lds, lds_ready))
    return fail(TTPA_ERR_LAUNCH, "fp8 chunk: cannot configure the kernel of few rows");
  const int units = a.batch * a.hkv * a.parts;
  launch_dominant(&few_rows_kernel<D>, dim3((unsigned)((units + 7) / 8 * 8 * a.row_blocks)), dim3(256), lds, st, a);
  if (const int rc = check_launch("fp8 chunk (few rows)")) return rc;
  if (a.parts == 1) return TTPA_OK;
  few_rows_merge_kernel<D><<<dim3(a.batch * a.hkv * a.row_blocks, ROWS * D / 4 / 256), dim3(256), 0, st>>>(a);
  return check_launch("fp8 chunk (merge)");
}

}  // namespace
}  // namespace decode

namespace fp8 {

// Blocks of rows per KV head, and parts of the keys.  What counts is rounds of workgroups, each as long as a wavefront's tiles and about three more for its
// beginning and end (264 workgroups took nearly twice as long as 256).  Returns that number of tiles.
static int64_t few_split(int batch, int kv_heads, int64_t rows, int head_size, int64_t keys, int &row_blocks, int &parts) {
  const int per = head_size == 64 ? 64 : 32, tile = head_size <= 128 ? 64 : 32;
  row_blocks = (int)((rows + per - 1) / per);
  const int64_t segments = (int64_t)batch * kv_heads * row_blocks, tiles = (keys + tile - 1) / tile;
  const int64_t at_once = std::max(device_cus(), 1) * (head_size == 128 ? decode::few_per_cu<128>() : 1);
  int64_t best = INT64_MAX;
  parts = 1;
  for (int64_t p = 1; p <= std::min<int64_t>(32, (tiles + 3) / 4); ++p) {
    const int64_t cost = (segments * p + at_once - 1) / at_once * ((tiles + 4 * p - 1) / (4 * p) + 3);
    if (cost < best) best = cost, parts = (int)p;
  }
  return best;
}

// us that this form is expected to take, with which the other one's (copies, then the prefill kernels) is compared.  32/8 heads of 128, one user: 128 rows of a KV
// head behind 8192 tokens 23.9 (expected 23.9), 256 29.8 (29.2), 512 40.6 (39.8), 768 62.3 (61.0); five users behind 4096: 256 53.7 (55.7), 768 110 (114).
double chunk_few_us(int batch, int q_heads, int kv_heads, int q_len, int head_size, int64_t keys) {
  int row_blocks, parts;
  const int64_t tiles = few_split(batch, kv_heads, (int64_t)(q_heads / kv_heads) * q_len, head_size, keys, row_blocks, parts);
  return 8.0 + (head_size == 64 ? 1.9 : head_size == 128 ? 2.65 : 2.25) * (double)tiles;
}

int64_t chunk_few_bytes(int batch, int q_heads, int kv_heads, int q_len, int head_size, int64_t keys) {
  int row_blocks, parts;
  few_split(batch, kv_heads, (int64_t)(q_heads / kv_heads) * q_len, head_size, keys, row_blocks, parts);
  const int64_t slot = (head_size == 64 ? 64 : 32) * (int64_t)(head_size + 2) * 4;
  return parts == 1 ? 256 : (int64_t)batch * kv_heads * row_blocks * parts * slot;
}

int chunk_few(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q, int64_t q_batch_stride,
              int64_t q_head_stride, int64_t q_token_stride, const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
              const int32_t *page_table, int64_t page_table_row_stride, const int32_t *chunk_start, int batch, int q_heads, int kv_heads, int q_len,
              int head_size, int block_size, int table_width, int num_blocks, float scale, int64_t keys, void *workspace, hipStream_t st) {
  decode::FewArgs a = {};
  a.q = static_cast<const uint16_t *>(q), a.q_bs = q_batch_stride, a.q_hs = q_head_stride, a.q_ts = q_token_stride;
  a.out = static_cast<uint16_t *>(out), a.o_bs = out_batch_stride, a.o_hs = out_head_stride, a.o_ts = out_token_stride;
  a.k = static_cast<const uint8_t *>(k_cache), a.v = static_cast<const uint8_t *>(v_cache), a.k_scales = k_scales, a.v_scales = v_scales;
  a.pt = page_table, a.pt_rs = page_table_row_stride, a.chunk_start = chunk_start;
  a.batch = batch, a.hkv = kv_heads, a.g = q_heads / kv_heads, a.s = q_len, a.bs = block_size, a.w = table_width, a.nb = num_blocks;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.runs = (uint32_t)block_size / (head_size <= 128 ? 16 : 8), a.runs_inv = 0xffffffffu / a.runs;
  few_split(batch, kv_heads, (int64_t)a.g * q_len, head_size, keys, a.row_blocks, a.parts);
  a.slots = static_cast<float *>(workspace);
  TTPA_REQUIRE(((int64_t)batch * kv_heads * a.parts + 8) * a.row_blocks < (1ll << 24), "fp8 chunk: too many rows for one launch");
  switch (head_size) {
    case 64: return decode::launch_few<64>(a, st);
    case 128: return decode::launch_few<128>(a, st);
    default: return decode::launch_few<256>(a, st);
  }
}

}  // namespace fp8
}  // namespace ttpa
