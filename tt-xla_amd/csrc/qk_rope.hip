// Norms of queries and keys for each head with the position rotation in the same pass, alone and with a step's cache write.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (w one of two vectors of head_size, for queries and for keys; none: y = x)
//   (y_i, y_j) <- (y_i c - y_j s, y_j c + y_i s)  for the pairs (i, i + rotary / 2), or (2 i, 2 i + 1) interleaved;
//   features from `rotary` on are not turned.  Sums and products in 32 bits, one rounding to bfloat16 at the end.
//
// Bound by memory: a row is read and written once.  A head row lies in D / 16 lanes as two chunks of eight features that
// are `rotary / 2` apart, so that both features of a pair are a lane's own and the norm's sum is a few
// cross-lane moves; 16-byte loads and stores, 128 consecutive bytes of a row at a time.  A wavefront takes U
// groups of 1024 / D heads of one token: its cosines, sines and weights are read once for all of them, and 2 U loads of rows are in flight.
// 8192 tokens of 32 + 8 heads of 128: 168 MB in 32.5 us, 5.2 TB/s (a large copy by torch reaches 4.9).
#include "fp8_rows.h"

#include <algorithm>
#include <type_traits>

namespace ttpa {
namespace {

using fp8::RowPart;
using fp8::u32x4;

struct RopeArgs {
  uint16_t *q_out, *k_out;
  int64_t qo_ts, qo_hs, ko_ts, ko_hs;
  const uint16_t *q, *k;
  int64_t q_ts, q_hs, k_ts, k_hs;
  const void *angles;  // [max_positions, rotary]: cosines, then sines
  int64_t angle_rs;
  int angles_f32, weights_f32;
  int64_t max_positions;
  const void *positions;
  int positions_i64;
  const void *q_weight, *k_weight;
  float eps;
  int tokens, hq, hk;  // hk: key heads that this launch turns
  int rotary, interleaved;
};

// Which features a lane holds: chunks a and b, and whether they are turned.  A row's turned part and the rest have their first halves in chunks a, so that a
// load or store of a wavefront takes neighbouring bytes (8192 tokens of 32 + 8 heads of 128, 32 features turned: 34.2 us, 41.5 with the rest's two chunks side by side).
template <int D>
struct Place {
  int fa, fb;    // first features of the chunks
  bool turned;
  int ca, cb;    // where the cosines of chunk a and b start (interleaved: four each; else eight, shared)
  __device__ __forceinline__ Place(const RopeArgs &a) {
    const int l = (int)(threadIdx.x & 63) % (D / 16), turning = a.rotary / 16;
    turned = l < turning;
    fa = turned ? 8 * l : a.rotary + 8 * (l - turning);
    fb = fa + (turned ? a.rotary : D - a.rotary) / 2;
    ca = a.interleaved ? fa / 2 : fa;
    cb = a.interleaved ? fb / 2 : fa + 4;
  }
};

__device__ __forceinline__ void load4(const void *p, int is_f32, int64_t at, float (&v)[4]) {
  if (is_f32) {
    const float4 t = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else {
    const uint2 t = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
    v[0] = bf16_lo(t.x), v[1] = bf16_hi(t.x), v[2] = bf16_lo(t.y), v[3] = bf16_hi(t.y);
  }
}

// The cosines and sines of a token for the lane's eight pairs, as four and four.  A position outside the table is not turned.
struct Angles {
  float c[2][4], s[2][4];
};
template <int D>
__device__ __forceinline__ Angles angles_of(const RopeArgs &a, const Place<D> &p, int64_t pos) {
  Angles t;
  const bool known = p.turned && pos >= 0 && pos < a.max_positions;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (known) {
      const int64_t at = pos * a.angle_rs + (h ? p.cb : p.ca);
      load4(a.angles, a.angles_f32, at, t.c[h]);
      load4(a.angles, a.angles_f32, at + a.rotary / 2, t.s[h]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) t.c[h][i] = 1.f, t.s[h][i] = 0.f;
    }
  }
  return t;
}

struct Weights {
  float a[8], b[8];
};
template <int D>
__device__ __forceinline__ void load_weights(const void *w, int is_f32, const Place<D> &p, Weights &o) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float t[4];
    load4(w, is_f32, p.fa + 4 * j, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.a[4 * j + i] = t[i];
    load4(w, is_f32, p.fb + 4 * j, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.b[4 * j + i] = t[i];
  }
}

__device__ __forceinline__ RowPart load_part(const uint16_t *row, int fa, int fb) {
  return {*reinterpret_cast<const u32x4 *>(row + fa), *reinterpret_cast<const u32x4 *>(row + fb)};
}

// One row: norm (NORM; `w` its weights) and rotation.
template <int D>
__device__ __forceinline__ RowPart turn_row(const RopeArgs &a, const Place<D> &p, const RowPart &x, bool norm, const Weights &w, const Angles &t) {
  float fa[8], fb[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    fa[2 * i] = bf16_lo(x.a[i]), fa[2 * i + 1] = bf16_hi(x.a[i]);
    fb[2 * i] = bf16_lo(x.b[i]), fb[2 * i + 1] = bf16_hi(x.b[i]);
  }
  if (norm) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(fa[i], fa[i], fmaf(fb[i], fb[i], sum));
    sum += dpp_move<kDppXor1>(sum);
    sum += dpp_move<kDppXor2>(sum);
    if constexpr (D >= 128) sum += dpp_move<kDppHalfMirror>(sum);
    if constexpr (D >= 256) sum += dpp_move<kDppMirror>(sum);
    const float inv = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) fa[i] *= inv * w.a[i], fb[i] *= inv * w.b[i];
  }
  if (p.turned) {
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = fa[2 * i], x1 = fa[2 * i + 1], y0 = fb[2 * i], y1 = fb[2 * i + 1];
        fa[2 * i] = x0 * t.c[0][i] - x1 * t.s[0][i], fa[2 * i + 1] = x1 * t.c[0][i] + x0 * t.s[0][i];
        fb[2 * i] = y0 * t.c[1][i] - y1 * t.s[1][i], fb[2 * i + 1] = y1 * t.c[1][i] + y0 * t.s[1][i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = fa[i], x1 = fb[i], c = t.c[i >> 2][i & 3], s = t.s[i >> 2][i & 3];
        fa[i] = x0 * c - x1 * s, fb[i] = x1 * c + x0 * s;
      }
    }
  }
  RowPart o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.a[i] = pack_bf16x2(fa[2 * i], fa[2 * i + 1]), o.b[i] = pack_bf16x2(fb[2 * i], fb[2 * i + 1]);
  return o;
}

// Wavefront `part` of a token's: heads [part * U * R, ...) of the queries' and then the keys' (R rows per wavefront).
template <int D, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a, int parts) {
  constexpr int LPR = D / 16, R = 64 / LPR;
  const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int token = wave / parts, part = wave - token * parts;
  if (token >= a.tokens) return;
  const Place<D> p(a);
  const int r = (int)(threadIdx.x & 63) / LPR, heads = a.hq + a.hk;
  RowPart x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = min((part * U + u) * R + r, heads - 1);  // (rows past the last head: that one again, and not stored)
    x[u] = h < a.hq ? load_part(a.q + token * a.q_ts + h * a.q_hs, p.fa, p.fb) : load_part(a.k + token * a.k_ts + (h - a.hq) * a.k_hs, p.fa, p.fb);
  }
  const Angles t = angles_of<D>(a, p, load_index(a.positions, a.positions_i64, token));
  Weights wq, wk;
  if (a.q_weight) load_weights<D>(a.q_weight, a.weights_f32, p, wq);
  if (a.k_weight) load_weights<D>(a.k_weight, a.weights_f32, p, wk);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (part * U + u) * R + r;
    const bool is_q = h < a.hq;
    Weights w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.a[i] = is_q ? wq.a[i] : wk.a[i], w.b[i] = is_q ? wq.b[i] : wk.b[i];
    const RowPart y = turn_row<D>(a, p, x[u], (is_q ? a.q_weight : a.k_weight) != nullptr, w, t);
    if (h < heads) {
      uint16_t *dst = is_q ? a.q_out + token * a.qo_ts + h * a.qo_hs : a.k_out + token * a.ko_ts + (h - a.hq) * a.ko_hs;
      if constexpr (U > 1) {
        __builtin_nontemporal_store(y.a, reinterpret_cast<u32x4 *>(dst + p.fa));
        __builtin_nontemporal_store(y.b, reinterpret_cast<u32x4 *>(dst + p.fb));
      } else {
        *reinterpret_cast<u32x4 *>(dst + p.fa) = y.a;
        *reinterpret_cast<u32x4 *>(dst + p.fb) = y.b;
      }
    }
  }
}

// The same over the rows of all tokens in order (row = token * heads + head), U * R consecutive ones per wavefront, each with angles of its own: for so
// few heads that a token's own one or two wavefronts stay partly empty.  us a pass, a token's wavefronts / this: 12056 tokens of 8 + 2 heads of 64 14.1 / 8.8,
// 16384 of 8 + 1 of 128 24.0 / 19.4 and of 4 + 1 18.2 / 12.7, 8192 of 2 + 1 of 256 11.2 / 8.4; with three wavefronts per token 8192 of 16 + 2 of 128 17.7 / 18.9.
// (One, three and four rows per lane 10.1, 9.5 and 9.5 on the first.)
template <int D, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_rows_kernel(RopeArgs a, uint32_t heads_inv) {
  constexpr int LPR = D / 16, R = 64 / LPR;
  const Place<D> p(a);
  const uint32_t heads = a.hq + a.hk, rows = (uint32_t)a.tokens * heads;
  const uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (U * R) + (threadIdx.x & 63) / LPR;
  RowPart x[U];
  int token[U], head[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t row = min(first + u * R, rows - 1);  // (rows past the last: that one again, and not stored)
    uint32_t n = __umulhi(row, heads_inv), h = row - n * heads;  // one too few at most
    if (h >= heads) ++n, h -= heads;
    token[u] = (int)n, head[u] = (int)h;
  }
  int64_t pos[U];
#pragma unroll
  for (int u = 0; u < U; ++u) pos[u] = load_index(a.positions, a.positions_i64, token[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = head[u] - a.hq;
    x[u] = load_part(h < 0 ? a.q + token[u] * a.q_ts + head[u] * a.q_hs : a.k + token[u] * a.k_ts + h * a.k_hs, p.fa, p.fb);
  }
  Angles t[U];
#pragma unroll
  for (int u = 0; u < U; ++u) t[u] = angles_of<D>(a, p, pos[u]);
  Weights wq, wk;
  if (a.q_weight) load_weights<D>(a.q_weight, a.weights_f32, p, wq);
  if (a.k_weight) load_weights<D>(a.k_weight, a.weights_f32, p, wk);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = head[u] - a.hq;
    Weights w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.a[i] = h < 0 ? wq.a[i] : wk.a[i], w.b[i] = h < 0 ? wq.b[i] : wk.b[i];
    const RowPart y = turn_row<D>(a, p, x[u], (h < 0 ? a.q_weight : a.k_weight) != nullptr, w, t[u]);
    if (first + u * R < rows) {
      uint16_t *dst = h < 0 ? a.q_out + token[u] * a.qo_ts + head[u] * a.qo_hs : a.k_out + token[u] * a.ko_ts + h * a.ko_hs;
      __builtin_nontemporal_store(y.a, reinterpret_cast<u32x4 *>(dst + p.fa));
      __builtin_nontemporal_store(y.b, reinterpret_cast<u32x4 *>(dst + p.fb));
    }
  }
}

struct StepArgs {
  RopeArgs rope;
  fp8::Caches c;
  const uint16_t *v;
  int64_t v_ts, v_hs;
  int rotate;  // 0: keys are written as they are, and there are no queries
};

// A step's write: one token per user, its keys (turned first, if `rotate`) and values into the cache; with the turned queries
// written out by the wavefronts in front.  Bound by latency: position, page, scale and bounds are a chain of three reads, of a few
// KiB in all; so every wavefront has one group of heads of one operand, a workgroup is one wavefront, and whatever a read does not wait for is asked
// for before it: the row and the weights beside the position, the angles beside the page.  Users whose tokens go to the same block write in
// turn, by the first one's wavefront.
template <int D>
__global__ __launch_bounds__(64) void step_write_kernel(StepArgs a, int q_parts, int kv_parts) {
  constexpr int LPR = D / 16, R = 64 / LPR;
  const int parts = q_parts + 2 * kv_parts;
  const int token = blockIdx.x / parts, part = blockIdx.x - token * parts;
  const RopeArgs &ra = a.rope;
  const Place<D> p(ra);
  const int r = (int)threadIdx.x / LPR;
  const fp8::Turn turn{ra.positions, ra.positions_i64, ra.tokens};
  if (part < q_parts) {
    const int h = min(part * R + r, ra.hq - 1);  // (rows past the last head: that one again, and not stored)
    const RowPart x = load_part(ra.q + token * ra.q_ts + h * ra.q_hs, p.fa, p.fb);
    Weights w;
    if (ra.q_weight) load_weights<D>(ra.q_weight, ra.weights_f32, p, w);
    const Angles t = angles_of<D>(ra, p, turn.position(token));
    const RowPart y = turn_row<D>(ra, p, x, ra.q_weight != nullptr, w, t);
    if (part * R + r < ra.hq) {
      uint16_t *dst = ra.q_out + token * ra.qo_ts + h * ra.qo_hs;
      *reinterpret_cast<u32x4 *>(dst + p.fa) = y.a;
      *reinterpret_cast<u32x4 *>(dst + p.fb) = y.b;
    }
    return;
  }
  const bool is_v = part >= q_parts + kv_parts;
  const int h = (part - q_parts - (is_v ? kv_parts : 0)) * R + r;
  const bool live = h < a.c.hkv, turned = !is_v && a.rotate;
  const int head = live ? h : 0;
  uint8_t *const cache = is_v ? a.c.v : a.c.k;
  float *const scales = is_v ? a.c.v_scales : a.c.k_scales;
  uint16_t *const bounds = is_v ? nullptr : a.c.bounds;
  const auto load_row = [&](int u) {
    return is_v ? load_part(a.v + u * a.v_ts + head * a.v_hs, p.fa, p.fb) : load_part(ra.k + u * ra.k_ts + head * ra.k_hs, p.fa, p.fb);
  };
  int u = token;
  RowPart x = load_row(u);
  Weights w;
  if (turned && ra.k_weight) load_weights<D>(ra.k_weight, ra.weights_f32, p, w);
  fp8::Blocks blocks;
  fp8::request_positions(turn, 0, blocks);
  int64_t pos = turn.position(u);
  int col, row;
  if (!fp8::place_of(a.c, pos, col, row)) return;
  int phys = a.c.pt[u * a.c.pt_rs + col];
  fp8::request_blocks(a.c, turn, 0, blocks);
  Angles t;
  if (turned) t = angles_of<D>(ra, p, pos);
  if ((unsigned)phys >= (unsigned)a.c.nb) return;
  fp8::Held held = fp8::load_held<D>(scales, bounds, a.c, head, phys, row, p.fa, p.fb);
  bool before;
  int next = fp8::next_in_block(a.c, turn, u, phys, blocks, before);
  if (before) return;  // an earlier user's wavefront writes this one's token, too
  for (;;) {
    if (turned) x = turn_row<D>(ra, p, x, ra.k_weight != nullptr, w, t);
    fp8::write_row<D>(cache, scales, bounds, a.c, head, live, phys, row, x, held, p.fa, p.fb);
    if (next == ra.tokens) return;
    // what has been written is read again, by other lanes of the wavefront, too
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
    u = next;
    x = load_row(u);
    pos = turn.position(u);
    (void)fp8::place_of(a.c, pos, col, row);  // (of the same block)
    if (turned) t = angles_of<D>(ra, p, pos);
    held = fp8::load_held<D>(scales, bounds, a.c, head, phys, row, p.fa, p.fb);
    next = fp8::next_in_block(a.c, turn, u, phys, blocks, before);
  }
}

template <int D>
int launch_rope(const RopeArgs &a, hipStream_t st) {
  constexpr int R = 1024 / D;
  const int groups = (a.hq + a.hk + R - 1) / R;
  const auto go = [&](auto tag) {
    constexpr int U = decltype(tag)::value;
    const int parts = (groups + U - 1) / U;
    const int64_t waves = (int64_t)a.tokens * parts;
    qk_norm_rope_kernel<D, U><<<dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st>>>(a, parts);
  };
  // Few rows want to be everywhere at once; many, three to five groups per wavefront, as many as leave no slot without a group, or else five: its angles and
  // weights are read once.  8192 tokens of 32 + 8 heads of 128 (168 MB), us a pass with 1 / 2 / 3 / 5 groups 44.1 / 41.4 / 36.8 / 32.5; with ordinary
  // stores 44.5 / 41.9 / 39.0 / 36.9.  (Those of few rows are ordinary: what is read next is read from L2.)
  int best = 1;
  if ((int64_t)a.tokens * groups >= 8192) {
    if (groups <= 2) {
      constexpr int U = 2, PER = 4 * U * R;  // rows of a workgroup
      const int64_t rows = (int64_t)a.tokens * (a.hq + a.hk);
      qk_norm_rope_rows_kernel<D, U><<<dim3((unsigned)((rows + PER - 1) / PER)), dim3(256), 0, st>>>(a, 0xffffffffu / (uint32_t)(a.hq + a.hk));
      return check_launch("qk_norm_rope");
    }
    for (int u = 3; u <= std::min(groups, 5); ++u)
      if ((groups + u - 1) / u * u <= (groups + best - 1) / best * best || (u == 5 && best == 1)) best = u;
  }
  switch (best) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    default: go(std::integral_constant<int, 5>{}); break;
  }
  return check_launch("qk_norm_rope");
}

template <int D>
int launch_step(const StepArgs &a, hipStream_t st) {
  constexpr int R = 1024 / D;
  const int q_parts = a.rotate ? (a.rope.hq + R - 1) / R : 0, kv_parts = (a.c.hkv + R - 1) / R;
  step_write_kernel<D><<<dim3((unsigned)((int64_t)a.rope.tokens * (q_parts + 2 * kv_parts))), dim3(64), 0, st>>>(a, q_parts, kv_parts);
  return check_launch("fp8 step write");
}

int check_rope(RopeArgs &a, int head_size, bool outputs_k) {
  TTPA_REQUIRE(a.q && a.k && a.q_out && (!outputs_k || a.k_out) && a.angles && a.positions, "qk_norm_rope: null pointer argument");
  TTPA_REQUIRE(a.tokens >= 0 && a.hq > 0 && a.max_positions > 0, "qk_norm_rope: non-positive dimension");
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return fail(TTPA_ERR_UNSUPPORTED, "qk_norm_rope: head_size %d; supported 64, 128, 256", head_size);
  TTPA_REQUIRE(a.rotary > 0 && a.rotary <= head_size && a.rotary % 16 == 0, "qk_norm_rope: rotary %d must be a multiple of 16 up to head_size %d",
               a.rotary, head_size);
  TTPA_REQUIRE(a.eps >= 0.f, "qk_norm_rope: eps %g is negative", (double)a.eps);
  TTPA_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.q_out) && (!outputs_k || aligned16(a.k_out)) && aligned16(a.angles) &&
                   (!a.q_weight || aligned16(a.q_weight)) && (!a.k_weight || aligned16(a.k_weight)),
               "qk_norm_rope: operands must be 16-byte aligned");
  TTPA_REQUIRE(a.q_ts % 8 == 0 && a.q_hs % 8 == 0 && a.k_ts % 8 == 0 && a.k_hs % 8 == 0 && a.qo_ts % 8 == 0 && a.qo_hs % 8 == 0 &&
                   a.ko_ts % 8 == 0 && a.ko_hs % 8 == 0 && a.angle_rs % 8 == 0,
               "qk_norm_rope: strides must be multiples of 8 elements");
  TTPA_REQUIRE((int64_t)a.tokens * ((a.hq + a.hk) / (1024 / head_size) + 3) < (1ll << 26), "qk_norm_rope: too many rows for one launch");
  return TTPA_OK;
}

}  // namespace

namespace fp8 {
// Checks of an 8-bit cache shared by its entry points.
int check_cache(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table, int kv_heads,
                int head_size, int block_size, int table_width, int num_blocks) {
  TTPA_REQUIRE(k_cache && v_cache && k_scales && v_scales && page_table, "fp8 cache: null pointer argument");
  TTPA_REQUIRE(kv_heads > 0 && block_size > 0 && table_width > 0 && num_blocks > 0, "fp8 cache: non-positive dimension");
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return fail(TTPA_ERR_UNSUPPORTED, "fp8 cache: head_size %d; supported 64, 128, 256", head_size);
  if (block_size % 16 || block_size > 4096)
    return fail(TTPA_ERR_UNSUPPORTED, "fp8 cache: block_size %d must be a multiple of 16 up to 4096", block_size);
  TTPA_REQUIRE((int64_t)table_width * block_size < (1ll << 31) - 8192, "fp8 cache: a page-table row holds too many tokens");
  TTPA_REQUIRE((int64_t)num_blocks * kv_heads < (1ll << 31), "fp8 cache: num_blocks * kv_heads must stay below 2^31");
  TTPA_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "fp8 cache: caches must be 16-byte aligned");
  return TTPA_OK;
}
}  // namespace fp8
}  // namespace ttpa

using namespace ttpa;

extern "C" int ttpa_qk_norm_rope(void *q_out, int64_t q_out_token_stride, int64_t q_out_head_stride, void *k_out, int64_t k_out_token_stride,
                                 int64_t k_out_head_stride, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
                                 int64_t k_token_stride, int64_t k_head_stride, const void *cos_sin, int cos_sin_is_f32, int64_t cos_sin_row_stride,
                                 int64_t max_positions, const void *positions, int positions_is_i64, const void *q_weight, const void *k_weight,
                                 int weights_are_f32, float eps, int32_t tokens, int32_t q_heads, int32_t k_heads, int32_t head_size,
                                 int32_t rotary, int interleaved, void *stream) {
  RopeArgs a = {static_cast<uint16_t *>(q_out), static_cast<uint16_t *>(k_out), q_out_token_stride, q_out_head_stride, k_out_token_stride,
                k_out_head_stride, static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k), q_token_stride, q_head_stride, k_token_stride,
                k_head_stride, cos_sin, cos_sin_row_stride, cos_sin_is_f32, weights_are_f32, max_positions, positions, positions_is_i64, q_weight,
                k_weight, eps, tokens, q_heads, k_heads, rotary, interleaved};
  TTPA_REQUIRE(k_heads > 0, "qk_norm_rope: non-positive dimension");
  if (int rc = check_rope(a, head_size, true)) return rc;
  if (tokens == 0) return TTPA_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (head_size) {
    case 64: return launch_rope<64>(a, st);
    case 128: return launch_rope<128>(a, st);
    default: return launch_rope<256>(a, st);
  }
}

static int step_write(StepArgs &a, int head_size, hipStream_t st) {
  const int64_t waves = (int64_t)a.rope.tokens * ((a.rope.hq + 2 * a.c.hkv) / (1024 / head_size) + 3);
  TTPA_REQUIRE(waves < (1ll << 26), "fp8 step write: too many rows for one launch");  // (a grid has less than 2^32 threads)
  if (a.rope.tokens == 0) return TTPA_OK;
  switch (head_size) {
    case 64: return launch_step<64>(a, st);
    case 128: return launch_step<128>(a, st);
    default: return launch_step<256>(a, st);
  }
}

extern "C" int ttpa_qk_norm_rope_update_fp8(
    void *q_out, int64_t q_out_token_stride, int64_t q_out_head_stride, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
    int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, const void *cos_sin,
    int cos_sin_is_f32, int64_t cos_sin_row_stride, int64_t max_positions, const void *positions, int positions_is_i64, const void *q_weight,
    const void *k_weight, int weights_are_f32, float eps, void *k_cache, void *v_cache, float *k_scales, float *v_scales, void *key_bounds,
    const int32_t *page_table, int64_t page_table_row_stride, int32_t users, int32_t q_heads, int32_t kv_heads, int32_t head_size, int32_t rotary,
    int interleaved, int32_t block_size, int32_t table_width, int32_t num_blocks, void *stream) {
  StepArgs a = {{static_cast<uint16_t *>(q_out), nullptr, q_out_token_stride, q_out_head_stride, 0, 0, static_cast<const uint16_t *>(q),
                 static_cast<const uint16_t *>(k), q_token_stride, q_head_stride, k_token_stride, k_head_stride, cos_sin, cos_sin_row_stride,
                 cos_sin_is_f32, weights_are_f32, max_positions, positions, positions_is_i64, q_weight, k_weight, eps, users, q_heads, kv_heads,
                 rotary, interleaved},
                {static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache), k_scales, v_scales, static_cast<uint16_t *>(key_bounds),
                 page_table, page_table_row_stride, kv_heads, block_size, table_width, num_blocks, fp8::block_inverse(block_size)},
                static_cast<const uint16_t *>(v), v_token_stride, v_head_stride, 1};
  if (int rc = check_rope(a.rope, head_size, false)) return rc;
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  TTPA_REQUIRE(v && aligned16(v) && v_token_stride % 8 == 0 && v_head_stride % 8 == 0 && (!key_bounds || aligned16(key_bounds)),
               "fp8 step write: values and bounds must be 16-byte aligned, strides multiples of 8 elements");
  return step_write(a, head_size, static_cast<hipStream_t>(stream));
}

extern "C" int ttpa_paged_update_fp8_cache(void *k_cache, void *v_cache, float *k_scales, float *v_scales, void *key_bounds, const void *k_fill,
                                           int64_t k_user_stride, int64_t k_head_stride, const void *v_fill, int64_t v_user_stride,
                                           int64_t v_head_stride, const void *update_indices, int indices_is_i64, const int32_t *page_table,
                                           int64_t page_table_row_stride, int32_t users, int32_t kv_heads, int32_t block_size, int32_t head_size,
                                           int32_t table_width, int32_t num_blocks, void *stream) {
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  TTPA_REQUIRE(users >= 0 && k_fill && v_fill && update_indices, "fp8 step write: null pointer argument");
  TTPA_REQUIRE(aligned16(k_fill) && aligned16(v_fill) && (!key_bounds || aligned16(key_bounds)) && k_user_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                   v_user_stride % 8 == 0 && v_head_stride % 8 == 0,
               "fp8 step write: rows and bounds must be 16-byte aligned, strides multiples of 8 elements");
  StepArgs a = {};
  a.rope.k = static_cast<const uint16_t *>(k_fill), a.rope.k_ts = k_user_stride, a.rope.k_hs = k_head_stride;
  a.rope.positions = update_indices, a.rope.positions_i64 = indices_is_i64;
  a.rope.tokens = users, a.rope.rotary = head_size;
  a.c = {static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache), k_scales, v_scales, static_cast<uint16_t *>(key_bounds), page_table,
         page_table_row_stride, kv_heads, block_size, table_width, num_blocks, fp8::block_inverse(block_size)};
  a.v = static_cast<const uint16_t *>(v_fill), a.v_ts = v_user_stride, a.v_hs = v_head_stride;
  return step_write(a, head_size, static_cast<hipStream_t>(stream));
}
