// One token's rows on their way into the 8-bit cache: what the step's write and the fused norm, rotation and write share.
//
// A head row of D values lies in D / 16 neighbouring lanes, 16 values (two chunks of eight) in each; a wavefront holds
// 1024 / D rows, KV heads of one token.
#pragma once

#include "fp8.h"

namespace ttpa {
namespace fp8 {

// A lane's part of a row: chunks of eight bfloat16 values, a and b.
struct RowPart {
  u32x4 a, b;
};

// Maximum over the D / 16 lanes of a row.
template <int D>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor1, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor2, 0xf, 0xf, true));
  if constexpr (D >= 128) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppHalfMirror, 0xf, 0xf, true));
  if constexpr (D >= 256) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppMirror, 0xf, 0xf, true));
  return v;
}

// Rounds rows [0, rows) of a block slab again for a scale that has grown by 1 / ratio; the whole wavefront, 1 KiB at a time.
template <int D>
__device__ __forceinline__ void rescale_rows(uint8_t *slab, int rows, float ratio) {
  const int bytes = rows * D;
  for (int at = 16 * (int)(threadIdx.x & 63); at < bytes; at += 1024) {
    u32x4 w = *reinterpret_cast<const u32x4 *>(slab + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = rescale4(w[i], ratio);
    *reinterpret_cast<u32x4 *>(slab + at) = w;
  }
}

// What the block holds already for the lane's row: its scale and, where there are any, the bounds of the lane's features.
struct Held {
  float scale;
  u32x4 low[2], high[2];
};
template <int D>
__device__ __forceinline__ Held load_held(const float *scales, const uint16_t *bounds, const Caches &c, int head, int phys, int row, int fa, int fb) {
  const int64_t slab = (int64_t)phys * c.hkv + head;
  Held h = {};
  if (row > 0) {
    h.scale = scales[slab];
    if (bounds) {
      const uint16_t *low = bounds + slab * 2 * D, *high = low + D;
      h.low[0] = *reinterpret_cast<const u32x4 *>(low + fa), h.low[1] = *reinterpret_cast<const u32x4 *>(low + fb);
      h.high[0] = *reinterpret_cast<const u32x4 *>(high + fa), h.high[1] = *reinterpret_cast<const u32x4 *>(high + fb);
    }
  }
  return h;
}

// Writes the wavefront's rows (KV heads `head` of one token; `live`: the lane's row is one) into row `row` of block `phys`.
// Chunk a of the lane starts at feature fa, chunk b at fb.  Row 0 begins the block: its scale and bounds are the row's own.  A later row may
// make the scale grow; the rows before it are then rounded again, by the whole wavefront, head after head (a block's largest
// magnitude rarely crosses a power of two behind its first rows).
template <int D>
__device__ __forceinline__ void write_row(uint8_t *cache, float *scales, uint16_t *bounds, const Caches &c, int head, bool live, int phys,
                                          int row, const RowPart &x, const Held &held, int fa, int fb) {
  constexpr int LPR = D / 16;
  const int lane = threadIdx.x & 63;
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, max(finite_magnitude(x.a[i]), finite_magnitude(x.b[i])));
  most = row_max<D>(most);
  const int64_t slab = (int64_t)phys * c.hkv + head;
  const float need = scale_for(most);
  const float old = row > 0 ? held.scale : 0.f;
  const float scale = row > 0 ? fmaxf(old, need) : need;
  if (row > 0) {
    uint64_t grown = __builtin_amdgcn_ballot_w64(live && scale > old);
    while (grown) {
      const int first = __builtin_ctzll(grown) / LPR * LPR;  // a row's lanes agree
      grown &= ~((((uint64_t)1 << LPR) - 1) << first);
      const float s_old = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, old), first));
      const float s_new = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), first));
      const int h = __builtin_amdgcn_readlane(head, first);
      // (a block that was never begun has scale 0: its rows become zeros)
      rescale_rows<D>(cache + ((int64_t)phys * c.hkv + h) * c.bs * D, row, s_old > 0.f ? s_old * inverse_scale(s_new) : 0.f);
    }
  }
  if (!live) return;
  const float inv = inverse_scale(scale);
  uint8_t *dst = cache + (slab * c.bs + row) * D;
  *reinterpret_cast<u32x2 *>(dst + fa) = encode8(x.a, inv);
  *reinterpret_cast<u32x2 *>(dst + fb) = encode8(x.b, inv);
  if (lane % LPR == 0 && scale != old) scales[slab] = scale;
  if (bounds) {
    uint16_t *low = bounds + slab * 2 * D, *high = low + D;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x4 v = half ? x.b : x.a;
      const int f = half ? fb : fa;
      u32x4 lo = held.low[half], hi = held.high[half];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (a NaN is no bound: fminf and fmaxf return the other operand; a first NaN leaves a bound that nothing passes)
        const float v0 = bf16_lo(v[i]), v1 = bf16_hi(v[i]);
        const float l0 = fminf(row > 0 ? bf16_lo(lo[i]) : INFINITY, v0), l1 = fminf(row > 0 ? bf16_hi(lo[i]) : INFINITY, v1);
        const float h0 = fmaxf(row > 0 ? bf16_lo(hi[i]) : -INFINITY, v0), h1 = fmaxf(row > 0 ? bf16_hi(hi[i]) : -INFINITY, v1);
        lo[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, l1), __builtin_bit_cast(uint32_t, l0), 0x07060302u);
        hi[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, h1), __builtin_bit_cast(uint32_t, h0), 0x07060302u);
      }
      *reinterpret_cast<u32x4 *>(low + f) = lo;
      *reinterpret_cast<u32x4 *>(high + f) = hi;
    }
  }
}

// The users of a step whose tokens go to the same block write in turn, all of them by the first one's wavefront.  Every wavefront
// therefore looks where everybody's token goes: a user per lane, four at a time, so that the look-ups of a step of up to 256 users are two round
// trips, beside the wavefront's own.
struct Turn {
  const void *pos;
  int pos_i64, users;
  __device__ __forceinline__ int64_t position(int u) const { return load_index(pos, pos_i64, u); }
};
constexpr int kTurnBatch = 4, kTurnUsers = 64 * kTurnBatch;
struct Blocks {
  int64_t pos[kTurnBatch];
  int block[kTurnBatch];
};
__device__ __forceinline__ void request_positions(const Turn &t, int first, Blocks &b) {
#pragma unroll
  for (int j = 0; j < kTurnBatch; ++j) b.pos[j] = t.position(min(first + 64 * j + (int)(threadIdx.x & 63), t.users - 1));
}
__device__ __forceinline__ void request_blocks(const Caches &c, const Turn &t, int first, Blocks &b) {
#pragma unroll
  for (int j = 0; j < kTurnBatch; ++j) {
    const int v = first + 64 * j + (int)(threadIdx.x & 63);
    int col, row;
    b.block[j] = -1;
    if (v < t.users && place_of(c, b.pos[j], col, row)) b.block[j] = c.pt[v * c.pt_rs + col];
  }
}
// Whether a user in front of u writes into its block `phys`, too, and the next one behind it that does (`users`: nobody).  `b`: the first look-ups.
__device__ inline int next_in_block(const Caches &c, const Turn &t, int u, int phys, Blocks b, bool &before) {
  const int lane = threadIdx.x & 63;
  before = false;
  int next = t.users;
  for (int at = 0;;) {
#pragma unroll
    for (int j = 0; j < kTurnBatch; ++j) {
      const int v = at + 64 * j + lane;
      const uint64_t earlier = __builtin_amdgcn_ballot_w64(b.block[j] == phys && v < u);
      const uint64_t later = __builtin_amdgcn_ballot_w64(b.block[j] == phys && v > u);
      before |= earlier != 0;
      if (later && next == t.users) next = at + 64 * j + __builtin_ctzll(later);
    }
    at += kTurnUsers;
    if (at >= t.users || next != t.users) return next;
    request_positions(t, at, b);
    request_blocks(c, t, at, b);
  }
}

}  // namespace fp8
}  // namespace ttpa
