// Prompts into the 8-bit cache: every block of a prompt gets the scale of its own rows, and the bounds of its keys.
//
// Bound by memory: a row of bfloat16 is read once and half of it written.  A workgroup owns a block of tokens of one head
// and operand, or for blocks of up to 4096 values a wavefront does; the values stay in registers (PIECES of eight per thread) between the search for
// the largest magnitude and the encoding, with one exchange through LDS in between.  16 bytes per load, 8 per store: an instruction writes 512 consecutive
// bytes.  Blocks of more values than 256 threads hold (64 KiB) are read twice (PIECES = 0), the second time from L2.
// The rows are asked for before their page is looked up (a prompt of 1999 tokens: 5.3 us; 6.9 in turn), and loads and stores are streaming
// ones: eight prompts of 4096 tokens of 8 heads of 128 (203 MB) take 41 us, 4.9 TB/s and the rate of a large copy, in blocks of 16 ... 128 tokens (64: 50
// with ordinary loads and stores; 16 and 32: 65 and 46 with a workgroup each; 128: 65 with twice the registers it needs); at head size 64 22.
// A grid with the heads of a block side by side is no faster for the workgroups' form (42).
// With a length per row of the page table the block in which a length ends asks for its rows a second time, the last that counts in place of those behind it: the other
// blocks take as long as without lengths (43, 41, 40 in blocks of 64, 16, 128; as predicates on every piece 44 in blocks of 16, and 25 for 21 at head size 64).
#include "fp8.h"

#include <algorithm>

namespace ttpa {
namespace fp8 {
int check_cache(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table, int kv_heads,
                int head_size, int block_size, int table_width, int num_blocks);

namespace {

struct FillArgs {
  Caches c;
  const uint16_t *k, *v;
  int64_t k_us, k_hs, k_ts, v_us, v_hs, v_ts;
  const void *bidx;
  int bidx_i64;
  int table_rows, s, blocks;  // blocks of a prompt
  const void *lens;  // [table_rows] rows that count of those that go to a table row's blocks, or null: all
  int lens_i64;
};

// Of `rows` rows of a block, from row `first` of a prompt on: how many count.
__device__ __forceinline__ int counted_rows(const FillArgs &a, int64_t table_row, int first, int rows) {
  return a.lens ? (int)max(min(max(load_index(a.lens, a.lens_i64, table_row), (int64_t)0) - first, (int64_t)rows), (int64_t)0) : rows;
}

// Whether a later fill row has the same index: of fill rows with one index the last one counts, so that blocks are written whole, and never with
// another row's scale.  The same in every wavefront.
__device__ __forceinline__ bool replaced(const FillArgs &a, int user, int users, int64_t table_row) {
  for (int j = user + 1; j < users; j += 64) {
    const int v = j + (int)(threadIdx.x & 63);
    if (__builtin_amdgcn_ballot_w64(v < users && load_index(a.bidx, a.bidx_i64, min(v, users - 1)) == table_row)) return true;
  }
  return false;
}
// Bounds of eight features, widened by a piece.  (A NaN is no bound: fminf and fmaxf return the other operand.)
__device__ __forceinline__ void widen(const u32x4 &w, float (&low)[8], float (&high)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    low[2 * i] = fminf(low[2 * i], bf16_lo(w[i])), low[2 * i + 1] = fminf(low[2 * i + 1], bf16_hi(w[i]));
    high[2 * i] = fmaxf(high[2 * i], bf16_lo(w[i])), high[2 * i + 1] = fmaxf(high[2 * i + 1], bf16_hi(w[i]));
  }
}
// Eight bfloat16 values held as floats, in a piece.
__device__ __forceinline__ u32x4 packed(const float (&v)[8]) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, v[2 * i + 1]), __builtin_bit_cast(uint32_t, v[2 * i]), 0x07060302u);
  return o;
}

template <int D, int PIECES>
__global__ __launch_bounds__(256) void fill_kernel(FillArgs a) {
  constexpr int CPR = D / 8;  // pieces (of eight values) per row
  __shared__ uint32_t s_most[4];
  __shared__ float s_low[4][D], s_high[4][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = blockIdx.x, user = blockIdx.z >> 1, users = gridDim.z >> 1, h = blockIdx.y;
  const bool is_v = blockIdx.z & 1;
  const int first = col * a.c.bs, rows = min(a.c.bs, a.s - first);
  const int64_t ts = is_v ? a.v_ts : a.k_ts;
  const uint16_t *src = (is_v ? a.v + user * a.v_us + h * a.v_hs : a.k + user * a.k_us + h * a.k_hs) + first * ts;
  const int f = 8 * (tid % CPR);  // the thread's features, in every piece of it
  const int pieces = rows * CPR;
  constexpr int HELD = PIECES ? PIECES : 1;
  u32x4 x[HELD];
  uint32_t most = 0;
  float low[8], high[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) low[i] = INFINITY, high[i] = -INFINITY;
  const bool bounded = !is_v && a.c.bounds;
  const auto look = [&](const u32x4 &w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, finite_magnitude(w[i]));
    if (bounded) widen(w, low, high);
  };
  const auto load = [&](int piece) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + (piece / CPR) * ts + f)); };
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
      x[j] = load(min(tid + 256 * j, pieces - 1));
  }
  // (uniform in the workgroup, like the next)
  const int64_t table_row = a.bidx ? load_index(a.bidx, a.bidx_i64, user) : 0;
  if (table_row < 0 || table_row >= a.table_rows || replaced(a, user, users, table_row)) return;
  const int phys = a.c.pt[table_row * a.c.pt_rs + col], counted = counted_rows(a, table_row, first, rows) * CPR;
  if ((unsigned)phys >= (unsigned)a.c.nb || counted == 0) return;
  if constexpr (PIECES > 0) {
    if (counted < pieces) {  // (the last ones that count again, in place of those behind)
#pragma unroll
      for (int j = 0; j < PIECES; ++j) x[j] = load(min(tid + 256 * j, counted - 1));
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) look(x[j]);  // (a piece again changes nothing)
  } else {
    for (int p = tid; p < counted; p += 256) look(load(p));
  }
  // over the wavefront, then over the workgroup
  for (int m = 1; m < 64; m <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
  if (lane == 0) s_most[wave] = most;
  if (bounded) {
#pragma unroll
    for (int m = CPR; m < 64; m <<= 1)  // the lanes of a wavefront with the same features
#pragma unroll
      for (int i = 0; i < 8; ++i) low[i] = fminf(low[i], __shfl_xor(low[i], m)), high[i] = fmaxf(high[i], __shfl_xor(high[i], m));
    if (lane < CPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s_low[wave][8 * lane + i] = low[i], s_high[wave][8 * lane + i] = high[i];
    }
  }
  __syncthreads();
  most = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
  const float scale = scale_for(most), inv = inverse_scale(scale);
  const int64_t slab = (int64_t)phys * a.c.hkv + h;
  uint8_t *dst = (is_v ? a.c.v : a.c.k) + slab * a.c.bs * D;
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
      if (tid + 256 * j < counted) __builtin_nontemporal_store(encode8(x[j], inv), reinterpret_cast<u32x2 *>(dst + 8 * (tid + 256 * j)));
  } else {
    for (int p = tid; p < counted; p += 256) *reinterpret_cast<u32x2 *>(dst + 8 * p) = encode8(load(p), inv);
  }
  if (tid == 0) (is_v ? a.c.v_scales : a.c.k_scales)[slab] = scale;
  if (bounded)
    for (int i = tid; i < 2 * D; i += 256) {
      const int g = i & (D - 1);
      const float v = i < D ? fminf(fminf(s_low[0][g], s_low[1][g]), fminf(s_low[2][g], s_low[3][g]))
                            : fmaxf(fmaxf(s_high[0][g], s_high[1][g]), fmaxf(s_high[2][g], s_high[3][g]));
      a.c.bounds[slab * 2 * D + i] = (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16);
    }
}

// The same for small blocks (up to 512 pieces): a wavefront owns a block of one head and operand, and nothing is exchanged through LDS.
template <int D, int PIECES>
__global__ __launch_bounds__(256) void fill_small_kernel(FillArgs a) {
  constexpr int CPR = D / 8;
  const int lane = threadIdx.x & 63;
  const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = (int)(unit / (uint32_t)a.c.hkv), h = (int)(unit - (uint32_t)col * a.c.hkv);  // (the heads of a block side by side)
  const int user = blockIdx.z, users = gridDim.z;
  const bool is_v = blockIdx.y;
  if (col >= a.blocks) return;
  const int first = col * a.c.bs, rows = min(a.c.bs, a.s - first);
  const int64_t ts = is_v ? a.v_ts : a.k_ts;
  const int f = 8 * (lane % CPR);
  const uint16_t *src = (is_v ? a.v + user * a.v_us + h * a.v_hs : a.k + user * a.k_us + h * a.k_hs) + first * ts + f;
  const auto load = [&](int row, int end) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + min(row, end - 1) * ts)); };
  u32x4 x[PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; ++j) x[j] = load((lane + 64 * j) / CPR, rows);
  const int64_t table_row = a.bidx ? load_index(a.bidx, a.bidx_i64, user) : 0;
  if (table_row < 0 || table_row >= a.table_rows || replaced(a, user, users, table_row)) return;
  const int phys = a.c.pt[table_row * a.c.pt_rs + col], counted = counted_rows(a, table_row, first, rows) * CPR;
  if ((unsigned)phys >= (unsigned)a.c.nb || counted == 0) return;
  if (counted < rows * CPR) {  // (the last row that counts again, in place of those behind)
#pragma unroll
    for (int j = 0; j < PIECES; ++j) x[j] = load((lane + 64 * j) / CPR, counted / CPR);
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < PIECES; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, finite_magnitude(x[j][i]));  // (a row again changes nothing)
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
  const float scale = scale_for(most), inv = inverse_scale(scale);
  const int64_t slab = (int64_t)phys * a.c.hkv + h;
  uint8_t *dst = (is_v ? a.c.v : a.c.k) + slab * a.c.bs * D;
#pragma unroll
  for (int j = 0; j < PIECES; ++j)
    if (lane + 64 * j < counted) __builtin_nontemporal_store(encode8(x[j], inv), reinterpret_cast<u32x2 *>(dst + 8 * (lane + 64 * j)));
  if (lane == 0) (is_v ? a.c.v_scales : a.c.k_scales)[slab] = scale;
  if (!is_v && a.c.bounds) {
    float low[8], high[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) low[i] = INFINITY, high[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) widen(x[j], low, high);
#pragma unroll
    for (int m = CPR; m < 64; m <<= 1)  // the lanes with the same features
#pragma unroll
      for (int i = 0; i < 8; ++i) low[i] = fminf(low[i], __shfl_xor(low[i], m)), high[i] = fmaxf(high[i], __shfl_xor(high[i], m));
    if (lane < CPR) {
      uint16_t *b = a.c.bounds + slab * 2 * D + f;
      *reinterpret_cast<u32x4 *>(b) = packed(low);
      *reinterpret_cast<u32x4 *>(b + D) = packed(high);
    }
  }
}

template <int D>
int launch_fill(const FillArgs &a, int users, hipStream_t st) {
  const dim3 grid(a.blocks, a.c.hkv, 2 * users);
  const int pieces = std::min(a.c.bs, a.s) * (D / 8);
  const dim3 small((unsigned)(((int64_t)a.blocks * a.c.hkv + 3) / 4), 2, users);
  if (pieces <= 128) fill_small_kernel<D, 2><<<small, dim3(256), 0, st>>>(a);
  else if (pieces <= 256) fill_small_kernel<D, 4><<<small, dim3(256), 0, st>>>(a);
  else if (pieces <= 512) fill_small_kernel<D, 8><<<small, dim3(256), 0, st>>>(a);
  else if (pieces <= 1024) fill_kernel<D, 4><<<grid, dim3(256), 0, st>>>(a);
  else if (pieces <= 2048) fill_kernel<D, 8><<<grid, dim3(256), 0, st>>>(a);
  else if (pieces <= 4096) fill_kernel<D, 16><<<grid, dim3(256), 0, st>>>(a);
  else fill_kernel<D, 0><<<grid, dim3(256), 0, st>>>(a);
  return check_launch("fp8 fill");
}

}  // namespace
}  // namespace fp8
}  // namespace ttpa

using namespace ttpa;

extern "C" int ttpa_paged_fill_fp8_cache_lens(void *k_cache, void *v_cache, float *k_scales, float *v_scales, void *key_bounds, const void *k_fill,
                                              int64_t k_user_stride, int64_t k_head_stride, int64_t k_token_stride, const void *v_fill,
                                              int64_t v_user_stride, int64_t v_head_stride, int64_t v_token_stride, const int32_t *page_table,
                                              int64_t page_table_row_stride, const void *batch_idx, int batch_idx_is_i64, const void *lens,
                                              int lens_is_i64, int32_t fill_users, int32_t table_rows, int32_t kv_heads, int32_t seq_len,
                                              int32_t block_size, int32_t head_size, int32_t table_width, int32_t num_blocks, void *stream) {
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  TTPA_REQUIRE(k_fill && v_fill, "fp8 fill: null pointer argument");
  TTPA_REQUIRE(fill_users >= 0 && seq_len >= 0 && table_rows > 0, "fp8 fill: non-positive dimension");
  TTPA_REQUIRE(batch_idx != nullptr || fill_users <= 1, "fp8 fill: batch_idx may only be omitted for a single user");
  TTPA_REQUIRE((int64_t)seq_len <= (int64_t)table_width * block_size, "fp8 fill: seq_len %d does not fit %d page-table columns of %d tokens",
               seq_len, table_width, block_size);
  TTPA_REQUIRE(fill_users < 32768 && kv_heads < 65536 && (int64_t)((seq_len - 1) / block_size) * kv_heads < (1 << 25) &&
                   (seq_len - 1) / block_size < (1 << 23), "fp8 fill: too many users, heads or blocks for one launch");
  TTPA_REQUIRE(aligned16(k_fill) && aligned16(v_fill) && (!key_bounds || aligned16(key_bounds)) && k_user_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                   k_token_stride % 8 == 0 && v_user_stride % 8 == 0 && v_head_stride % 8 == 0 && v_token_stride % 8 == 0,
               "fp8 fill: rows and bounds must be 16-byte aligned, strides multiples of 8 elements");
  if (fill_users == 0 || seq_len == 0) return TTPA_OK;
  fp8::FillArgs a = {{static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache), k_scales, v_scales, static_cast<uint16_t *>(key_bounds),
                      page_table, page_table_row_stride, kv_heads, block_size, table_width, num_blocks, fp8::block_inverse(block_size)},
                     static_cast<const uint16_t *>(k_fill), static_cast<const uint16_t *>(v_fill), k_user_stride, k_head_stride, k_token_stride,
                     v_user_stride, v_head_stride, v_token_stride, batch_idx, batch_idx_is_i64, table_rows, seq_len,
                     (seq_len + block_size - 1) / block_size, lens, lens_is_i64};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (head_size) {
    case 64: return fp8::launch_fill<64>(a, fill_users, st);
    case 128: return fp8::launch_fill<128>(a, fill_users, st);
    default: return fp8::launch_fill<256>(a, fill_users, st);
  }
}

extern "C" int ttpa_paged_fill_fp8_cache(void *k_cache, void *v_cache, float *k_scales, float *v_scales, void *key_bounds, const void *k_fill,
                                         int64_t k_user_stride, int64_t k_head_stride, int64_t k_token_stride, const void *v_fill,
                                         int64_t v_user_stride, int64_t v_head_stride, int64_t v_token_stride, const int32_t *page_table,
                                         int64_t page_table_row_stride, const void *batch_idx, int batch_idx_is_i64, int32_t fill_users,
                                         int32_t table_rows, int32_t kv_heads, int32_t seq_len, int32_t block_size, int32_t head_size,
                                         int32_t table_width, int32_t num_blocks, void *stream) {
  return ttpa_paged_fill_fp8_cache_lens(k_cache, v_cache, k_scales, v_scales, key_bounds, k_fill, k_user_stride, k_head_stride, k_token_stride, v_fill,
                                        v_user_stride, v_head_stride, v_token_stride, page_table, page_table_row_stride, batch_idx, batch_idx_is_i64,
                                        nullptr, 0, fill_users, table_rows, kv_heads, seq_len, block_size, head_size, table_width, num_blocks, stream);
}
