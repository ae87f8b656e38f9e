// Attention of a prompt's chunk over the 8-bit cache: the blocks that the pass reads become bfloat16 copies in the caller's scratch, unless the chunk has few rows
// (fp8_chunk_few.hip); exactly, as an element times its block's power of two is a bfloat16 value.  The bfloat16 prefill kernels run over the copies.
//
// A chunk is bound by its matrix products, 4 D q_heads operations per (row, key) pair, and every workgroup of 128 rows reads every key, so keys
// are expanded once here and not once per workgroup; the copies cost 1 byte read and 2 written per element, at the rate of a large
// copy: 22 us for 4 x 4608 keys of 8 heads (113 MB; 27 when every piece of 512 elements looked its block up), 13 for 8704 (53 MB).
// The pass as a whole takes 284 us there (where both were timed in turn, 292, and 298 with the piece-wise look-up).
// The blocks are read by streaming loads and the copies written by ordinary stores: what follows reads them from the caches.
//
// The prefill kernels take keys by tiles of 64 and give what is behind the last row's own position weight zero, whatever it is, so it has to be
// numbers: rows behind the chunk are copied as zeros, up to the end of the tile, and block 0 of the copies, which stands in for
// whatever the table does not hold, is zeros.
#include "fp8.h"

#include <algorithm>
#include <cstdlib>
#include <cstring>

namespace ttpa {
namespace fp8 {
int check_cache(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table, int kv_heads,
                int head_size, int block_size, int table_width, int num_blocks);

// A chunk of few rows (fp8_chunk_few.hip).
int64_t chunk_few_bytes(int batch, int q_heads, int kv_heads, int q_len, int head_size, int64_t keys);
double chunk_few_us(int batch, int q_heads, int kv_heads, int q_len, int head_size, int64_t keys);
int chunk_few(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q, int64_t q_batch_stride,
              int64_t q_head_stride, int64_t q_token_stride, const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
              const int32_t *page_table, int64_t page_table_row_stride, const int32_t *chunk_start, int batch, int q_heads, int kv_heads, int q_len,
              int head_size, int block_size, int table_width, int num_blocks, float scale, int64_t keys, void *workspace, hipStream_t st);

namespace {

// Keys that the host knows a pass to read at most.  (Both forms take the table as if it ended with the block that holds the last of them.)
int64_t keys_at_most(int block_size, int table_width, int64_t most_keys) {
  const int64_t room = (int64_t)table_width * block_size;
  return most_keys > 0 ? std::min(most_keys, room) : room;
}
// Whether the cache is read as it is, and not by copies; TTPA_CHUNK_FORM=few|copies (read on every call) overrides.  By what the two are expected to
// take: the copies 20 us (24 at head size 256), their bytes at the rate of a large copy and the products at 1.2 PFLOP/s (32/8 heads of 128, one user: 128 rows of a
// KV head behind 8192 tokens 37, expected 34, 512 45 (45), 768 54 (52); five users behind 4096: 128 51 (55), 512 82 (84)).  Chosen so, us copies / few rows: 512 rows
// behind 8192 45 / 41, 768 54 / 62; five users, 384 rows 72 / 60, 512 82 / 87; behind 1000 tokens 512 rows 23 / 17, 768 26 / 20; of 256, 256 rows behind 8192 58 / 53, 384 64 / 80.
bool few_rows(int batch, int q_heads, int kv_heads, int q_len, int head_size, int64_t keys) {
  const char *form = getenv("TTPA_CHUNK_FORM");
  if (form && !strcmp(form, "few")) return true;
  if (form && !strcmp(form, "copies")) return false;
  if ((int64_t)batch * kv_heads * ((int64_t)(q_heads / kv_heads) * q_len / 32 + 1) >= (1 << 18)) return false;  // (more than its grid takes)
  const double values = (double)batch * kv_heads * keys * head_size, flops = 4.0 * batch * q_heads * q_len * (double)keys * head_size;
  return chunk_few_us(batch, q_heads, kv_heads, q_len, head_size, keys) < (head_size <= 128 ? 20.0 : 24.0) + 6.0 * values / 4.9e6 + flops / 1.2e9;
}

struct ExpandArgs {
  const uint8_t *k, *v;
  const float *k_scales, *v_scales;
  uint16_t *k_copy, *v_copy;  // [1 + batch * width][kv_heads][block_size][head_size]
  int32_t *table;             // [batch][width]: the copies' page table
  const int32_t *pt;
  int64_t pt_rs;
  const int32_t *chunk_start;
  int batch, w, hkv, bs, nb, q_len, d;
};

constexpr int kExpandWorkgroups = 16384, kPieces = 4;

// A workgroup takes blocks of one head and operand (blockIdx.y), by pieces of 2048 elements.
__global__ __launch_bounds__(256) void fp8_expand_kernel(ExpandArgs e) {
  // keys 0 .. chunk_start + q_len - 1 are read, in tiles of 64
  const int64_t end = (int64_t)(e.chunk_start ? max(*e.chunk_start, 0) : 0) + e.q_len;
  const uint32_t cols = (uint32_t)min((int64_t)e.w, ((end + 63) / 64 * 64 + e.bs - 1) / e.bs);
  const int slab = blockIdx.y;
  if (slab == 0)
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < (uint32_t)e.batch * e.w; i += gridDim.x * 256)
      e.table[i] = i % (uint32_t)e.w < cols ? (int)i + 1 : 0;
  const bool is_v = slab >= e.hkv;
  const int h = slab - (is_v ? e.hkv : 0);
  const uint8_t *src = is_v ? e.v : e.k;
  const float *scales = is_v ? e.v_scales : e.k_scales;
  uint16_t *copy = is_v ? e.v_copy : e.k_copy;
  const int elements = e.bs * e.d, pieces = elements / 2048;
  const uint32_t blocks = (uint32_t)e.batch * cols + 1;
  for (uint32_t r = blockIdx.x; r < blocks; r += gridDim.x) {
    // r = 0: the block of zeros; then the users' columns
    const uint32_t b = r ? (r - 1) / cols : 0, col = r ? r - 1 - b * cols : 0;
    const int64_t x = r ? (int64_t)b * e.w + col + 1 : 0;
    int phys = e.pt[(int64_t)b * e.pt_rs + col];
    if ((unsigned)phys >= (unsigned)e.nb) phys = 0;
    const int64_t from = (int64_t)phys * e.hkv + h;
    const uint8_t *in = src + from * elements;
    uint16_t *out = copy + (x * e.hkv + h) * elements;
    const int64_t left = r ? (end - (int64_t)col * e.bs) * e.d : 0;  // elements of the block in front of the chunk's end
    const float scale = scales[from];
    for (int p = 0; p < pieces; p += kPieces) {
      u32x2 raw[kPieces];
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        raw[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(in + 2048 * min(p + j, pieces - 1)) + threadIdx.x);
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int at = 2048 * (p + j) + 8 * (int)threadIdx.x;
        if (p + j < pieces) *reinterpret_cast<u32x4 *>(out + at) = at < left ? decode8(raw[j].x, raw[j].y, scale) : u32x4{0, 0, 0, 0};
      }
    }
  }
}

struct ChunkLayout {
  int width;       // columns of the copies
  int64_t copy, table, parts;
};
ChunkLayout chunk_layout(int batch, int q_heads, int kv_heads, int q_len, int head_size, int block_size, int table_width, int64_t most_keys) {
  ChunkLayout l;
  const int64_t keys = most_keys > 0 ? std::min<int64_t>(most_keys, (int64_t)table_width * block_size) : (int64_t)table_width * block_size;
  l.width = (int)((keys + block_size - 1) / block_size);
  l.copy = ((int64_t)batch * l.width + 1) * kv_heads * block_size * head_size * 2;
  l.table = ((int64_t)batch * l.width * 4 + 255) / 256 * 256;
  l.parts = ttpa_sdpa_prefill_bounded_scratch_bytes(batch, q_heads, kv_heads, q_len, head_size, block_size, l.width, TTPA_KV_BF16, most_keys);
  return l;
}

}  // namespace
}  // namespace fp8
}  // namespace ttpa

using namespace ttpa;

extern "C" int64_t ttpa_chunked_fp8_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t q_len, int32_t head_size,
                                                              int32_t block_size, int32_t table_width, int64_t most_keys) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_len <= 0 || head_size <= 0 || block_size <= 0 || table_width <= 0)
    return 0;
  const int64_t keys = fp8::keys_at_most(block_size, table_width, most_keys);
  if (fp8::few_rows(batch, q_heads, kv_heads, q_len, head_size, keys)) return fp8::chunk_few_bytes(batch, q_heads, kv_heads, q_len, head_size, keys);
  const fp8::ChunkLayout l = fp8::chunk_layout(batch, q_heads, kv_heads, q_len, head_size, block_size, table_width, most_keys);
  return 2 * l.copy + l.table + l.parts;
}

extern "C" int ttpa_chunked_fp8_attention(void *out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_token_stride, const void *q,
                                          int64_t q_batch_stride, int64_t q_head_stride, int64_t q_token_stride, const void *k_cache,
                                          const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *page_table,
                                          int64_t page_table_row_stride, const int32_t *chunk_start, int32_t batch, int32_t q_heads,
                                          int32_t kv_heads, int32_t q_len, int32_t head_size, int32_t block_size, int32_t table_width,
                                          int32_t num_blocks, float scale, int64_t most_keys, void *workspace, int64_t workspace_bytes,
                                          void *stream) {
  if (int rc = fp8::check_cache(k_cache, v_cache, k_scales, v_scales, page_table, kv_heads, head_size, block_size, table_width, num_blocks)) return rc;
  TTPA_REQUIRE(out && q, "fp8 chunk: null pointer argument");
  TTPA_REQUIRE(batch > 0 && q_heads > 0 && q_len > 0 && most_keys >= 0, "fp8 chunk: non-positive dimension");
  TTPA_REQUIRE(q_heads % kv_heads == 0, "fp8 chunk: q_heads %d not divisible by kv_heads %d", q_heads, kv_heads);
  if (block_size % 32) return fail(TTPA_ERR_UNSUPPORTED, "fp8 chunk: block_size %d must be a multiple of 32", block_size);
  const int64_t keys = fp8::keys_at_most(block_size, table_width, most_keys);
  const bool few = fp8::few_rows(batch, q_heads, kv_heads, q_len, head_size, keys);
  const fp8::ChunkLayout l = few ? fp8::ChunkLayout{} : fp8::chunk_layout(batch, q_heads, kv_heads, q_len, head_size, block_size, table_width, most_keys);
  const int64_t need = ttpa_chunked_fp8_attention_workspace_bytes(batch, q_heads, kv_heads, q_len, head_size, block_size, table_width, most_keys);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(TTPA_ERR_WORKSPACE, "fp8 chunk: workspace of %lld bytes (256-byte aligned) required, got %lld", (long long)need,
                (long long)workspace_bytes);
  if (few) {
    TTPA_REQUIRE(aligned16(q) && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0 && q_token_stride % 8 == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 7u) == 0 && out_batch_stride % 4 == 0 && out_head_stride % 4 == 0 && out_token_stride % 4 == 0 && scale > 0,
                 "fp8 chunk: q must be 16-byte aligned, its strides multiples of 8 elements, the output's of 4, the scale positive");
    return fp8::chunk_few(out, out_batch_stride, out_head_stride, out_token_stride, q, q_batch_stride, q_head_stride, q_token_stride, k_cache, v_cache,
                          k_scales, v_scales, page_table, page_table_row_stride, chunk_start, batch, q_heads, kv_heads, q_len, head_size, block_size,
                          (int)((keys + block_size - 1) / block_size), num_blocks, scale, keys, workspace, static_cast<hipStream_t>(stream));
  }
  TTPA_REQUIRE((int64_t)batch * l.width < (1ll << 31) - 2 && kv_heads < 32768, "fp8 chunk: too many blocks or heads");
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  fp8::ExpandArgs e = {static_cast<const uint8_t *>(k_cache), static_cast<const uint8_t *>(v_cache), k_scales, v_scales,
                       reinterpret_cast<uint16_t *>(ws), reinterpret_cast<uint16_t *>(ws + l.copy), reinterpret_cast<int32_t *>(ws + 2 * l.copy),
                       page_table, page_table_row_stride, chunk_start, batch, l.width, kv_heads, block_size, num_blocks, q_len, head_size};
  hipStream_t st = static_cast<hipStream_t>(stream);
  // armed events: the pair brackets both launches
  hipEvent_t before, after;
  take_profile_events(before, after);
  const dim3 grid((unsigned)std::min<int64_t>((int64_t)batch * l.width + 1, std::max(1, fp8::kExpandWorkgroups / (2 * kv_heads))), 2 * kv_heads);
  if (before)
    hipExtLaunchKernelGGL(fp8::fp8_expand_kernel, grid, dim3(256), 0u, st, before, nullptr, 0u, e);
  else
    fp8::fp8_expand_kernel<<<grid, dim3(256), 0, st>>>(e);
  if (const int rc = check_launch("fp8 chunk (expansion)")) return rc;
  if (after) arm_profile_events(nullptr, after);
  return ttpa_sdpa_prefill_bounded(out, out_batch_stride, out_head_stride, out_token_stride, q, q_batch_stride, q_head_stride, q_token_stride,
                                   e.k_copy, e.v_copy, 0, 0, 0, e.table, l.width, chunk_start, nullptr, 0, 0, batch, q_heads, kv_heads, q_len,
                                   l.width * block_size, head_size, block_size, l.width, batch * l.width + 1, 1, scale, 0, TTPA_KV_BF16, most_keys,
                                   l.parts ? ws + 2 * l.copy + l.table : nullptr, l.parts, stream);
}
