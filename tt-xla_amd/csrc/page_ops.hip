// Moves inside paged caches, for all layers in one call: copies of whole blocks (forks of sequences, moves of pages) and compaction of sequences
// (chosen tokens move together).  Bytes are moved as they are, so any element type will do.  Both are bound by memory: read once, written once; a large copy by torch
// reaches 5.3 TB/s both ways together on this card.  Three states in turn: 250 blocks of 64 x 8 heads x 128 bytes in 24 caches (786 MB) 153 us, 5.1 TB/s; half of the
// last three quarters of 4 x 8192 tokens, K and V of 16 layers of 8 heads of 128 (1.6 GB), 326 us, 4.9; of 2048 ... 8192 tokens (867 MB), where the longest user's
// chain of batches ends the launch, 200 us, 4.3.  (Of one state again and again, of which the last cache holds a part, the last takes 175 us; 203 with one batch on its way and
// 191 with streaming stores, where these took 178.)
#include "common.h"

#include <algorithm>

namespace ttpa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMostCaches = 192;        // of one launch: their addresses are arguments
constexpr int kMostPairs = 4096;        // of one launch: a longer list takes several, one after the other
constexpr int kMostMarks = 1 << 18;     // blocks of a cache that a workgroup can mark (32 KiB of LDS)
constexpr int kThreads = 256, kChunks = 4, kAtOnce = 2;  // 16-byte chunks of a block per thread, pairs on their way at a time

struct CopyArgs {
  uint8_t *caches[kMostCaches];
  uint32_t block_units[kMostCaches];  // of what a thread moves at a time
  const int32_t *source, *target;
  int pairs, nb, parts;
};

__device__ __forceinline__ bool copies(const CopyArgs &a, int s, int t) { return (unsigned)s < (unsigned)a.nb && (unsigned)t < (unsigned)a.nb && s != t; }

// Whether a block is the target of two pairs, or of one and the source of another: only then does the order of the pairs matter.
__device__ __forceinline__ bool order_matters(const CopyArgs &a, uint32_t *marks) {
  if (a.pairs == 1) return false;
  const int lane = threadIdx.x & 63;
  if (a.pairs <= 64) {
    int s = -1, t = -1;
    if (lane < a.pairs) s = a.source[lane], t = a.target[lane];
    const bool mine = lane < a.pairs && copies(a, s, t);
    bool found = false;
    for (int i = 0; i < a.pairs; ++i) {
      const int other = __builtin_amdgcn_readlane(t, i), live = __builtin_amdgcn_readlane((int)mine, i);
      found = found || (live && mine && lane != i && (s == other || t == other));
    }
    return __builtin_amdgcn_ballot_w64(found) != 0;
  }
  __shared__ int s_found;
  if (threadIdx.x == 0) s_found = 0;
  for (int i = threadIdx.x; i < (a.nb + 31) / 32; i += kThreads) marks[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.pairs; i += kThreads) {
    const int s = a.source[i], t = a.target[i];
    if (copies(a, s, t) && (atomicOr(marks + (t >> 5), 1u << (t & 31)) >> (t & 31) & 1u)) s_found = 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.pairs; i += kThreads) {
    const int s = a.source[i], t = a.target[i];
    if (copies(a, s, t) && (marks[s >> 5] >> (s & 31) & 1u)) s_found = 1;
  }
  __syncthreads();
  return s_found != 0;
}

// A workgroup has kThreads * kChunks chunks of every block of one cache, and every `parts`-th run of kAtOnce pairs.  A thread has the same bytes of every block,
// so pairs that depend on each other are its own business: where the order matters, the workgroups of part 0 take all pairs one by one.
template <typename T>
__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(CopyArgs a) {
  extern __shared__ uint32_t marks[];
  const int part = blockIdx.z;
  const int64_t block_bytes = (int64_t)a.block_units[blockIdx.y] * (int64_t)sizeof(T), first = ((int64_t)blockIdx.x * (kThreads * kChunks) + threadIdx.x) * (int64_t)sizeof(T);
  if ((int64_t)blockIdx.x * (kThreads * kChunks) * (int64_t)sizeof(T) >= block_bytes) return;  // (another cache's blocks are larger)
  const bool ordered = order_matters(a, marks);
  if (ordered && part > 0) return;
  uint8_t *const cache = a.caches[blockIdx.y];
  constexpr int kStep = kThreads * (int)sizeof(T);
  if (ordered) {
    for (int j = 0; j < a.pairs; ++j) {
      const int s = a.source[j], t = a.target[j];
      if (!copies(a, s, t)) continue;
      T x[kChunks];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        if (first + c * kStep < block_bytes) x[c] = *reinterpret_cast<const T *>(cache + s * block_bytes + first + c * kStep);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        if (first + c * kStep < block_bytes) *reinterpret_cast<T *>(cache + t * block_bytes + first + c * kStep) = x[c];
    }
    return;
  }
  for (int j0 = part * kAtOnce; j0 < a.pairs; j0 += a.parts * kAtOnce) {
    T x[kAtOnce][kChunks];
    int s[kAtOnce], t[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int j = min(j0 + i, a.pairs - 1);
      s[i] = a.source[j], t[i] = a.target[j];
      if (j0 + i >= a.pairs) t[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (copies(a, s[i], t[i])) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (first + c * kStep < block_bytes) x[i][c] = __builtin_nontemporal_load(reinterpret_cast<const T *>(cache + s[i] * block_bytes + first + c * kStep));
      }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (copies(a, s[i], t[i])) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (first + c * kStep < block_bytes) __builtin_nontemporal_store(x[i][c], reinterpret_cast<T *>(cache + t[i] * block_bytes + first + c * kStep));
      }
  }
}

struct KeepArgs {
  uint8_t *caches[kMostCaches];
  const int32_t *pt, *kept, *kept_lens, *first;
  int64_t pt_rs, kept_rs;
  int most, hkv, bs, w, nb, row_bytes, n_caches, at_once;  // at_once: caches that a workgroup of few rows takes
  int col_shift;  // log2 of the 16-byte chunks of a row that a workgroup takes
};

// Where the rows of one user and head go: row first + i takes what row kept[i] held.  A row never moves back: an entry that would is skipped, and so is what stays where it
// is, or lies outside the table's room or the cache.
struct KeepPlan {
  const KeepArgs &a;
  const int u, h, n;
  const int64_t first;
  struct Pages {
    int from, to;
  };
  struct Offsets {
    int64_t from, to;  // bytes in a cache, or -1
  };
  __device__ __forceinline__ KeepPlan(const KeepArgs &args, int user, int head)
      : a(args), u(user), h(head), n(max(min(args.kept_lens[user], args.most), 0)), first(args.first ? args.first[user] : 0) {}
  __device__ __forceinline__ int entry(int64_t i) const { return i < n ? a.kept[u * a.kept_rs + i] : -1; }
  __device__ __forceinline__ bool moves(int64_t i, int s) const { return first + i >= 0 && (int64_t)s > first + i && s < (int64_t)a.w * a.bs; }
  __device__ __forceinline__ Pages pages(int64_t i, int s) const {
    Pages p = {-1, -1};
    if (moves(i, s)) p.from = a.pt[u * a.pt_rs + s / a.bs], p.to = a.pt[u * a.pt_rs + (int)(first + i) / a.bs];
    return p;
  }
  __device__ __forceinline__ Offsets offsets(int64_t i, int s, const Pages &p) const {
    Offsets o = {-1, -1};
    if (moves(i, s) && (unsigned)p.from < (unsigned)a.nb && (unsigned)p.to < (unsigned)a.nb) {
      o.from = (((int64_t)p.from * a.hkv + h) * a.bs + s % a.bs) * a.row_bytes;
      o.to = (((int64_t)p.to * a.hkv + h) * a.bs + (int)(first + i) % a.bs) * a.row_bytes;
    }
    return o;
  }
};

// Many rows of one user and head of one cache, in batches in order.  No row is read behind the batch that overwrites it (rows do not move back), and all rows of a
// batch are read before one of them is written: a barrier per batch.  Two batches of rows are on their way, and the pages and entries of the next two.
__global__ __launch_bounds__(256) void keep_rows_kernel(KeepArgs a) {
  constexpr int U = 8, THREADS = 256;
  __shared__ KeepPlan::Offsets s_plan[3][THREADS];
  const int u = blockIdx.x / a.hkv;
  const KeepPlan plan(a, u, blockIdx.x - u * a.hkv);
  if (plan.n == 0) return;
  const int cols = 1 << a.col_shift, col = threadIdx.x & (cols - 1), row = (int)threadIdx.x >> a.col_shift;
  const int per = THREADS >> a.col_shift, batch = min(per * U, THREADS), batches = (plan.n + batch - 1) / batch;  // rows of a pass, of a batch
  uint8_t *const cache = a.caches[blockIdx.y] + (int64_t)(((int)blockIdx.z << a.col_shift) + col) * 16;
  // thread j plans row j of a batch
  const auto at = [&](int b) { return (int64_t)b * batch + threadIdx.x; };
  const bool plans = (int)threadIdx.x < batch;
  const auto put = [&](int b, int s, const KeepPlan::Pages &p) {
    if (plans) s_plan[b % 3][threadIdx.x] = plan.offsets(at(b), s, p);
  };
  u32x4 x[2][U];
  const auto load = [&](int b, u32x4 (&v)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = row + i * per;
      const int64_t from = b < batches && r < batch ? s_plan[b % 3][r].from : -1;
      if (from >= 0) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(cache + from));
    }
  };
  const int s0 = plan.entry(at(0)), s1 = plan.entry(at(1));
  int s2 = plan.entry(at(2)), s3 = plan.entry(at(3));
  put(0, s0, plan.pages(at(0), s0)), put(1, s1, plan.pages(at(1), s1));
  KeepPlan::Pages p2 = plan.pages(at(2), s2);
  __syncthreads();  // the first two plans are there
  load(0, x[0]);
  const auto step = [&](int b, u32x4 (&now)[U], u32x4 (&next)[U]) {
    load(b + 1, next);
    put(b + 2, s2, p2);
    s2 = s3, p2 = plan.pages(at(b + 3), s2), s3 = plan.entry(at(b + 4));
    int64_t to[U];
#pragma unroll
    for (int i = 0; i < U; ++i) to[i] = row + i * per < batch ? s_plan[b % 3][row + i * per].to : -1;
#pragma unroll
    for (int i = 0; i < U; ++i) asm volatile("" : "+v"(now[i]));  // (they have arrived)
    __syncthreads();  // everybody has read batch b, and plan b + 2 is there
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (to[i] >= 0) *reinterpret_cast<u32x4 *>(cache + to[i]) = now[i];
  };
  for (int b = 0; b < batches; b += 2) {
    step(b, x[0], x[1]);
    if (b + 1 < batches) step(b + 1, x[1], x[0]);
  }
}

// Few rows (no more than a wavefront takes in a pass of U loads): one wavefront per user and head plans them once and moves them in up to kCachesAtOnce caches, one after
// the other with the next one's rows on their way.  32 users' six of 16 drafted tokens, K and V of 32 layers of 8 heads of 128 (50 MB): 11.2 us, 13.4 with a wavefront per
// cache; one user's 20 of 40 3.5.
constexpr int kCachesAtOnce = 8, kFewPasses = 8;
__global__ __launch_bounds__(64) void keep_few_rows_kernel(KeepArgs a) {
  constexpr int U = kFewPasses;
  __shared__ KeepPlan::Offsets s_plan[64];
  const int u = blockIdx.x / a.hkv;
  const KeepPlan plan(a, u, blockIdx.x - u * a.hkv);
  if (plan.n == 0) return;
  const int cols = 1 << a.col_shift, col = threadIdx.x & (cols - 1), row = (int)threadIdx.x >> a.col_shift, per = 64 >> a.col_shift;
  const int s = plan.entry(threadIdx.x);
  s_plan[threadIdx.x] = plan.offsets(threadIdx.x, s, plan.pages(threadIdx.x, s));
  __syncthreads();
  int64_t from[U], to[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int r = row + i * per;
    from[i] = r < min(plan.n, 64) ? s_plan[r].from : -1, to[i] = r < min(plan.n, 64) ? s_plan[r].to : -1;
  }
  const int64_t chunk = (int64_t)(((int)blockIdx.z << a.col_shift) + col) * 16;
  const int c0 = blockIdx.y * a.at_once, end = min(c0 + a.at_once, a.n_caches);
  u32x4 x[2][U];
  const auto load = [&](int c, u32x4 (&v)[U]) {
    const uint8_t *const cache = a.caches[min(c, a.n_caches - 1)] + chunk;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i * per < plan.n && from[i] >= 0) v[i] = *reinterpret_cast<const u32x4 *>(cache + from[i]);
  };
  const auto step = [&](int c, u32x4 (&now)[U], u32x4 (&next)[U]) {
    load(c + 1, next);
#pragma unroll
    for (int i = 0; i < U; ++i) asm volatile("" : "+v"(now[i]));  // (all of a cache's rows have arrived before one of them is written)
    uint8_t *const cache = a.caches[c] + chunk;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i * per < plan.n && to[i] >= 0) *reinterpret_cast<u32x4 *>(cache + to[i]) = now[i];
  };
  load(c0, x[0]);
  for (int c = c0; c < end; c += 2) {
    step(c, x[0], x[1]);
    if (c + 1 < end) step(c + 1, x[1], x[0]);
  }
}

int check_caches(const char *what, void *const *caches, int n) {
  TTPA_REQUIRE(n >= 0 && (n == 0 || caches), "%s: null pointer argument", what);
  for (int i = 0; i < n; ++i) TTPA_REQUIRE(caches[i], "%s: null cache", what);
  return TTPA_OK;
}

template <typename T>
int launch_copy(CopyArgs &a, int caches, hipStream_t st) {
  int64_t most = 0, all = 0;
  for (int i = 0; i < caches; ++i) most = std::max<int64_t>(most, a.block_units[i]), all += a.block_units[i];
  const int64_t slices = (most + kThreads * kChunks - 1) / (kThreads * kChunks), busy = (all + kThreads * kChunks - 1) / (kThreads * kChunks);
  // Workgroups for every CU many times over, a run of pairs each at least: 250 blocks of 64 KiB in 24 caches, three states in turn, 159 us with eight per CU and four pairs
  // on their way, 154 with sixteen and two, 151 with sixty-four and one, which takes blocks of 8 KiB 14 % longer
  const int64_t runs = (a.pairs + kAtOnce - 1) / kAtOnce, want = (16ll * std::max(device_cus(), 1) + busy - 1) / busy;
  a.parts = (int)std::max<int64_t>(1, std::min(runs, want));
  const size_t lds = a.pairs > 64 ? (size_t)(a.nb + 31) / 32 * 4 : 0;
  copy_blocks_kernel<T><<<dim3((unsigned)slices, (unsigned)caches, (unsigned)a.parts), dim3(kThreads), lds, st>>>(a);
  return check_launch("copy_cache_blocks");
}

}  // namespace
}  // namespace ttpa

using namespace ttpa;

extern "C" int ttpa_copy_cache_blocks(void *const *caches_host, const int64_t *block_bytes_host, int32_t n_caches, const int32_t *source_blocks,
                                      const int32_t *target_blocks, int32_t pairs, int32_t num_blocks, void *stream) {
  if (int rc = check_caches("copy_cache_blocks", caches_host, n_caches)) return rc;
  TTPA_REQUIRE(source_blocks && target_blocks && (n_caches == 0 || block_bytes_host), "copy_cache_blocks: null pointer argument");
  TTPA_REQUIRE(num_blocks > 0 && pairs >= 0, "copy_cache_blocks: non-positive dimension");
  for (int i = 0; i < n_caches; ++i)
    TTPA_REQUIRE(block_bytes_host[i] > 0 && block_bytes_host[i] < (1ll << 31), "copy_cache_blocks: blocks of %lld bytes; supported are 1 to 2^31 - 1",
                 (long long)block_bytes_host[i]);
  hipStream_t st = static_cast<hipStream_t>(stream);
  CopyArgs a = {};
  a.nb = num_blocks;
  const auto unit_of = [&](int i) {
    const uint64_t bits = (uint64_t)block_bytes_host[i] | reinterpret_cast<uint64_t>(caches_host[i]);
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  };
  const int32_t most = num_blocks <= kMostMarks ? kMostPairs : 64;  // (more blocks than can be marked: pairs that a wavefront compares)
  for (int32_t p0 = 0; p0 < pairs; p0 += std::min(pairs - p0, most)) {
    a.source = source_blocks + p0, a.target = target_blocks + p0, a.pairs = std::min(pairs - p0, most);
    for (const int unit : {16, 4, 1})  // (caches of one unit together, for twelve 8-bit layers with their bounds and scales one launch, not three: 1 block 6.5 -> 2.9 us, 8 13.3 -> 7.8)
      for (int32_t i = 0; i < n_caches;) {
        int n = 0;
        for (; i < n_caches && n < kMostCaches; ++i)
          if (unit_of(i) == unit) a.caches[n] = static_cast<uint8_t *>(caches_host[i]), a.block_units[n++] = (uint32_t)(block_bytes_host[i] / unit);
        if (n == 0) continue;
        const int rc = unit == 16 ? launch_copy<u32x4>(a, n, st) : unit == 4 ? launch_copy<uint32_t>(a, n, st) : launch_copy<uint8_t>(a, n, st);
        if (rc) return rc;
      }
  }
  return TTPA_OK;
}

extern "C" int ttpa_keep_cache_tokens(void *const *caches_host, int32_t n_caches, const int32_t *page_table, int64_t page_table_row_stride,
                                      const int32_t *kept, int64_t kept_row_stride, const int32_t *kept_lens, const int32_t *first, int32_t users,
                                      int32_t most_kept, int32_t heads, int32_t row_bytes, int32_t block_size, int32_t table_width,
                                      int32_t num_blocks, void *stream) {
  if (int rc = check_caches("keep_cache_tokens", caches_host, n_caches)) return rc;
  TTPA_REQUIRE(page_table && kept && kept_lens, "keep_cache_tokens: null pointer argument");
  TTPA_REQUIRE(users >= 0 && most_kept >= 0 && heads > 0 && row_bytes > 0 && block_size > 0 && table_width > 0 && num_blocks > 0,
               "keep_cache_tokens: non-positive dimension");
  if (row_bytes % 16) return fail(TTPA_ERR_UNSUPPORTED, "keep_cache_tokens: rows of %d bytes; supported are multiples of 16", row_bytes);
  TTPA_REQUIRE((int64_t)table_width * block_size < (1ll << 31), "keep_cache_tokens: a page-table row holds too many tokens");
  TTPA_REQUIRE((int64_t)users * heads < (1ll << 24) && row_bytes / 16 < (1 << 16), "keep_cache_tokens: too many rows for one launch");
  for (int i = 0; i < n_caches; ++i) TTPA_REQUIRE(aligned16(caches_host[i]), "keep_cache_tokens: caches must be 16-byte aligned");
  if (users == 0 || most_kept == 0) return TTPA_OK;
  KeepArgs a = {};
  a.pt = page_table, a.pt_rs = page_table_row_stride, a.kept = kept, a.kept_rs = kept_row_stride, a.kept_lens = kept_lens, a.first = first;
  a.most = most_kept, a.hkv = heads, a.bs = block_size, a.w = table_width, a.nb = num_blocks, a.row_bytes = row_bytes;
  const int chunks = row_bytes / 16;
  while (a.col_shift < 4 && chunks % (2 << a.col_shift) == 0) ++a.col_shift;
  // narrower slices of rows, down to 128 bytes, while the workgroups leave CUs without one: one user's 4096 tokens of 8 heads of 128, half of them kept, K and V of one
  // layer 21.6 -> 12.7 us, of four 26.5 -> 16.7 (64 bytes 11.7 and 15.7)
  while (a.col_shift > 3 && (int64_t)users * heads * n_caches * (chunks >> a.col_shift) < std::max(device_cus(), 1)) --a.col_shift;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int32_t c0 = 0; c0 < n_caches; c0 += kMostCaches) {
    const int n = std::min(n_caches - c0, kMostCaches);
    for (int i = 0; i < n; ++i) a.caches[i] = static_cast<uint8_t *>(caches_host[c0 + i]);
    a.n_caches = n;
    const unsigned segments = (unsigned)(users * heads), slices = (unsigned)(chunks >> a.col_shift);
    // (wavefronts for every SIMD twice first)
    a.at_once = (int)std::min<int64_t>(kCachesAtOnce, std::max<int64_t>(1, (int64_t)segments * slices * n / (8 * std::max(device_cus(), 1))));
    if (most_kept <= std::min(64, kFewPasses * (64 >> a.col_shift)))
      keep_few_rows_kernel<<<dim3(segments, (unsigned)((n + a.at_once - 1) / a.at_once), slices), dim3(64), 0, st>>>(a);
    else
      keep_rows_kernel<<<dim3(segments, (unsigned)n, slices), dim3(256), 0, st>>>(a);
    if (const int rc = check_launch("keep_cache_tokens")) return rc;
  }
  return TTPA_OK;
}
