// torch.ops.tt.* around the 8-bit cache and the rotation, over the C ABI.
//
// Registered from C++ because most of these calls are a few microseconds of GPU time: through Python views, checks and ctypes a call
// is issued in 15 .. 30 us, from here in 3 .. 5.  Every operator runs on its tensors' device, on that device's current stream; scratch comes from
// the caching allocator on that stream, call by call, so streams, threads and graph captures need no care of their own.  Nothing here has a
// backward pass: a call that autograd would have to watch is refused.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>

#include "ttpa.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kScratchLimit = int64_t(8) << 30;  // as the other operators'

void ok(const char *entry, int rc) { TORCH_CHECK(rc == TTPA_OK, entry, " failed (", rc, "): ", ttpa_last_error()); }
int32_t i32(int64_t v) {
  TORCH_CHECK(v >= std::numeric_limits<int32_t>::min() && v <= std::numeric_limits<int32_t>::max(), "a size of ", v, " does not fit 32 bits");
  return (int32_t)v;
}

// One call: the device of its tensors made current, and its stream.
class Call {
 public:
  Call(const char *name, const Tensor &first) : name_(name), device_(first.device()), guard_(first.device()) {
    see(first, "the first operand");
    stream_ = c10::hip::getCurrentHIPStream(device_.index()).stream();
  }
  void see(const Tensor &t, const char *what) const {
    TORCH_CHECK_NOT_IMPLEMENTED(t.is_cuda(), name_, ": ", what, " is not on a HIP device");
    TORCH_CHECK_VALUE(t.device() == device_, name_, ": ", what, " is on ", t.device(), ", not on ", device_);
    TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t.requires_grad()), name_, " has no backward pass, and ", what,
                                " requires a gradient: call it under torch.no_grad()");
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name_, " has no derivative, and ", what, " carries a tangent");
  }
  void see(const OptTensor &t, const char *what) const {
    if (t) see(*t, what);
  }
  void type(const Tensor &t, at::ScalarType want, const char *what) const {
    see(t, what);
    TORCH_CHECK_VALUE(t.scalar_type() == want, name_, ": ", what, " must be ", want, ", got ", t.scalar_type());
  }
  void *stream() const { return stream_; }
  const char *name() const { return name_; }
  // (straight from the allocator: through the dispatcher an allocation costs as much again, 0.5 of a call's 6.4 us)
  Tensor fresh(at::IntArrayRef sizes, at::ScalarType type = at::kBFloat16) const { return at::detail::empty_cuda(sizes, type, device_, std::nullopt); }
  Tensor scratch(int64_t bytes) const { return fresh({bytes}, at::kByte); }

 private:
  const char *name_;
  c10::Device device_;
  c10::DeviceGuard guard_;
  void *stream_;
};

bool aligned16(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Last dimension contiguous, every other stride (of a dimension of more than one) a multiple of `unit` elements, 16-byte base.
bool has_rows(const Tensor &t, int64_t unit = 8) {
  if (t.dim() == 0 || (t.size(-1) != 1 && t.stride(-1) != 1) || !aligned16(t)) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % unit) return false;
  return true;
}
// (a contiguous tensor at an odd address comes back from contiguous() as it is)
Tensor compact(const Tensor &t) {
  const Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}
Tensor rows(const Tensor &t) { return has_rows(t) ? t : compact(t); }
// A stride for the kernels: of a dimension of one element it is never used, and torch may leave anything there.
int64_t step_of(const Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
Tensor indices(const Call &c, const Tensor &t, const char *what) {
  c.see(t, what);
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), c.name(), ": ", what, " must hold whole numbers");
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong ? t : t.to(at::kLong)).contiguous();
}
int is_i64(const Tensor &t) { return t.scalar_type() == at::kLong; }
// Whole numbers as 32-bit ones; what does not fit stays outside every table and cache.
Tensor narrow(const Tensor &t) {
  if (t.scalar_type() == at::kInt) return t;
  if (t.scalar_type() != at::kLong) return t.to(at::kInt);
  return t.clamp(std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max()).to(at::kInt);
}
Tensor table(const Call &c, const Tensor &t) {
  c.see(t, "page_table");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) > 0, c.name(), ": page_table must be [users, blocks_per_user]");
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), c.name(), ": page_table must hold whole numbers");
  const Tensor p = narrow(t);
  return p.size(1) == 1 || p.stride(1) == 1 ? p : p.contiguous();
}
const int32_t *int_ptr(const Tensor &t) { return static_cast<const int32_t *>(t.data_ptr()); }
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A tensor that is written: no element may stand for several.  (Strides in order, each at least as long as what lies inside it: what is laid out
// in another way without overlapping is refused, too.)
void single(const Call &c, const Tensor &t, const char *what) {
  int64_t end = 1, last = 0;  // elements that the dimensions so far reach over
  for (int64_t n = 0; n < t.dim(); ++n) {
    int64_t stride = std::numeric_limits<int64_t>::max(), size = 1, alike = 0;  // the next longer stride's
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) <= 1 || t.stride(i) <= last) {
        TORCH_CHECK_VALUE(t.size(i) <= 1 || t.stride(i) > 0, c.name(), ": ", what, " is written and must not be expanded");
        continue;
      }
      if (t.stride(i) < stride) stride = t.stride(i), size = t.size(i), alike = 0;
      alike += t.stride(i) == stride;
    }
    if (size == 1) break;
    TORCH_CHECK_VALUE(stride >= end && alike == 1, c.name(), ": ", what, " is written and must not overlap itself");
    end += (size - 1) * stride, last = stride;
  }
}
// Whether two [tokens, heads, head_size] tensors of one shape but for the heads, neither overlapping itself, have an element in common;
// true also where that is not looked into (different token strides, tokens that reach into each other).
bool overlap(const Tensor &x, const Tensor &y) {
  if (!x.is_alias_of(y)) return false;
  const int64_t d = x.size(2), tokens = x.size(0), xs = x.storage_offset(), ys = y.storage_offset();
  const int64_t xh = step_of(x, 1), yh = step_of(y, 1), xt = step_of(x, 0), yt = step_of(y, 0);
  const int64_t xe = xs + (x.size(1) - 1) * xh + (d - 1) * x.stride(2) + 1, ye = ys + (y.size(1) - 1) * yh + (d - 1) * y.stride(2) + 1;
  if (xe + (tokens - 1) * xt <= ys || ye + (tokens - 1) * yt <= xs) return false;
  if (xt != yt || (tokens > 1 && std::max(xe, ye) - std::min(xs, ys) > xt)) return true;
  if (xe <= ys || ye <= xs) return false;
  if (x.stride(2) != 1 || y.stride(2) != 1) return true;
  for (int64_t i = 0; i < x.size(1); ++i)
    for (int64_t j = 0; j < y.size(1); ++j)
      if (std::abs(xs + i * xh - ys - j * yh) < d) return true;
  return false;
}

// The caches of a layer.
struct Cache {
  Tensor k, v, ks, vs;
  int64_t nb, hkv, bs, d;
  Cache(const Call &c, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales)
      : k(k_cache), v(v_cache), ks(k_scales), vs(v_scales) {
    for (const Tensor *t : {&k, &v}) {
      c.type(*t, at::kFloat8_e4m3fn, "a cache");
      TORCH_CHECK_VALUE(t->dim() == 4 && t->is_contiguous() && t->numel() > 0, c.name(),
                        ": a cache must be a contiguous [num_blocks, kv_heads, block_size, head_size] tensor");
    }
    TORCH_CHECK_VALUE(k.sizes() == v.sizes(), c.name(), ": K and V caches must have the same shape");
    nb = k.size(0), hkv = k.size(1), bs = k.size(2), d = k.size(3);
    for (const Tensor *t : {&ks, &vs}) {
      c.type(*t, at::kFloat, "a cache's scales");
      TORCH_CHECK_VALUE(t->dim() == 2 && t->is_contiguous() && t->size(0) == nb && t->size(1) == hkv, c.name(),
                        ": a cache's scales must be a contiguous [num_blocks, kv_heads] tensor");
    }
  }
  // What a writer needs besides: four tensors, not one twice.
  void writable(const Call &c) const {
    const auto apart = [](const Tensor &x, const Tensor &y) {  // (contiguous, of one shape)
      const char *const a = static_cast<const char *>(x.data_ptr()), *const b = static_cast<const char *>(y.data_ptr());
      return std::abs(a - b) >= (int64_t)x.nbytes();
    };
    TORCH_CHECK_VALUE(apart(k, v) && apart(ks, vs), c.name(), ": K and V caches must not share memory");
  }
  float *k_scales() const { return static_cast<float *>(ks.data_ptr()); }
  float *v_scales() const { return static_cast<float *>(vs.data_ptr()); }
  // The bounds of the keys of every block and head, or null.
  void *bounds(const Call &c, const OptTensor &b) const {
    if (!b) return nullptr;
    c.type(*b, at::kBFloat16, "key_bounds");
    TORCH_CHECK_VALUE(b->dim() == 4 && b->is_contiguous() && b->size(0) == nb && b->size(1) == hkv && b->size(2) == 2 && b->size(3) == d, c.name(),
                      ": key_bounds must be a contiguous [num_blocks, kv_heads, 2, head_size] tensor");
    return b->data_ptr();
  }
  void changed(const OptTensor &b) const {
    for (const Tensor *t : {&k, &v, &ks, &vs}) written(*t);
    if (b) written(*b);
  }
};

// ---- norms and rotation -----------------------------------------------------------------------------
struct Rotation {
  Tensor angles, positions, qw, kw;
  int weights_f32 = 0;
  Rotation(const Call &c, const Tensor &query, const Tensor &key, const Tensor &cos_sin, const Tensor &pos, const OptTensor &q_weight,
           const OptTensor &k_weight) {
    c.type(query, at::kBFloat16, "query");
    c.type(key, at::kBFloat16, "key");
    TORCH_CHECK_VALUE(query.dim() == 3 && key.dim() == 3 && query.size(0) == key.size(0) && query.size(2) == key.size(2) && query.size(1) > 0 &&
                          key.size(1) > 0,
                      c.name(), ": query and key must be [tokens, heads, head_size] of the same tokens and head size, got ", query.sizes(), " and ",
                      key.sizes());
    c.see(cos_sin, "cos_sin");
    TORCH_CHECK_VALUE(cos_sin.scalar_type() == at::kFloat || cos_sin.scalar_type() == at::kBFloat16, c.name(), ": cos_sin must be float32 or bfloat16");
    TORCH_CHECK_VALUE(cos_sin.dim() == 2 && cos_sin.size(0) > 0 && cos_sin.size(1) <= query.size(2) && cos_sin.size(1) > 0 && cos_sin.size(1) % 16 == 0,
                      c.name(), ": cos_sin must be [positions, rotary], rotary a multiple of 16 up to the head size");
    angles = rows(cos_sin);
    positions = indices(c, pos, "positions");
    TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == query.size(0), c.name(), ": positions must hold one number per token");
    c.see(q_weight, "q_weight");
    c.see(k_weight, "k_weight");
    bool f32 = false;
    for (const OptTensor *w : {&q_weight, &k_weight})
      if (*w) {
        TORCH_CHECK_VALUE((*w)->scalar_type() == at::kFloat || (*w)->scalar_type() == at::kBFloat16, c.name(), ": weights must be float32 or bfloat16");
        TORCH_CHECK_VALUE((*w)->numel() == query.size(2), c.name(), ": a weight must hold one number per feature of a head");
        f32 = f32 || (*w)->scalar_type() == at::kFloat;
      }
    weights_f32 = f32;
    const auto plain = [&](const OptTensor &w) {
      if (!w) return Tensor();
      if (w->dim() == 1 && has_rows(*w) && (w->scalar_type() == at::kFloat) == f32) return *w;  // (a view would cost as much as the launch)
      Tensor t = (f32 ? w->to(at::kFloat) : *w).reshape({-1}).contiguous();
      return aligned16(t) ? t : t.clone();
    };
    qw = plain(q_weight), kw = plain(k_weight);
  }
  const void *q_weight() const { return qw.defined() ? qw.data_ptr() : nullptr; }
  const void *k_weight() const { return kw.defined() ? kw.data_ptr() : nullptr; }
  int f32() const { return angles.scalar_type() == at::kFloat; }
};

void turn(const Call &c, const Rotation &r, const Tensor &q_out, const Tensor &k_out, const Tensor &q, const Tensor &k, double eps, bool interleaved) {
  ok("ttpa_qk_norm_rope",
     ttpa_qk_norm_rope(q_out.data_ptr(), step_of(q_out, 0), step_of(q_out, 1), k_out.data_ptr(), step_of(k_out, 0), step_of(k_out, 1), q.data_ptr(),
                       step_of(q, 0), step_of(q, 1), k.data_ptr(), step_of(k, 0), step_of(k, 1), r.angles.data_ptr(), r.f32(), step_of(r.angles, 0),
                       r.angles.size(0), r.positions.data_ptr(), is_i64(r.positions), r.q_weight(), r.k_weight(), r.weights_f32, (float)eps,
                       i32(q.size(0)), i32(q.size(1)), i32(k.size(1)), i32(q.size(2)), i32(r.angles.size(1)), interleaved, c.stream()));
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor &query, const Tensor &key, const Tensor &cos_sin, const Tensor &positions,
                                        const OptTensor &q_weight, const OptTensor &k_weight, double eps, bool interleaved) {
  const Call c("tt::qk_norm_rope", query);
  const Rotation r(c, query, key, cos_sin, positions, q_weight, k_weight);
  const Tensor q_out = c.fresh(query.sizes()), k_out = c.fresh(key.sizes());
  if (query.size(0)) turn(c, r, q_out, k_out, rows(query), rows(key), eps, interleaved);
  return {q_out, k_out};
}

void qk_norm_rope_(const Tensor &query, const Tensor &key, const Tensor &cos_sin, const Tensor &positions, const OptTensor &q_weight,
                   const OptTensor &k_weight, double eps, bool interleaved) {
  const Call c("tt::qk_norm_rope_", query);
  const Rotation r(c, query, key, cos_sin, positions, q_weight, k_weight);
  if (query.size(0) == 0) return;
  single(c, query, "query"), single(c, key, "key");
  TORCH_CHECK_VALUE(!overlap(query, key), c.name(), ": query and key must not overlap");
  const Tensor q = rows(query), k = rows(key);
  turn(c, r, q, k, q, k, eps, interleaved);
  if (!q.is_same(query)) query.copy_(q);
  if (!k.is_same(key)) key.copy_(k);
  written(query), written(key);
}

// ---- cache writes -----------------------------------------------------------------------------------
Tensor qk_norm_rope_update_fp8_(const Tensor &query, const Tensor &key, const Tensor &value, const Tensor &cos_sin, const Tensor &positions,
                                const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales,
                                const Tensor &page_table, const OptTensor &q_weight, const OptTensor &k_weight, const OptTensor &key_bounds,
                                double eps, bool interleaved) {
  const Call c("tt::qk_norm_rope_update_fp8_", query);
  const Rotation r(c, query, key, cos_sin, positions, q_weight, k_weight);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  cache.writable(c);
  void *bounds = cache.bounds(c, key_bounds);
  c.type(value, at::kBFloat16, "value");
  const int64_t users = query.size(0), hq = query.size(1);
  TORCH_CHECK_VALUE(value.sizes() == key.sizes() && key.size(1) == cache.hkv && key.size(2) == cache.d, c.name(), ": key ", key.sizes(), " and value ",
                    value.sizes(), " do not match the caches' kv_heads=", cache.hkv, ", head_size=", cache.d);
  const Tensor pt = table(c, page_table);
  TORCH_CHECK_VALUE(pt.size(0) == users, c.name(), ": page_table must have one row per user");
  const Tensor out = c.fresh(query.sizes());
  if (users == 0) return out;
  const Tensor q = rows(query), k = rows(key), v = rows(value);
  ok("ttpa_qk_norm_rope_update_fp8",
     ttpa_qk_norm_rope_update_fp8(out.data_ptr(), step_of(out, 0), step_of(out, 1), q.data_ptr(), step_of(q, 0), step_of(q, 1), k.data_ptr(),
                                  step_of(k, 0), step_of(k, 1), v.data_ptr(), step_of(v, 0), step_of(v, 1), r.angles.data_ptr(), r.f32(),
                                  step_of(r.angles, 0), r.angles.size(0), r.positions.data_ptr(), is_i64(r.positions), r.q_weight(), r.k_weight(),
                                  r.weights_f32, (float)eps, k_cache.data_ptr(), v_cache.data_ptr(), cache.k_scales(), cache.v_scales(), bounds,
                                  int_ptr(pt), step_of(pt, 0), i32(users), i32(hq), i32(cache.hkv), i32(cache.d), i32(r.angles.size(1)), interleaved,
                                  i32(cache.bs), i32(pt.size(1)), i32(cache.nb), c.stream()));
  cache.changed(key_bounds);
  return out;
}

void paged_update_fp8_cache_(const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales, const Tensor &k_fill,
                             const Tensor &v_fill, const Tensor &update_indices, const Tensor &page_table, const OptTensor &key_bounds) {
  const Call c("tt::paged_update_fp8_cache_", k_cache);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  cache.writable(c);
  void *bounds = cache.bounds(c, key_bounds);
  c.type(k_fill, at::kBFloat16, "k_fill");
  c.type(v_fill, at::kBFloat16, "v_fill");
  const Tensor idx = indices(c, update_indices, "update_indices"), pt = table(c, page_table);
  TORCH_CHECK_VALUE(idx.dim() == 1, c.name(), ": update_indices must hold one number per user");
  const int64_t users = idx.size(0);
  for (const Tensor *t : {&k_fill, &v_fill})
    TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == 1 && t->size(1) == users && t->size(2) >= cache.hkv && t->size(3) == cache.d, c.name(), ": fill ",
                      t->sizes(), " does not match users=", users, ", kv_heads=", cache.hkv, ", head_size=", cache.d);
  TORCH_CHECK_VALUE(pt.size(0) >= users, c.name(), ": page_table must be [users, blocks_per_user]");
  if (users == 0) return;
  const Tensor k = rows(k_fill), v = rows(v_fill);
  ok("ttpa_paged_update_fp8_cache",
     ttpa_paged_update_fp8_cache(k_cache.data_ptr(), v_cache.data_ptr(), cache.k_scales(), cache.v_scales(), bounds, k.data_ptr(), step_of(k, 1),
                                 step_of(k, 2), v.data_ptr(), step_of(v, 1), step_of(v, 2), idx.data_ptr(), is_i64(idx), int_ptr(pt), step_of(pt, 0),
                                 i32(users), i32(cache.hkv), i32(cache.bs), i32(cache.d), i32(pt.size(1)), i32(cache.nb), c.stream()));
  cache.changed(key_bounds);
}

void paged_fill_fp8_cache_(const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales, const Tensor &k_fill,
                           const Tensor &v_fill, const Tensor &page_table, const OptTensor &batch_idx, const OptTensor &key_bounds) {
  const Call c("tt::paged_fill_fp8_cache_", k_cache);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  cache.writable(c);
  void *bounds = cache.bounds(c, key_bounds);
  c.type(k_fill, at::kBFloat16, "k_fill");
  c.type(v_fill, at::kBFloat16, "v_fill");
  TORCH_CHECK_VALUE(k_fill.dim() == 4 && k_fill.sizes() == v_fill.sizes() && k_fill.size(1) == cache.hkv && k_fill.size(3) == cache.d, c.name(),
                    ": fills ", k_fill.sizes(), " and ", v_fill.sizes(), " must be [users, kv_heads=", cache.hkv, ", seq_len, head_size=", cache.d, "]");
  const Tensor pt = table(c, page_table);
  const int64_t users = k_fill.size(0), s = k_fill.size(2);
  Tensor bidx;
  if (batch_idx) {
    bidx = indices(c, batch_idx->dim() == 1 ? *batch_idx : batch_idx->reshape({-1}), "batch_idx");
    TORCH_CHECK_VALUE(bidx.size(0) == users, c.name(), ": batch_idx must have one entry per fill row");
  } else {
    TORCH_CHECK_VALUE(users <= 1, c.name(), ": batch_idx is required when the fill holds more than one user");
  }
  TORCH_CHECK_VALUE(s <= pt.size(1) * cache.bs, c.name(), ": ", s, " tokens do not fit ", pt.size(1), " page-table columns of ", cache.bs, " tokens");
  if (users == 0 || s == 0) return;
  const Tensor k = rows(k_fill), v = rows(v_fill);
  ok("ttpa_paged_fill_fp8_cache",
     ttpa_paged_fill_fp8_cache(k_cache.data_ptr(), v_cache.data_ptr(), cache.k_scales(), cache.v_scales(), bounds, k.data_ptr(), step_of(k, 0),
                               step_of(k, 1), step_of(k, 2), v.data_ptr(), step_of(v, 0), step_of(v, 1), step_of(v, 2), int_ptr(pt), step_of(pt, 0),
                               bidx.defined() ? bidx.data_ptr() : nullptr, bidx.defined() && is_i64(bidx), i32(users), i32(pt.size(0)),
                               i32(cache.hkv), i32(s), i32(cache.bs), i32(cache.d), i32(pt.size(1)), i32(cache.nb), c.stream()));
  cache.changed(key_bounds);
}

// ---- attention --------------------------------------------------------------------------------------
// An output handed in by the caller: [.., heads, head_size] bfloat16; what the kernels' stores cannot take is copied to.
Tensor storable(const Tensor &out) { return has_rows(out, 4) ? out : at::empty(out.sizes(), out.options()); }
// Whether `distance` elements lie between two elements of t, whose dimensions `dims` from `at` on are in order, the longest stride first, each stride
// at least as long as what lies inside it.
bool apart_by(const Tensor &t, int64_t distance, const c10::SmallVector<int64_t, 6> &dims, size_t at = 0) {
  if (at == dims.size()) return distance == 0;
  const int64_t stride = t.stride(dims[at]), size = t.size(dims[at]);
  const int64_t below = distance / stride - (distance % stride < 0);
  for (int64_t i = below; i <= below + 1; ++i)
    if (std::abs(i) < size && apart_by(t, distance - i * stride, dims, at + 1)) return true;
  return false;
}
// Whether a call that reads `query` while it writes `out`, of one shape, would find its results there: they have elements in common, and not each its own.
// (out does not overlap itself.  True also where that is not looked into: views of one memory with different strides that reach into each other.)
bool collide(const Tensor &out, const Tensor &query) {
  if (!out.is_alias_of(query) || out.numel() == 0) return false;
  const int64_t distance = query.storage_offset() - out.storage_offset();
  int64_t out_reach = 0, query_reach = 0;
  bool alike = true;
  c10::SmallVector<int64_t, 6> dims;
  for (int64_t i = 0; i < out.dim(); ++i) {
    if (out.size(i) <= 1) continue;
    out_reach += (out.size(i) - 1) * out.stride(i), query_reach += (query.size(i) - 1) * query.stride(i);
    alike = alike && out.stride(i) == query.stride(i);
    dims.push_back(i);
  }
  if (distance > out_reach || -distance > query_reach) return false;
  if (!alike) return true;
  std::sort(dims.begin(), dims.end(), [&](int64_t a, int64_t b) { return out.stride(a) > out.stride(b); });
  return distance != 0 && apart_by(out, distance, dims);
}
void check_out(const Call &c, const Tensor &out, const Tensor &query) {
  c.type(out, at::kBFloat16, "out");
  single(c, out, "out");
  TORCH_CHECK_VALUE(out.sizes() == query.sizes(), c.name(), ": out must have the query's shape ", query.sizes(), ", got ", out.sizes());
  TORCH_CHECK_VALUE(query.scalar_type() != at::kBFloat16 || !collide(out, query), c.name(), ": out and query must be one view or not overlap");
}
void check_query(const Call &c, const Tensor &query, const Cache &cache, const Tensor &pt, const Tensor &cur) {
  c.type(query, at::kBFloat16, "query");
  TORCH_CHECK_VALUE(query.dim() == 4 && query.size(0) == 1, c.name(), ": query must be [1, users, heads, head_size]");
  TORCH_CHECK_VALUE(query.size(3) == cache.d && query.size(2) > 0 && query.size(2) % cache.hkv == 0, c.name(), ": query ", query.sizes(),
                    " does not match the caches' kv_heads=", cache.hkv, ", head_size=", cache.d);
  TORCH_CHECK_VALUE(cur.dim() == 1 && pt.size(0) == query.size(1) && cur.size(0) == query.size(1), c.name(),
                    ": page_table / cur_pos_tensor must have one row per user");
}
float scale_of(const std::optional<double> &scale, int64_t d) { return scale ? (float)*scale : (float)(1.0 / std::sqrt((double)d)); }

void decode_into(const Call &c, const Tensor &out, const Tensor &query, const Cache &cache, const Tensor &page_table, const Tensor &cur_pos,
                 const OptTensor &sink, const std::optional<double> &scale, const std::optional<int64_t> &window) {
  const Tensor pt = table(c, page_table), cur = indices(c, cur_pos, "cur_pos_tensor");
  check_query(c, query, cache, pt, cur);
  TORCH_CHECK_VALUE(!window || *window > 0, c.name(), ": sliding_window_size must be positive");
  const int64_t users = query.size(1), hq = query.size(2);
  Tensor logits;
  if (sink) {
    c.see(*sink, "attention_sink");
    TORCH_CHECK_VALUE(sink->numel() == hq, c.name(), ": attention_sink must hold one logit per query head (", hq, ")");
    logits = sink->scalar_type() == at::kFloat && sink->is_contiguous() ? *sink : sink->to(at::kFloat).contiguous();
  }
  if (users == 0) return;
  const Tensor q = rows(query), target = storable(out);
  const size_t bytes = ttpa_paged_decode_workspace_bytes(i32(users), i32(hq), i32(cache.hkv), i32(cache.d));
  const Tensor ws = c.scratch((int64_t)bytes);
  ok("ttpa_paged_fp8_decode",
     ttpa_paged_fp8_decode(target.data_ptr(), step_of(target, 1), step_of(target, 2), q.data_ptr(), step_of(q, 1), step_of(q, 2), cache.k.data_ptr(),
                           cache.v.data_ptr(), cache.k_scales(), cache.v_scales(), int_ptr(pt), step_of(pt, 0), cur.data_ptr(), is_i64(cur),
                           i32(users), i32(hq), i32(cache.hkv), i32(cache.d), i32(cache.bs), i32(pt.size(1)), i32(cache.nb),
                           scale_of(scale, cache.d), window ? i32(std::min<int64_t>(*window, std::numeric_limits<int32_t>::max())) : 0,
                           logits.defined() ? static_cast<const float *>(logits.data_ptr()) : nullptr, ws.data_ptr(), bytes, c.stream()));
  if (!target.is_same(out)) out.copy_(target);
}

Tensor paged_fp8_attention_decode(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales,
                                  const Tensor &page_table, const Tensor &cur_pos_tensor, const OptTensor &attention_sink,
                                  std::optional<double> scale, std::optional<int64_t> sliding_window_size) {
  const Call c("tt::paged_fp8_attention_decode", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  const Tensor out = c.fresh(query.sizes());
  decode_into(c, out, query, cache, page_table, cur_pos_tensor, attention_sink, scale, sliding_window_size);
  return out;
}

void paged_fp8_attention_decode_out(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales,
                                    const Tensor &v_scales, const Tensor &page_table, const Tensor &cur_pos_tensor, const Tensor &out,
                                    const OptTensor &attention_sink, std::optional<double> scale, std::optional<int64_t> sliding_window_size) {
  const Call c("tt::paged_fp8_attention_decode_out", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  check_out(c, out, query);
  decode_into(c, out, query, cache, page_table, cur_pos_tensor, attention_sink, scale, sliding_window_size);
  written(out);
}

Tensor sparse_into(const Call &c, const Tensor &out, const Tensor &query, const Cache &cache, const Tensor &key_bounds, const Tensor &page_table,
                   const Tensor &cur_pos, int64_t kept, const std::optional<double> &scale) {
  const Tensor pt = table(c, page_table), cur = indices(c, cur_pos, "cur_pos_tensor");
  check_query(c, query, cache, pt, cur);
  void *bounds = cache.bounds(c, key_bounds);
  TORCH_CHECK_VALUE(kept >= 2, c.name(), ": kept_blocks must be at least 2 (the first and the newest block are always kept), got ", kept);
  const int64_t users = query.size(1), hq = query.size(2);
  const Tensor columns = c.fresh({users, cache.hkv, kept}, at::kInt);
  if (users == 0) return columns;
  // (users and heads in one row of heads: a (user, KV head) is a user of the attention)
  const auto packed = [&](const Tensor &t) { return has_rows(t, 8) && (users == 1 || step_of(t, 1) == hq * (hq > 1 ? t.stride(2) : t.stride(1))); };
  const Tensor q = packed(query) ? query : compact(query), target = packed(out) ? out : at::empty(out.sizes(), out.options());
  const auto head_stride = [&](const Tensor &t) { return hq > 1 ? t.stride(2) : users > 1 ? t.stride(1) : cache.d; };
  const size_t bytes = ttpa_paged_fp8_sparse_decode_workspace_bytes(i32(users), i32(hq), i32(cache.hkv), i32(cache.d), i32(pt.size(1)), i32(kept));
  const Tensor ws = c.scratch((int64_t)bytes);
  ok("ttpa_paged_fp8_sparse_decode",
     ttpa_paged_fp8_sparse_decode(target.data_ptr(), head_stride(target), static_cast<int32_t *>(columns.data_ptr()), q.data_ptr(), head_stride(q),
                                  cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scales(), cache.v_scales(), bounds, int_ptr(pt), step_of(pt, 0),
                                  cur.data_ptr(), is_i64(cur), i32(users), i32(hq), i32(cache.hkv), i32(cache.d), i32(cache.bs), i32(pt.size(1)),
                                  i32(cache.nb), i32(kept), scale_of(scale, cache.d), ws.data_ptr(), bytes, c.stream()));
  if (!target.is_same(out)) out.copy_(target);
  return columns;
}

std::tuple<Tensor, Tensor> paged_fp8_sparse_attention_decode(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache,
                                                             const Tensor &k_scales, const Tensor &v_scales, const Tensor &key_bounds,
                                                             const Tensor &page_table, const Tensor &cur_pos_tensor, int64_t kept_blocks,
                                                             std::optional<double> scale) {
  const Call c("tt::paged_fp8_sparse_attention_decode", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  const Tensor out = c.fresh(query.sizes());
  const Tensor columns = sparse_into(c, out, query, cache, key_bounds, page_table, cur_pos_tensor, kept_blocks, scale);
  return {out, columns};
}

Tensor paged_fp8_sparse_attention_decode_out(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales,
                                             const Tensor &v_scales, const Tensor &key_bounds, const Tensor &page_table,
                                             const Tensor &cur_pos_tensor, const Tensor &out, int64_t kept_blocks, std::optional<double> scale) {
  const Call c("tt::paged_fp8_sparse_attention_decode_out", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  check_out(c, out, query);
  const Tensor columns = sparse_into(c, out, query, cache, key_bounds, page_table, cur_pos_tensor, kept_blocks, scale);
  written(out);
  return columns;
}

void chunk_into(const Call &c, const Tensor &out, const Tensor &query, const Cache &cache, const Tensor &page_table, const Tensor &chunk_start,
                const std::optional<double> &scale, int64_t most_keys) {
  c.type(query, at::kBFloat16, "query");
  TORCH_CHECK_VALUE(query.dim() == 4 && query.size(3) == cache.d && query.size(1) > 0 && query.size(1) % cache.hkv == 0, c.name(), ": query ",
                    query.sizes(), " must be [users, heads, chunk_len, head_size] and match the caches' kv_heads=", cache.hkv,
                    ", head_size=", cache.d);
  const Tensor pt = table(c, page_table);
  TORCH_CHECK_VALUE(pt.size(0) == query.size(0), c.name(), ": page_table must have one row per user");
  c.see(chunk_start, "chunk_start_idx_tensor");
  TORCH_CHECK_VALUE(chunk_start.numel() == 1 && at::isIntegralType(chunk_start.scalar_type(), false), c.name(),
                    ": chunk_start_idx_tensor must hold one whole number");
  TORCH_CHECK_VALUE(!scale || *scale > 0, c.name(), ": scale must be positive");
  TORCH_CHECK_VALUE(most_keys >= 0, c.name(), ": most_keys must not be negative");
  const int64_t users = query.size(0), hq = query.size(1), s = query.size(2);
  if (users == 0 || s == 0) return;
  const Tensor start = narrow(chunk_start);
  const Tensor q = rows(query), target = storable(out);
  // as many users at a time as the copies of their blocks have room for
  const auto bytes_of = [&](int64_t n) {
    return ttpa_chunked_fp8_attention_workspace_bytes(i32(n), i32(hq), i32(cache.hkv), i32(s), i32(cache.d), i32(cache.bs), i32(pt.size(1)), most_keys);
  };
  int64_t per = users;
  while (per > 1 && bytes_of(per) > kScratchLimit) per = (per + 1) / 2;
  const int64_t rest = users % per, bytes = std::max(bytes_of(per), rest ? bytes_of(rest) : 0);  // (fewer users may want more parts)
  const Tensor ws = c.scratch(bytes);
  for (int64_t u = 0; u < users; u += per) {
    const int64_t n = std::min(per, users - u);
    ok("ttpa_chunked_fp8_attention",
       ttpa_chunked_fp8_attention(static_cast<uint16_t *>(target.data_ptr()) + u * step_of(target, 0), step_of(target, 0), step_of(target, 1),
                                  step_of(target, 2), static_cast<const uint16_t *>(q.data_ptr()) + u * step_of(q, 0), step_of(q, 0), step_of(q, 1),
                                  step_of(q, 2), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scales(), cache.v_scales(),
                                  int_ptr(pt) + u * step_of(pt, 0), step_of(pt, 0), int_ptr(start), i32(n), i32(hq), i32(cache.hkv), i32(s),
                                  i32(cache.d), i32(cache.bs), i32(pt.size(1)), i32(cache.nb), scale_of(scale, cache.d), most_keys, ws.data_ptr(),
                                  bytes, c.stream()));
  }
  if (!target.is_same(out)) out.copy_(target);
}

Tensor chunked_fp8_attention(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales,
                             const Tensor &page_table, const Tensor &chunk_start_idx_tensor, std::optional<double> scale, int64_t most_keys) {
  const Call c("tt::chunked_fp8_attention", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  const Tensor out = at::empty_like(query);  // keeps the query's (possibly token-major) strides
  chunk_into(c, out, query, cache, page_table, chunk_start_idx_tensor, scale, most_keys);
  return out;
}

void chunked_fp8_attention_out(const Tensor &query, const Tensor &k_cache, const Tensor &v_cache, const Tensor &k_scales, const Tensor &v_scales,
                               const Tensor &page_table, const Tensor &chunk_start_idx_tensor, const Tensor &out, std::optional<double> scale,
                               int64_t most_keys) {
  const Call c("tt::chunked_fp8_attention_out", query);
  const Cache cache(c, k_cache, v_cache, k_scales, v_scales);
  check_out(c, out, query);
  chunk_into(c, out, query, cache, page_table, chunk_start_idx_tensor, scale, most_keys);
  written(out);
}

#define TT_ROPE "Tensor cos_sin, Tensor positions"
#define TT_CACHE "Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales"
#define TT_CACHE_W "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales"

TORCH_LIBRARY_FRAGMENT(tt, m) {
  m.def("qk_norm_rope(Tensor query, Tensor key, " TT_ROPE ", Tensor? q_weight=None, Tensor? k_weight=None, float eps=1e-06, "
        "bool interleaved=False) -> (Tensor, Tensor)");
  m.def("qk_norm_rope_(Tensor(a!) query, Tensor(b!) key, " TT_ROPE ", Tensor? q_weight=None, Tensor? k_weight=None, float eps=1e-06, "
        "bool interleaved=False) -> ()");
  m.def("qk_norm_rope_update_fp8_(Tensor query, Tensor key, Tensor value, " TT_ROPE ", " TT_CACHE_W ", Tensor page_table, "
        "Tensor? q_weight=None, Tensor? k_weight=None, Tensor(e!)? key_bounds=None, float eps=1e-06, bool interleaved=False) -> Tensor");
  m.def("paged_update_fp8_cache_(" TT_CACHE_W ", Tensor k_fill, Tensor v_fill, Tensor update_indices, Tensor page_table, "
        "Tensor(e!)? key_bounds=None) -> ()");
  m.def("paged_fill_fp8_cache_(" TT_CACHE_W ", Tensor k_fill, Tensor v_fill, Tensor page_table, Tensor? batch_idx=None, "
        "Tensor(e!)? key_bounds=None) -> ()");
  m.def("paged_fp8_attention_decode(Tensor query, " TT_CACHE ", Tensor page_table, Tensor cur_pos_tensor, Tensor? attention_sink=None, "
        "float? scale=None, int? sliding_window_size=None) -> Tensor");
  m.def("paged_fp8_attention_decode_out(Tensor query, " TT_CACHE ", Tensor page_table, Tensor cur_pos_tensor, Tensor(a!) out, "
        "Tensor? attention_sink=None, float? scale=None, int? sliding_window_size=None) -> ()");
  m.def("paged_fp8_sparse_attention_decode(Tensor query, " TT_CACHE ", Tensor key_bounds, Tensor page_table, Tensor cur_pos_tensor, "
        "int kept_blocks, float? scale=None) -> (Tensor, Tensor)");
  m.def("paged_fp8_sparse_attention_decode_out(Tensor query, " TT_CACHE ", Tensor key_bounds, Tensor page_table, Tensor cur_pos_tensor, "
        "Tensor(a!) out, int kept_blocks, float? scale=None) -> Tensor");
  m.def("chunked_fp8_attention(Tensor query, " TT_CACHE ", Tensor page_table, Tensor chunk_start_idx_tensor, float? scale=None, "
        "int most_keys=0) -> Tensor");
  m.def("chunked_fp8_attention_out(Tensor query, " TT_CACHE ", Tensor page_table, Tensor chunk_start_idx_tensor, Tensor(a!) out, "
        "float? scale=None, int most_keys=0) -> ()");
}

TORCH_LIBRARY_IMPL(tt, CUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_", &qk_norm_rope_);
  m.impl("qk_norm_rope_update_fp8_", &qk_norm_rope_update_fp8_);
  m.impl("paged_update_fp8_cache_", &paged_update_fp8_cache_);
  m.impl("paged_fill_fp8_cache_", &paged_fill_fp8_cache_);
  m.impl("paged_fp8_attention_decode", &paged_fp8_attention_decode);
  m.impl("paged_fp8_attention_decode_out", &paged_fp8_attention_decode_out);
  m.impl("paged_fp8_sparse_attention_decode", &paged_fp8_sparse_attention_decode);
  m.impl("paged_fp8_sparse_attention_decode_out", &paged_fp8_sparse_attention_decode_out);
  m.impl("chunked_fp8_attention", &chunked_fp8_attention);
  m.impl("chunked_fp8_attention_out", &chunked_fp8_attention_out);
}

}  // namespace
