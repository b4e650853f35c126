// _flash_attn_host: the torch side of the cache and norm + rotary operators (argument checks, allocations, strides,
// autograd) in C++, for flash_attn/kvcache_interface.py and flash_attn/layers/qk_norm.py.
//
// A decoding step launches kernels of 5 to 15 us; the same checks and calls through Python and ctypes took
// 15 to 30 us a call, and a forward with its backward 180 us, which the GPU spent waiting.  Here they take
// 6 to 12 us (50 to 90 us by machine, of which a product of two tensors and its gradient takes half).  The
// kernels stay behind the C ABI of libflash_attn_mi355x.so: bind() is handed the addresses of its entry points
// by flash_attn_2_cuda, which loads it, so that one library serves both.
#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <optional>
#include <string>
#include <unordered_map>

#include "../../include/flash_attn.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Library {
  decltype(&flash_attn_qk_norm_rotary) norm = nullptr;
  decltype(&flash_attn_qk_norm_rotary_bwd) norm_bwd = nullptr;
  decltype(&flash_attn_qk_norm_rotary_workspace) norm_workspace = nullptr;
  decltype(&flash_attn_kvcache) kvcache = nullptr;
  decltype(&flash_attn_kvcache_workspace) kvcache_workspace = nullptr;
  decltype(&flash_attn_kvcache_evict) evict = nullptr;
  decltype(&flash_attn_kvcache_commit) commit = nullptr;
  decltype(&flash_attn_error) error = nullptr;
} lib;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
#define BIND(field, name) lib.field = reinterpret_cast<decltype(lib.field)>(at.at(#name))
  BIND(norm, flash_attn_qk_norm_rotary);
  BIND(norm_bwd, flash_attn_qk_norm_rotary_bwd);
  BIND(norm_workspace, flash_attn_qk_norm_rotary_workspace);
  BIND(kvcache, flash_attn_kvcache);
  BIND(kvcache_workspace, flash_attn_kvcache_workspace);
  BIND(evict, flash_attn_kvcache_evict);
  BIND(commit, flash_attn_kvcache_commit);
  BIND(error, flash_attn_error);
#undef BIND
}

void check_call(bool ok, const char* op) {
  if (ok) return;
  const char* e = lib.error();
  TORCH_CHECK(false, op, ": ", e ? e : "unknown error");
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* mut(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// {batch, row, head} element strides of (b, s, h, d)
struct Strides {
  int64_t v[3] = {0, 0, 0};
  Strides() = default;
  explicit Strides(const Tensor& t) {
    for (int i = 0; i < 3; ++i) v[i] = t.stride(i);
  }
};

// 16-byte vector access: base and strides
bool aligned(const Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 != 0) return false;
  return true;
}
// a kernel writes into t: what autograd saved of it before must not be taken for what it holds now
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor vec_ok(const Tensor& t) { return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
// Whether two views of one storage share an element: their offsets differ by sum x_i stride_i for some x_i in
// [1 - size_i of b, size_i of a - 1].  Looked for from the largest stride down, where what the smaller ones reach
// leaves one or two x_i to try.  Views of unlike strides stay undecided (false).
bool share_elements(const Tensor& a, const Tensor& b) {
  if (!a.storage().is_alias_of(b.storage()) || a.numel() == 0 || b.numel() == 0) return false;
  if (a.dim() != b.dim() || a.scalar_type() != b.scalar_type()) return false;
  struct Dim { int64_t stride, lo, hi; };
  Dim dims[8];
  int n = 0;
  for (int64_t i = 0; i < a.dim(); ++i) {
    if (a.size(i) == 1 && b.size(i) == 1) continue;
    if (n == 8 || (a.size(i) > 1 && b.size(i) > 1 && a.stride(i) != b.stride(i))) return false;
    dims[n++] = {a.size(i) > 1 ? a.stride(i) : b.stride(i), 1 - b.size(i), a.size(i) - 1};
  }
  std::sort(dims, dims + n, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  int64_t low[9] = {}, high[9] = {};   // what dims i .. reach
  for (int i = n; i-- > 0;) {
    low[i] = low[i + 1] + dims[i].stride * dims[i].lo;
    high[i] = high[i + 1] + dims[i].stride * dims[i].hi;
  }
  int tries = 256;                     // (strides that do not nest could ask for more)
  const std::function<bool(int, int64_t)> reach = [&](int i, int64_t rest) {
    if (rest < low[i] || rest > high[i] || --tries < 0) return false;
    if (i == n) return rest == 0;
    if (dims[i].stride == 0) return reach(i + 1, rest);
    const int64_t mid = rest / dims[i].stride;
    for (int64_t x = std::max(dims[i].lo, mid - 1); x <= std::min(dims[i].hi, mid + 1); ++x)
      if (reach(i + 1, rest - x * dims[i].stride)) return true;
    return false;
  };
  return reach(0, b.storage_offset() - a.storage_offset());
}

// t is written: an expanded tensor, or two that share elements, would be by several rows at once
void check_writable(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* a : ts) {
    if (a == nullptr) continue;
    TORCH_CHECK(at::has_internal_overlap(*a) != at::MemOverlap::Yes, op, ": written tensors must not be expanded");
    for (const Tensor* b : ts) {
      if (b == a) break;
      if (b == nullptr) continue;
      const auto overlap = at::get_overlap_status(*a, *b);
      TORCH_CHECK(a->unsafeGetTensorImpl() != b->unsafeGetTensorImpl() && overlap != at::MemOverlapStatus::Full &&
                      overlap != at::MemOverlapStatus::Partial && !share_elements(*a, *b),
                  op, ": written tensors must not share memory");
    }
  }
}

// the last of the checks: everything on one GPU (its architecture is checked behind the C ABI)
void check_device(const char* op, std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (t == nullptr) continue;
    TORCH_CHECK(t->is_cuda(), op, ": tensors must be on the GPU");
    if (first == nullptr) first = t;
    TORCH_CHECK(t->device() == first->device(), op, ": tensors must share a device");
  }
}
const Tensor* opt(const OptTensor& t) { return t ? &*t : nullptr; }

// A dual tensor's tangent would be lost without a word: its requires_grad is false.
void check_no_tangent(const char* op, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK(t == nullptr || !t->_fw_grad(/*level=*/0).defined(), op, ": no forward-mode derivative");
}

void check_no_grad(std::initializer_list<const Tensor*> ts) {
  check_no_tangent("kvcache", ts);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK(t == nullptr || !t->requires_grad(), "kvcache: the cache has no backward; call it under torch.no_grad()");
}

// ------------------------------------------------------------------------------------------------
// key/value cache
// ------------------------------------------------------------------------------------------------
constexpr int64_t kMaxSlots = 0x7fff0000;   // (the C ABI's limit: the kernels' int counters run past the last slot)
struct Cache {
  int64_t b, slots, page = 0, pages = 0, hk, d, table_stride = 0;
  Strides strides;
  Cache(const Tensor& k, const Tensor& v, const Tensor& lens, const OptTensor& table) {
    TORCH_CHECK(half_type(k.scalar_type()), "kvcache: only fp16 and bf16 are supported");
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), "kvcache: k_cache and v_cache must have the same dtype");
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(),
                "kvcache: k_cache and v_cache must both be (batch or pages, slots, nheads_k, headdim)");
    TORCH_CHECK(k.numel() > 0, "kvcache: the cache is empty");
    TORCH_CHECK(v.strides() == k.strides(), "kvcache: k_cache and v_cache must have the same strides");
    hk = k.size(2);
    d = k.size(3);
    TORCH_CHECK(d % 8 == 0 && d <= 256, "kvcache: headdim must be a multiple of 8, at most 256");
    TORCH_CHECK(k.stride(3) == 1, "kvcache: the cache must have a contiguous last dimension");
    TORCH_CHECK(aligned(k) && aligned(v), "kvcache: the cache must be 16-byte aligned in its base and strides");
    TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.is_contiguous(),
                "kvcache: cache_seqlens must be a contiguous int32 vector");
    b = lens.size(0);
    TORCH_CHECK(b > 0 && b < (1 << 30), "kvcache: batch size must be positive");
    strides = Strides(k);
    if (!table) {
      TORCH_CHECK(k.size(0) == b, "kvcache: the cache and cache_seqlens must have the same batch size");
      slots = k.size(1);
    } else {
      TORCH_CHECK(table->scalar_type() == at::kInt && table->dim() == 2 && table->size(0) == b,
                  "kvcache: block_table must be int32 (batch, blocks)");
      TORCH_CHECK(table->size(1) > 0 && table->stride(1) == 1,
                  "kvcache: block_table must have a contiguous last dimension");
      page = k.size(1);
      pages = k.size(0);
      slots = table->size(1) * page;
      table_stride = table->stride(0);
    }
    TORCH_CHECK(slots <= kMaxSlots && page <= kMaxSlots && pages <= kMaxSlots && hk < (1 << 24),
                "kvcache: too many slots");
  }
  // weights of fewer columns than there are slots limit the room of a sequence
  void limit(const Tensor& w) {
    TORCH_CHECK(w.scalar_type() == at::kFloat && w.dim() == 3 && w.size(0) == b && w.size(1) == hk && w.size(2) > 0,
                "kvcache: attn_weight must be fp32 (batch, nheads_k, slots)");
    TORCH_CHECK(w.stride(2) == 1, "kvcache: attn_weight must have a contiguous last dimension");
    slots = std::min(slots, w.size(2));
  }
};

Tensor flag_bytes(const Tensor& m, const char* name) {
  TORCH_CHECK(m.scalar_type() == at::kBool, "kvcache: ", name, " must be bool");
  return m.stride(-1) == 1 ? m : m.contiguous();
}

std::pair<Tensor, Tensor> kvcache(const Tensor& q_in, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lens,
                                  const OptTensor& k_in, const OptTensor& v_in, const OptTensor& table,
                                  const OptTensor& mask_in, std::optional<double> softmax_scale,
                                  const OptTensor& weight) {
  Cache c(k_cache, v_cache, lens, table);
  TORCH_CHECK(q_in.scalar_type() == k_cache.scalar_type(), "kvcache: q and the cache must have the same dtype");
  TORCH_CHECK(q_in.dim() == 4 && q_in.size(0) == c.b && q_in.size(3) == c.d,
              "kvcache: q must have shape (batch, seqlen_q, nheads, headdim)");
  const int64_t sq = q_in.size(1), h = q_in.size(2);
  if (weight) c.limit(*weight);
  TORCH_CHECK(sq > 0, "kvcache: at least one drafted token");
  TORCH_CHECK(h > 0 && h % c.hk == 0, "Number of heads in key/value must divide number of heads in query");
  TORCH_CHECK(sq <= c.slots, "kvcache: more drafted tokens than slots");
  TORCH_CHECK(k_in.has_value() == v_in.has_value(), "kvcache: k and v come together");
  TORCH_CHECK(q_in.stride(3) == 1, "kvcache: q must have a contiguous last dimension");
  if (k_in)
    for (const Tensor* t : {&*k_in, &*v_in}) {
      TORCH_CHECK(t->scalar_type() == q_in.scalar_type(), "kvcache: k and v must have the cache's dtype");
      TORCH_CHECK(t->dim() == 4 && t->size(0) == c.b && t->size(1) == sq && t->size(2) == c.hk && t->size(3) == c.d,
                  "kvcache: k and v must have shape (batch, seqlen_q, nheads_k, headdim)");
      TORCH_CHECK(t->stride(3) == 1, "kvcache: k and v must have a contiguous last dimension");
    }
  check_no_grad({&q_in, opt(k_in), opt(v_in), &k_cache, &v_cache, opt(weight)});
  if (k_in) check_writable("kvcache", {&k_cache, &v_cache, opt(weight)});
  else check_writable("kvcache", {opt(weight)});
  OptTensor mask;
  int64_t mask_strides[2] = {0, 0};
  if (mask_in) {
    const int64_t n = mask_in->dim();
    TORCH_CHECK((n == 2 || (n == 3 && mask_in->size(0) == c.b)) && mask_in->size(-1) == sq && mask_in->size(-2) == sq,
                "kvcache: tree_mask must be bool (seqlen_q, seqlen_q) or (batch, seqlen_q, seqlen_q)");
    mask = flag_bytes(*mask_in, "tree_mask");
    if (n == 3) mask_strides[0] = mask->stride(0);
    mask_strides[1] = mask->stride(-2);
  }
  const double scale = softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)c.d);
  TORCH_CHECK(scale > 0.0 && (float)scale > 0.f && std::isfinite((float)scale),
              "kvcache: softmax_scale must be positive and finite");
  check_device("kvcache", {&k_cache, &v_cache, &lens, opt(table), &q_in, opt(k_in), opt(v_in), opt(mask), opt(weight)});
  const c10::DeviceGuard guard(q_in.device());
  const Tensor q = vec_ok(q_in);
  OptTensor k, v;
  Strides ks, vs;
  if (k_in) {
    k = vec_ok(*k_in);
    v = vec_ok(*v_in);
    ks = Strides(*k);
    vs = Strides(*v);
  }
  Tensor out = at::empty({c.b, sq, h, c.d}, q.options());
  Tensor lse = at::empty({c.b, h, sq}, q.options().dtype(at::kFloat));
  const size_t bytes = lib.kvcache_workspace((int)c.b, (int)sq, (int)c.slots, (int)h, (int)c.hk, (int)c.d,
                                             weight.has_value());
  Tensor work;
  if (bytes) work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  int64_t ws[2] = {0, 0};
  if (weight) { ws[0] = weight->stride(0); ws[1] = weight->stride(1); }
  check_call(lib.kvcache(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ptr(k), ptr(v), out.data_ptr(),
                         lse.data_ptr<float>(), static_cast<float*>(mut(weight)), lens.data_ptr<int32_t>(),
                         static_cast<const int32_t*>(ptr(table)), static_cast<const uint8_t*>(ptr(mask)),
                         bytes ? work.data_ptr() : nullptr, (int)c.b, (int)sq, (int)c.slots, (int)h, (int)c.hk, (int)c.d,
                         (int)c.page, (int)c.pages, (float)scale, Strides(q).v, c.strides.v, ks.v, vs.v, Strides(out).v,
                         c.table_stride, mask_strides, ws, q.scalar_type() == at::kBFloat16, stream_of(q)),
             "flash_attn_kvcache");
  if (k) { written(k_cache); written(v_cache); }
  if (weight) written(*weight);
  return {out, lse};
}

Tensor commit(const Tensor& k_cache, const Tensor& v_cache, const Tensor& lens, const Tensor& accepted_in,
              const OptTensor& table, const OptTensor& weight) {
  Cache c(k_cache, v_cache, lens, table);
  TORCH_CHECK(accepted_in.dim() == 2 && accepted_in.size(0) == c.b, "kvcache: accepted must be bool (batch, seqlen_q)");
  const int64_t sq = accepted_in.size(1);
  if (weight) c.limit(*weight);
  TORCH_CHECK(0 < sq && sq <= 8192 && sq <= c.slots, "kvcache: between 1 and min(8192, slots) drafted tokens");
  const Tensor accepted = flag_bytes(accepted_in, "accepted");
  check_no_grad({&k_cache, &v_cache, opt(weight)});
  check_writable("kvcache", {&k_cache, &v_cache, opt(weight)});
  check_device("kvcache", {&k_cache, &v_cache, &lens, opt(table), &accepted, opt(weight)});
  const c10::DeviceGuard guard(k_cache.device());
  Tensor out = at::empty_like(lens);
  int64_t ws[2] = {0, 0};
  if (weight) { ws[0] = weight->stride(0); ws[1] = weight->stride(1); }
  check_call(lib.commit(k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr<int32_t>(),
                        static_cast<const uint8_t*>(accepted.data_ptr()), static_cast<const int32_t*>(ptr(table)),
                        out.data_ptr<int32_t>(), static_cast<float*>(mut(weight)), (int)c.b, (int)sq, (int)c.slots,
                        (int)c.hk, (int)c.d, (int)c.page, (int)c.pages, c.strides.v, c.table_stride, accepted.stride(0), ws,
                        stream_of(k_cache)),
             "flash_attn_kvcache_commit");
  written(k_cache);
  written(v_cache);
  if (weight) written(*weight);
  return out;
}

std::tuple<Tensor, Tensor, Tensor> evict(const Tensor& k_cache, const Tensor& v_cache, const Tensor& lens,
                                         const Tensor& weight, int64_t budget, int64_t sink, int64_t recent,
                                         const OptTensor& table) {
  Cache c(k_cache, v_cache, lens, table);
  TORCH_CHECK(budget > 0 && budget <= kMaxSlots && sink >= 0 && recent >= 0 && sink <= budget && recent <= budget - sink,
              "kvcache: budget must be positive, at least sink + recent and at most 2^31 - 2^16");
  TORCH_CHECK(c.b <= 65535, "kvcache: batch size must be at most 65535");
  c.limit(weight);
  check_no_grad({&k_cache, &v_cache, &weight});
  check_writable("kvcache", {&k_cache, &v_cache});
  check_device("kvcache", {&k_cache, &v_cache, &lens, opt(table), &weight});
  const c10::DeviceGuard guard(k_cache.device());
  Tensor out = at::empty_like(lens);
  Tensor weight_out = at::empty({c.b, c.hk, weight.size(2)}, weight.options());
  if (weight.size(2) > c.slots) {   // columns that no slot belongs to: 0 behind a sequence's keys as well
    const Tensor held = lens.ge(0).logical_and_(lens.le(c.slots)).unsqueeze(1).unsqueeze(2);
    weight_out.slice(2, c.slots).copy_(weight.slice(2, c.slots).masked_fill(held, 0.0));
  }
  Tensor kept = at::empty({c.b, c.hk, budget}, lens.options());
  Tensor work = at::empty({c.b * c.hk}, lens.options());
  const int64_t ws[2] = {weight.stride(0), weight.stride(1)}, wo[2] = {weight_out.stride(0), weight_out.stride(1)};
  check_call(lib.evict(k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr<int32_t>(), weight.data_ptr<float>(),
                       static_cast<const int32_t*>(ptr(table)), out.data_ptr<int32_t>(), weight_out.data_ptr<float>(),
                       kept.data_ptr<int32_t>(), work.data_ptr(), (int)c.b, (int)c.slots, (int)c.hk, (int)c.d, (int)c.page,
                       (int)c.pages, (int)budget, (int)sink, (int)recent, c.strides.v, c.table_stride, ws, wo,
                       stream_of(k_cache)),
             "flash_attn_kvcache_evict");
  written(k_cache);
  written(v_cache);
  return {out, weight_out, kept};
}

// ------------------------------------------------------------------------------------------------
// norm + rotary
// ------------------------------------------------------------------------------------------------
Tensor rows(const Tensor& t) { return t.dim() == 4 ? t : t.unsqueeze(0); }

// what both directions hand over, in the form the C ABI takes
struct NormArgs {
  Tensor q, k;                       // (b, s, h, d)
  OptTensor wq, wk, cos, sin, pos;
  int b, s, h, hk, d, rd = 0, table_rows = 0;
  int64_t pos_stride = 0, cos_stride = 0;
  bool weight_f32, table_f32, bf16;
  NormArgs(const Tensor& q_, const Tensor& k_, const OptTensor& wq_, const OptTensor& wk_, const OptTensor& cos_,
           const OptTensor& sin_, const OptTensor& pos_)
      : q(rows(q_)), k(rows(k_)), cos(cos_), sin(sin_) {
    if (wq_) wq = wq_->contiguous();
    if (wk_) wk = wk_->contiguous();
    if (cos && (cos->stride(1) != 1 || sin->strides() != cos->strides())) {
      cos = cos->contiguous();
      sin = sin->contiguous();
    }
    b = (int)q.size(0); s = (int)q.size(1); h = (int)q.size(2); hk = (int)k.size(2); d = (int)q.size(3);
    if (pos_) {
      pos = pos_->dim() == 2 ? *pos_ : pos_->unsqueeze(0);
      if (pos->stride(1) != 1) pos = pos->contiguous();
      pos_stride = pos->stride(0);
    }
    if (cos) { rd = 2 * (int)cos->size(1); table_rows = (int)cos->size(0); cos_stride = cos->stride(0); }
    const OptTensor& w = wq ? wq : wk;
    weight_f32 = w && w->scalar_type() == at::kFloat;
    table_f32 = cos && cos->scalar_type() == at::kFloat;
    bf16 = q.scalar_type() == at::kBFloat16;
  }
};

void check_norm(const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk, const OptTensor& cos,
                const OptTensor& sin, const OptTensor& pos, double eps) {
#define CHECK(cond, ...) TORCH_CHECK(cond, "qk_norm_rotary: ", __VA_ARGS__)
  CHECK(eps >= 0.0, "eps must not be negative");
  CHECK(half_type(q.scalar_type()), "only fp16 and bf16 are supported");
  CHECK(k.scalar_type() == q.scalar_type(), "q and k must have the same dtype");
  CHECK((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim(),
        "q and k must be (batch, seqlen, nheads, headdim) or (total, nheads, headdim)");
  bool agree = q.size(-1) == k.size(-1) && q.size(-3) == k.size(-3);
  if (q.dim() == 4) agree = agree && q.size(0) == k.size(0);
  CHECK(agree, "q and k must agree in batch, seqlen and headdim");
  CHECK(q.size(-2) > 0 && k.size(-2) > 0, "q and k need a head each");
  const int64_t d = q.size(-1);
  CHECK(0 < d && d <= 256, "headdim must be at most 256");
  CHECK(q.stride(-1) == 1 && k.stride(-1) == 1, "last dim must be contiguous");
  CHECK(q.numel() / d < ((int64_t)1 << 31) && k.numel() / d < ((int64_t)1 << 31), "too many rows");
  for (const OptTensor* w : {&wq, &wk})
    if (*w) {
      CHECK((*w)->dim() == 1 && (*w)->size(0) == d, "weights must have shape (headdim,)");
      CHECK((*w)->scalar_type() == q.scalar_type() || (*w)->scalar_type() == at::kFloat,
            "weights must be fp32 or of q's dtype");
    }
  CHECK(!wq || !wk || wq->scalar_type() == wk->scalar_type(), "weights must share a dtype");
  CHECK(cos.has_value() == sin.has_value(), "cos and sin come together");
  if (!cos) {
    CHECK(!pos, "positions without cos and sin");
  } else {
    CHECK(cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->scalar_type() == sin->scalar_type(), "bad cos/sin shape");
    CHECK(cos->scalar_type() == q.scalar_type() || cos->scalar_type() == at::kFloat,
          "cos and sin must be fp32 or of q's dtype");
    CHECK(0 < cos->size(1) && 2 * cos->size(1) <= d && cos->size(0) > 0 && cos->size(0) < 0x7fffffff, "bad cos/sin shape");
    if (!pos) {
      CHECK(cos->size(0) >= q.size(-3), "cos/sin have fewer rows than the sequence");
    } else {
      CHECK(pos->scalar_type() == at::kInt, "positions must have dtype int32");
      CHECK(pos->sizes() == q.sizes().slice(0, q.dim() - 2), "positions must have the shape of q's tokens");
    }
  }
#undef CHECK
  check_device("qk_norm_rotary", {&q, &k, opt(wq), opt(wk), opt(cos), opt(sin), opt(pos)});
}

void norm_forward(const NormArgs& a, const Tensor& q_out, const Tensor& k_out, bool interleaved, double eps) {
  if (a.q.numel() == 0) return;
  const c10::DeviceGuard guard(a.q.device());
  check_call(lib.norm(a.q.data_ptr(), a.k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), ptr(a.wq), ptr(a.wk), ptr(a.cos),
                      ptr(a.sin), static_cast<const int32_t*>(ptr(a.pos)), a.b, a.s, a.h, a.hk, a.d, a.rd, a.table_rows,
                      (float)eps, Strides(a.q).v, Strides(a.k).v, Strides(rows(q_out)).v, Strides(rows(k_out)).v,
                      a.pos_stride, a.cos_stride, a.weight_f32, a.table_f32, interleaved, a.bf16, stream_of(a.q)),
             "flash_attn_qk_norm_rotary");
}

Tensor value(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct QkNormRotary : torch::autograd::Function<QkNormRotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const OptTensor& wq, const OptTensor& wk, const OptTensor& cos,
                                                const OptTensor& sin, const OptTensor& pos, bool interleaved, double eps) {
    const c10::DeviceGuard guard(q.device());
    Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
    norm_forward(NormArgs(q, k, wq, wk, cos, sin, pos), q_out, k_out, interleaved, eps);
    ctx->save_for_backward({q, k, value(wq), value(wk), value(cos), value(sin), value(pos)});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    return {q_out, k_out};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list out;
    {
      const at::AutoGradMode no_grad(false);
      out = gradients(ctx, saved, grads);
    }
    if (at::GradMode::is_enabled()) {   // create_graph: differentiating these again raises
      torch::autograd::variable_list defined;
      for (Tensor& t : out)
        if (t.defined()) defined.push_back(t.detach().set_requires_grad(true));
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "qk_norm_rotary is differentiable once", (int64_t)defined.size());
      defined = (*error)(std::move(defined));
      size_t i = 0;
      for (Tensor& t : out)
        if (t.defined()) t = defined[i++];
    }
    return out;
  }

  static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx,
                                                  const torch::autograd::variable_list& saved,
                                                  const torch::autograd::variable_list& grads) {
    const Tensor &q = saved[0], &k = saved[1];
    const NormArgs a(q, k, maybe(saved[2]), maybe(saved[3]), maybe(saved[4]), maybe(saved[5]), maybe(saved[6]));
    const c10::DeviceGuard guard(q.device());
    // (a sum's gradient is an expanded scalar, for instance)
    const Tensor gq = rows(grads[0].stride(-1) == 1 ? grads[0] : grads[0].contiguous());
    const Tensor gk = rows(grads[1].stride(-1) == 1 ? grads[1] : grads[1].contiguous());
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dwq, dwk, work;
    const bool any = q.numel() > 0;
    // (the edges of a node are those of the tensors that there are)
    if (a.wq && ctx->needs_input_grad(2)) dwq = any ? at::empty_like(*a.wq) : at::zeros_like(*a.wq);
    if (a.wk && ctx->needs_input_grad(a.wq ? 3 : 2)) dwk = any ? at::empty_like(*a.wk) : at::zeros_like(*a.wk);
    if (any) {
      if (dwq.defined() || dwk.defined())
        work = at::empty({(int64_t)lib.norm_workspace(a.d)}, q.options().dtype(at::kByte));
      check_call(lib.norm_bwd(gq.data_ptr(), gk.data_ptr(), a.q.data_ptr(), a.k.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                              ptr(a.wq), ptr(a.wk), dwq.defined() ? dwq.data_ptr() : nullptr,
                              dwk.defined() ? dwk.data_ptr() : nullptr, ptr(a.cos), ptr(a.sin),
                              static_cast<const int32_t*>(ptr(a.pos)), work.defined() ? work.data_ptr() : nullptr, a.b, a.s,
                              a.h, a.hk, a.d, a.rd, a.table_rows, (float)ctx->saved_data["eps"].toDouble(), Strides(gq).v,
                              Strides(gk).v, Strides(a.q).v, Strides(a.k).v, Strides(rows(dq)).v, Strides(rows(dk)).v,
                              a.pos_stride, a.cos_stride, a.weight_f32, a.table_f32,
                              ctx->saved_data["interleaved"].toBool(), a.bf16, stream_of(q)),
                 "flash_attn_qk_norm_rotary_bwd");
    }
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// A gradient accumulator that an eager graph keeps alive belongs to that graph's stream, and a backward that is
// being captured makes this stream part of the capture.  A side stream joins and is let go at the end; the default
// stream cannot be captured: torch cannot end such a capture, and the process ends.
void check_capture(std::initializer_list<const Tensor*> ts) {
  const auto device = (*ts.begin())->device().index();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device).stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone)
    return;
  const auto eager = c10::hip::getDefaultHIPStream(device).id();
  for (const Tensor* t : ts) {
    if (t == nullptr || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto of = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!of || of->id() != eager,
                "qk_norm_rotary: captured while an eager graph of the same leaves, on the default stream, is alive; let go of "
                "its outputs first, or make it (and a wrapper that holds their accumulators) on a side stream");
  }
}

std::pair<Tensor, Tensor> norm_rotary(const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk,
                                      const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, bool interleaved,
                                      double eps, bool inplace) {
  check_no_tangent("qk_norm_rotary", {&q, &k, opt(wq), opt(wk), opt(cos), opt(sin)});
  if (inplace) check_writable("qk_norm_rotary", {&q, &k});
  check_norm(q, k, wq, wk, cos, sin, pos, eps);
  bool grad = false;
  if (at::GradMode::is_enabled())
    for (const Tensor* t : {&q, &k, opt(wq), opt(wk)}) grad = grad || (t != nullptr && t->requires_grad());
  if (inplace) {
    TORCH_CHECK(!grad, "qk_norm_rotary: inplace=True is for inference; the backward needs the inputs");
    norm_forward(NormArgs(q, k, wq, wk, cos, sin, pos), q, k, interleaved, eps);
    written(q);
    written(k);
    return {q, k};
  }
  if (!grad) {   // (a decoding step waits for the host: none of autograd's part then)
    const c10::DeviceGuard guard(q.device());
    Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
    norm_forward(NormArgs(q, k, wq, wk, cos, sin, pos), q_out, k_out, interleaved, eps);
    return {q_out, k_out};
  }
  check_capture({&q, &k, opt(wq), opt(wk)});
  auto out = QkNormRotary::apply(q, k, wq, wk, cos, sin, pos, interleaved, eps);
  return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_flash_attn_host, m) {
  m.def("bind", &bind);
  m.def("kvcache", &kvcache);
  m.def("commit", &commit);
  m.def("evict", &evict);
  m.def("norm_rotary", &norm_rotary);
}
