// Python bindings of the attention operators. Unlike the library's other bindings they take torch tensors: checks,
// outputs, workspaces and launches of a call are done here, because in Python they take 20 us and more, several times
// what the kernels of a decode step take. What is refused raises ValueError or TypeError before anything touches a
// device.
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

#include "attention_kernels.hpp"

namespace py = pybind11;

namespace rocshmem {
namespace kernels {

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

template <typename... T>
std::string text(const T &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}
template <typename... T>
[[noreturn]] void bad_value(const T &...parts) { throw py::value_error(text(parts...)); }
template <typename... T>
[[noreturn]] void bad_type(const T &...parts) { throw py::type_error(text(parts...)); }

void check(int rc, const char *what) {
  if (rc != 0) throw std::runtime_error(text(what, ": CUDA error ", rc));
}

// The launchers' code of a type, -1 if they have none.
int code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return ATTN_BF16;
    case at::kHalf: return ATTN_F16;
    case at::kFloat: return ATTN_F32;
    case at::kFloat8_e4m3fn: return ATTN_E4M3;
    default: return -1;
  }
}
bool is_float(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }
bool is_half(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool aligned(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
void *data(const Tensor &t) { return const_cast<void *>(t.const_data_ptr()); }

// Tensors inside a torch.func transform are wrappers without memory of their own. Called before an address is taken.
void no_transform(const char *what, std::initializer_list<const Tensor *> tensors) {
  static const c10::DispatchKeySet wrappers({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
      c10::DispatchKey::Batched, c10::DispatchKey::Functionalize});
  for (const Tensor *t : tensors) {
    if (t != nullptr && t->key_set().has_any(wrappers)) {
      bad_value(what, " cannot be called inside a torch.func transform (vmap, grad, jvp and the like)");
    }
  }
}

const Tensor *or_null(const OptTensor &t) { return t.has_value() ? &*t : nullptr; }

// Strides of dimensions 0 and 1 of t [tokens, heads, dim], whose rows the kernels read 16 bytes at a time.
struct Strides {
  int64_t token, head;
};
Strides rows(const Tensor &t, const char *name, int64_t heads = -1, int64_t dim = -1) {
  if (t.dim() != 3 || (heads >= 0 && t.size(1) != heads) || (dim >= 0 && t.size(2) != dim)) {
    bad_value(name, " must be [tokens, ", heads >= 0 ? text(heads) : "heads", ", ", dim >= 0 ? text(dim) : "dim",
        "], got ", t.sizes());
  }
  const int64_t vec = 16 / static_cast<int64_t>(t.element_size());
  const Strides s{t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
  if ((t.size(2) > 1 && t.stride(2) != 1) || s.token % vec || s.head % vec || !aligned(t)) {
    bad_value(name, ": rows must be contiguous and 16-byte aligned (strides ", t.strides(), ")");
  }
  if (t.size(0) > INT32_MAX || t.size(1) > INT32_MAX) bad_value(name, " is too large: ", t.sizes());
  return s;
}

// 1 for 64-bit, 0 for 32-bit whole numbers.
int index(const Tensor &t, const char *name, int64_t count) {
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) bad_type(name, " must be int32 or int64");
  if (t.dim() != 1 || t.size(0) != count || !t.is_contiguous()) bad_value(name, " must be contiguous [", count, "]");
  return t.scalar_type() == at::kLong ? 1 : 0;
}

void no_grad(const char *what, std::initializer_list<const Tensor *> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor *t : tensors) {
    if (t != nullptr && t->requires_grad()) {
      bad_value(what, " has no backward pass: call it under torch.no_grad(), or detach its tensors");
    }
  }
}

// A dual tensor (forward-mode differentiation) does not require a gradient: its tangent would be dropped without a
// word.
void no_tangent(const char *what, std::initializer_list<const Tensor *> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor *t : tensors) {
    if (t != nullptr && t->_fw_grad(/*level=*/0).defined()) {
      bad_value(what, " has no forward-mode derivative: pass primals (torch.autograd.forward_ad.unpack_dual)");
    }
  }
}

void on_one_device(const char *what, std::initializer_list<const Tensor *> tensors) {
  const at::Device device = (*tensors.begin())->device();
  if (!device.is_cuda()) bad_value(what, ": tensors must be on a CUDA device");
  for (const Tensor *t : tensors) {
    if (t != nullptr && t->device() != device) bad_value(what, ": tensors are on ", device, " and ", t->device());
  }
}

// The inputs' device for the duration of a call, and its current stream.
struct Here {
  explicit Here(const Tensor &t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void *stream;
};

// Tells autograd that tensors were written through their addresses, so that a backward pass that has saved one of them
// is refused as after any other operation in place. Inference tensors have no version.
void written(std::initializer_list<const Tensor *> tensors) {
  for (const Tensor *t : tensors) {
    if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
}

// The addresses of a tensor's elements, first to last; nothing for one without elements.
struct Range {
  uintptr_t first = 0, end = 0;
  Range() = default;
  explicit Range(const Tensor &t) {
    if (t.numel() == 0) return;
    int64_t last = 0;
    const auto sizes = t.sizes(), strides = t.strides();
    for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
    first = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    end = first + static_cast<uintptr_t>(last + 1) * t.element_size();
  }
  bool meets(const Range &o) const { return first < o.end && o.first < end; }
};
bool overlap(const Tensor &a, const Tensor &b) { return Range(a).meets(Range(b)); }

void result(const Tensor &t, const char *name, at::IntArrayRef shape, std::initializer_list<at::ScalarType> types,
            std::initializer_list<const Tensor *> inputs) {
  bool ok = t.sizes() == shape && t.is_contiguous() && aligned(t), typed = false;
  for (at::ScalarType s : types) typed = typed || t.scalar_type() == s;
  if (!ok || !typed) bad_value(name, " must be a contiguous, 16-byte aligned tensor of shape ", shape, " and type ",
      *types.begin(),
                               types.size() > 1 ? " or float" : "", ", got ", t.sizes(), " ", t.scalar_type());
  for (const Tensor *x : inputs) {
    if (x != nullptr && overlap(t, *x)) bad_value(name, " shares memory with an input");
  }
}

// ---- norm and rotation --------------------------------------------------------------------------------------------

NormRopeArgs norm_rope_args(const Tensor &q, const Tensor &k, const Tensor &q_weight, const Tensor &k_weight,
    const Tensor &positions, const Tensor &table, double eps, bool interleaved) {
  no_transform("qk_norm_rope", {&q, &k, &q_weight, &k_weight, &positions, &table});
  if (!is_float(q.scalar_type()) || k.scalar_type() != q.scalar_type()) {
    bad_type("q and k must both be bf16, fp16 or fp32, got ", q.scalar_type(), " and ", k.scalar_type());
  }
  const Strides sq = rows(q, "q");
  const int64_t T = q.size(0), D = q.size(2);
  const Strides sk = rows(k, "k", -1, D);
  if (k.size(0) != T || q.size(1) < 1 || k.size(1) < 1) {
    bad_value("q and k must have the same tokens and at least one head, got ", q.sizes(), " and ", k.sizes());
  }
  if (D % 8 || D < 8 || D > 256) bad_value("the head dimension must be a multiple of 8 up to 256, got ", D);
  for (const auto &[w, name] : {std::make_pair(&q_weight, "q_weight"), std::make_pair(&k_weight, "k_weight")}) {
    if ((w->scalar_type() != q.scalar_type() && w->scalar_type() != at::kFloat) ||
        w->scalar_type() != q_weight.scalar_type()) {
      bad_type(name, " must be ", q.scalar_type(), " or fp32, both weights the same");
    }
    if (w->dim() != 1 || w->size(0) != D || !w->is_contiguous() || !aligned(*w)) {
      bad_value(name, " must be contiguous [", D, "], 16-byte aligned");
    }
  }
  if (table.scalar_type() != at::kFloat || table.dim() != 2 || !table.is_contiguous() || !aligned(table)) {
    bad_value("table must be contiguous fp32 [positions, rotary], 16-byte aligned");
  }
  const int64_t R = table.size(1);
  if (R % 16 || R < 16 || R > D || table.size(0) < 1 || table.size(0) > INT32_MAX) {
    bad_value("the table's rows must have a multiple of 16 elements up to ", D, ", got ", table.sizes());
  }
  // In the kernels' type: an eps that becomes zero there makes rows of zeros NaN.
  const float eps32 = static_cast<float>(eps);
  if (!(eps >= 0 && std::isfinite(eps32) && (eps32 > 0 || eps == 0))) {
    bad_value("eps must not be negative, and a finite fp32 number that is not zero unless it is 0 itself, got ", eps);
  }
  const int wide = index(positions, "positions", T);
  if (at::GradMode::is_enabled() && table.requires_grad()) {
    bad_value("qk_norm_rope has no gradient for its table: detach it");
  }
  no_tangent("qk_norm_rope", {&q, &k, &q_weight, &k_weight, &table});
  on_one_device("qk_norm_rope", {&q, &k, &q_weight, &k_weight, &positions, &table});
  NormRopeArgs a{};
  a.q = data(q);
  a.k = data(k);
  a.q_token = sq.token;
  a.q_head = sq.head;
  a.k_token = sk.token;
  a.k_head = sk.head;
  a.q_weight = data(q_weight);
  a.k_weight = data(k_weight);
  a.positions = data(positions);
  a.table = static_cast<const float *>(data(table));
  a.tokens = static_cast<int>(T);
  a.q_heads = static_cast<int>(q.size(1));
  a.k_heads = static_cast<int>(k.size(1));
  a.dim = static_cast<int>(D);
  a.rotary = static_cast<int>(R);
  a.table_rows = static_cast<int>(table.size(0));
  a.eps = eps32;
  a.interleaved = interleaved;
  a.type = code(q.scalar_type());
  a.weight_type = code(q_weight.scalar_type());
  a.wide_positions = wide;
  return a;
}

std::pair<Tensor, Tensor> py_qk_norm_rope(const Tensor &q, const Tensor &k, const Tensor &q_weight,
    const Tensor &k_weight, const Tensor &positions, const Tensor &table, double eps, bool interleaved) {
  const NormRopeArgs a = norm_rope_args(q, k, q_weight, k_weight, positions, table, eps, interleaved);
  const Here here(q);
  Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
  check(qk_norm_rope(a, data(q_out), data(k_out), here.stream), "qk_norm_rope");
  return {q_out, k_out};
}

// A leaf whose gradients an eager graph, alive at the time, accumulates on another stream cannot take part in a
// captured backward pass: the engine would make that stream wait for the captured one, which ends the process. Refused
// instead.
void check_capture(void *stream, int device, std::initializer_list<const Tensor *> tensors) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  check(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status), "qk_norm_rope");
  if (status == cudaStreamCaptureStatusNone) return;
  for (const Tensor *t : tensors) {
    if (!t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto of_node = node->stream();
    if (of_node.has_value() && *of_node != c10::cuda::getCurrentCUDAStream(device).unwrap()) {
      throw std::runtime_error("qk_norm_rope: a graph of the same leaves from outside the capture is alive; drop it "
                               "(its outputs and losses) before a backward pass is captured");
    }
  }
}

struct NormRopeFunction : torch::autograd::Function<NormRopeFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k,
      const Tensor &q_weight, const Tensor &k_weight, const Tensor &positions, const Tensor &table, double eps,
      bool interleaved) {
    ctx->save_for_backward({q, k, q_weight, k_weight, positions, table});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    auto both = py_qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved);
    return {both.first, both.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
      torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled()) {
      throw std::runtime_error("qk_norm_rope can be differentiated once: create_graph is refused");
    }
    no_transform("qk_norm_rope's backward pass", {&grads[0], &grads[1]});
    no_tangent("qk_norm_rope's backward pass", {&grads[0], &grads[1]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &q_weight = saved[2], &k_weight = saved[3], &table = saved[5];
    const NormRopeArgs a = norm_rope_args(q, k, q_weight, k_weight, saved[4], table, ctx->saved_data["eps"].toDouble(),
        ctx->saved_data["interleaved"].toBool());
    const Here here(q);
    // Gradients come in any layout (an expanded one behind a sum, for instance); the kernel reads plain rows.
    auto plain = [](const Tensor &g) {
      return g.is_contiguous() && aligned(g) ? g : g.clone(at::MemoryFormat::Contiguous);
    };
    const Tensor gq = plain(grads[0]), gk = plain(grads[1]);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dwq = at::empty(q_weight.sizes(), q_weight.options()), dwk = at::empty(k_weight.sizes(), k_weight.options());
    Tensor workspace = at::empty({static_cast<int64_t>(qk_norm_rope_workspace(a.dim))}, table.options());
    check(qk_norm_rope_backward(a, data(gq), data(gk), data(dq), data(dk), data(dwq), data(dwk),
        static_cast<float *>(data(workspace)), here.stream), "qk_norm_rope_backward");
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> py_qk_norm_rope_any(const Tensor &q, const Tensor &k, const Tensor &q_weight,
    const Tensor &k_weight, const Tensor &positions, const Tensor &table, double eps, bool interleaved) {
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || q_weight.requires_grad() ||
      k_weight.requires_grad())) {
    return py_qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved);
  }
  norm_rope_args(q, k, q_weight, k_weight, positions, table, eps, interleaved);  // refused before a graph is begun
  {
    const Here here(q);
    check_capture(here.stream, q.device().index(), {&q, &k, &q_weight, &k_weight});
  }
  auto both = NormRopeFunction::apply(q, k, q_weight, k_weight, positions, table, eps, interleaved);
  return {both[0], both[1]};
}

// ---- the paged cache ------------------------------------------------------------------------------------------------

struct Cache {
  Tensor k, v;
  OptTensor k_scale, v_scale;
};

KvCacheArgs cache_args(const Cache &c) {
  const Tensor &k = c.k, &v = c.v;
  no_transform("KvCache", {&k, &v, or_null(c.k_scale), or_null(c.v_scale)});
  if (k.dim() != 4 || v.sizes() != k.sizes() || k.scalar_type() != v.scalar_type() ||
      !(is_half(k.scalar_type()) || k.scalar_type() == at::kFloat8_e4m3fn)) {
    bad_value("KvCache: k and v must both be [pages, kv_heads, page_size, head_dim] in bf16, fp16 or e4m3");
  }
  const int64_t pages = k.size(0), heads = k.size(1), size = k.size(2), dim = k.size(3);
  if (size < 1 || size > (1 << 20) || (size & (size - 1))) {
    bad_value("KvCache: the page size must be a power of two up to 2^20, got ", size);
  }
  if (heads < 1 || heads > (1 << 20) || pages > INT32_MAX || dim % 8 || dim < 8 || dim > 256) {
    bad_value("KvCache: at least one head, head_dim a multiple of 8 up to 256");
  }
  if (pages * heads * size > INT32_MAX) {
    bad_value("KvCache: at most 2^31 - 1 rows (pages * kv_heads * page_size), got ", pages * heads * size);
  }
  const bool scaled = k.scalar_type() == at::kFloat8_e4m3fn;
  for (const OptTensor *s : {&c.k_scale, &c.v_scale}) {
    if (scaled && (!s->has_value() || (*s)->scalar_type() != at::kFloat || (*s)->sizes() != k.sizes().slice(0, 3))) {
      bad_value("KvCache: e4m3 needs k_scale and v_scale, fp32 [pages, kv_heads, page_size]");
    }
    if (!scaled && s->has_value()) bad_value("KvCache: only e4m3 caches have scales");
  }
  for (const Tensor *t : {&c.k, &c.v, or_null(c.k_scale), or_null(c.v_scale)}) {
    if (t != nullptr && (!t->is_contiguous() || !aligned(*t) || t->device() != k.device())) {
      bad_value("KvCache: tensors must be contiguous, 16-byte aligned and on one device");
    }
  }
  for (const Tensor *t : {&c.k, &c.v, or_null(c.k_scale), or_null(c.v_scale)}) {
    if (t != nullptr && t->requires_grad()) {
      bad_value("KvCache: the cache is written in place and cannot require a gradient");
    }
  }
  no_tangent("KvCache", {&c.k, &c.v, or_null(c.k_scale), or_null(c.v_scale)});
  int shift = 0;
  while ((int64_t{1} << shift) < size) ++shift;
  return KvCacheArgs{data(k), data(v), scaled ? static_cast<float *>(data(*c.k_scale)) : nullptr,
      scaled ? static_cast<float *>(data(*c.v_scale)) : nullptr, static_cast<int>(pages), static_cast<int>(heads),
      shift, static_cast<int>(dim), code(k.scalar_type())};
}

void py_kv_cache_write(const Cache &c, const Tensor &k, const Tensor &v, const Tensor &slots) {
  const KvCacheArgs a = cache_args(c);
  no_transform("kv_cache_write", {&k, &v, &slots});
  if (!is_float(k.scalar_type()) || v.scalar_type() != k.scalar_type()) {
    bad_type("k and v must both be bf16, fp16 or fp32, got ", k.scalar_type(), " and ", v.scalar_type());
  }
  const Strides sk = rows(k, "k", a.kv_heads, a.dim), sv = rows(v, "v", a.kv_heads, a.dim);
  if (v.size(0) != k.size(0)) bad_value("k and v must have the same tokens, got ", k.size(0), " and ", v.size(0));
  const int wide = index(slots, "slots", k.size(0));
  no_grad("kv_cache_write", {&k, &v});
  no_tangent("kv_cache_write", {&k, &v});
  const Range in[3] = {Range(k), Range(v), Range(slots)};
  Range parts[4];
  int n = 0;
  for (const Tensor *t : {&c.k, &c.v, or_null(c.k_scale), or_null(c.v_scale)}) {
    if (t == nullptr) continue;
    const Range r(*t);
    for (const Range &x : in) {
      if (r.meets(x)) bad_value("kv_cache_write: k, v or slots shares memory with the cache");
    }
    for (int i = 0; i < n; ++i) {
      if (r.meets(parts[i])) bad_value("kv_cache_write: the cache's tensors share memory with one another");
    }
    parts[n++] = r;
  }
  on_one_device("kv_cache_write", {&k, &v, &slots, &c.k});
  const Here here(k);
  check(kv_cache_write(a, data(k), data(v), sk.token, sk.head, sv.token, sv.head, data(slots), wide,
      static_cast<int>(k.size(0)), code(k.scalar_type()), here.stream), "kv_cache_write");
  written({&c.k, &c.v, or_null(c.k_scale), or_null(c.v_scale)});
}

std::pair<Tensor, Tensor> py_kv_cache_read(const Cache &c, const Tensor &slots, at::ScalarType dtype) {
  const KvCacheArgs a = cache_args(c);
  no_transform("kv_cache_read", {&slots});
  if (!is_float(dtype)) bad_type("dtype must be bf16, fp16 or fp32, got ", dtype);
  if (slots.dim() != 1 || slots.size(0) > INT32_MAX) bad_value("slots must be [T]");
  const int64_t T = slots.size(0);
  const int wide = index(slots, "slots", T);
  on_one_device("kv_cache_read", {&slots, &c.k});
  const Here here(slots);
  const auto options = c.k.options().dtype(dtype);
  Tensor k = at::empty({T, a.kv_heads, a.dim}, options), v = at::empty({T, a.kv_heads, a.dim}, options);
  check(kv_cache_read(a, data(k), data(v), data(slots), wide, static_cast<int>(T), code(dtype), here.stream),
      "kv_cache_read");
  return {k, v};
}

// ---- attention over the cache -------------------------------------------------------------------------------------

constexpr double kSmallest = 1e-30;

struct Paged {
  KvCacheArgs cache;
  PagedAttentionArgs args;
};

// Everything that does not depend on a device.
Paged check_paged(const Tensor &q, const Cache &c, const Tensor &block_table, const Tensor &lengths,
    std::optional<double> scale, double softcap, int64_t window) {
  Paged p{cache_args(c), {}};
  no_transform("paged_attention", {&q, &block_table, &lengths});
  if (!is_half(q.scalar_type()) || (p.cache.type != ATTN_E4M3 && p.cache.type != code(q.scalar_type()))) {
    bad_type("q must be bf16 or fp16, and of the cache's type unless that is e4m3: got ", q.scalar_type(), " and ",
        c.k.scalar_type());
  }
  const Strides s = rows(q, "q", -1, p.cache.dim);
  const int64_t B = q.size(0), H = q.size(1), D = q.size(2);
  if (H < 1 || H % p.cache.kv_heads) {
    bad_value("the ", H, " query heads must be a multiple of the cache's ", p.cache.kv_heads);
  }
  if (D != 64 && D != 96 && D != 128 && D != 256) {
    bad_value("paged_attention: the head dimension must be 64, 96, 128 or 256, got ", D);
  }
  if (block_table.scalar_type() != at::kInt || lengths.scalar_type() != at::kInt) {
    bad_type("block_table and lengths must be int32");
  }
  if (block_table.dim() != 2 || block_table.size(0) != B || (block_table.size(1) > 1 && block_table.stride(1) != 1)) {
    bad_value("block_table must be [", B, ", pages] with contiguous rows");
  }
  if (lengths.dim() != 1 || lengths.size(0) != B || !lengths.is_contiguous()) {
    bad_value("lengths must be contiguous [", B, "]");
  }
  const double f = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  if (!(f > 0 && f < 1e30) || !(softcap >= 0 && softcap < 1e30) || window < 0) {
    bad_value("scale must be positive, softcap and window not negative");
  }
  // The kernels take both as fp32 and the cap's reciprocal: what would become zero there, no cap at all, or lose digits
  // is refused.
  if (f < kSmallest || (softcap > 0 && softcap < kSmallest)) {
    bad_value("scale and softcap (unless it is 0) must be at least ", kSmallest, ", got ", f, " and ", softcap);
  }
  const int64_t most = block_table.size(1) * c.k.size(2);
  if (most > INT32_MAX - 256) {
    bad_value("paged_attention: a sequence's pages hold at most 2^31 - 257 tokens, got ", most);
  }
  PagedAttentionArgs &a = p.args;
  a.q = data(q);
  a.q_token = s.token;
  a.q_head = s.head;
  a.block_table = static_cast<const int *>(data(block_table));
  a.table_stride = block_table.stride(0);
  a.lengths = static_cast<const int *>(data(lengths));
  a.batch = static_cast<int>(B);
  a.heads = static_cast<int>(H);
  a.max_pages = static_cast<int>(block_table.size(1));
  a.window = static_cast<int>(std::min<int64_t>(window, INT32_MAX));
  a.scale = static_cast<float>(f);
  a.softcap = static_cast<float>(softcap);
  a.q_type = code(q.scalar_type());
  return p;
}

std::pair<Tensor, OptTensor> py_paged_attention(const Tensor &q, const Cache &c, const Tensor &block_table,
    const Tensor &lengths, std::optional<double> scale, double softcap, int64_t window, const OptTensor &out_given,
    const OptTensor &lse_given, bool want_lse) {
  Paged p = check_paged(q, c, block_table, lengths, scale, softcap, window);
  const std::initializer_list<const Tensor *> inputs = {&q, &block_table, &lengths, &c.k, &c.v, or_null(c.k_scale),
      or_null(c.v_scale)};
  no_transform("paged_attention", {or_null(out_given), or_null(lse_given)});
  if (out_given) {
    result(*out_given, "out", q.sizes(), {q.scalar_type(), at::kFloat}, inputs);
    if (lse_given && overlap(*out_given, *lse_given)) bad_value("out shares memory with lse");
  }
  if (lse_given) result(*lse_given, "lse", q.sizes().slice(0, 2), {at::kFloat}, inputs);
  no_grad("paged_attention", {&q, or_null(out_given), or_null(lse_given)});
  no_tangent("paged_attention", {&q, or_null(out_given), or_null(lse_given)});
  on_one_device("paged_attention", {&q, &block_table, &lengths, &c.k, or_null(out_given), or_null(lse_given)});
  const Here here(q);
  const auto fp32 = q.options().dtype(at::kFloat);
  Tensor out = out_given ? *out_given : at::empty(q.sizes(), q.options());
  OptTensor lse = lse_given;
  if (!lse && want_lse) lse = at::empty(q.sizes().slice(0, 2), fp32);
  const size_t bytes = paged_attention_workspace(p.cache, p.args);
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes / 4)}, fp32);
  p.args.out = data(out);
  p.args.out_type = code(out.scalar_type());
  p.args.lse = lse ? static_cast<float *>(data(*lse)) : nullptr;
  check(paged_attention(p.cache, p.args, bytes > 0 ? data(workspace) : nullptr, bytes, here.stream), "paged_attention");
  written({or_null(out_given), or_null(lse_given)});
  return {out, lse};
}

std::pair<Tensor, Tensor> py_attention_join(const Tensor &outs, const Tensor &lses,
    std::optional<at::ScalarType> dtype_given, const OptTensor &out_given) {
  no_transform("attention_join", {&outs, &lses, or_null(out_given)});
  if (!is_float(outs.scalar_type()) || lses.scalar_type() != at::kFloat) {
    bad_type("outs must be bf16, fp16 or fp32, lses fp32");
  }
  if (outs.dim() != 4 || lses.sizes() != outs.sizes().slice(0, 3) || outs.size(0) < 1 || outs.size(0) > INT32_MAX) {
    bad_value("outs must be [n, B, H, D] and lses [n, B, H], got ", outs.sizes(), " and ", lses.sizes());
  }
  const int64_t n = outs.size(0), B = outs.size(1), H = outs.size(2), D = outs.size(3);
  if (D % 8 || D < 8 || D > 256) bad_value("the head dimension must be a multiple of 8 up to 256, got ", D);
  auto packed = [](const Tensor &t) {  // every part contiguous
    int64_t expect = 1;
    for (int64_t i = t.dim() - 1; i > 0; --i) {
      if (t.size(i) > 1 && t.stride(i) != expect) return false;
      expect *= t.size(i);
    }
    return true;
  };
  if (outs.numel() > 0 && (!packed(outs) || !packed(lses))) bad_value("attention_join: every part must be contiguous");
  const int64_t outs_part = n > 1 ? outs.stride(0) : 0, lse_part = n > 1 ? lses.stride(0) : 0;
  if (!aligned(outs) || outs_part * static_cast<int64_t>(outs.element_size()) % 16) {
    bad_value("attention_join: every part of outs must be 16-byte aligned");
  }
  const at::ScalarType dtype = dtype_given ? *dtype_given : out_given ? out_given->scalar_type() : outs.scalar_type();
  if (!is_float(dtype)) bad_type("dtype must be bf16, fp16 or fp32, got ", dtype);
  if (out_given) result(*out_given, "out", outs.sizes().slice(1), {dtype}, {&outs, &lses});
  no_grad("attention_join", {&outs, &lses, or_null(out_given)});
  no_tangent("attention_join", {&outs, &lses, or_null(out_given)});
  on_one_device("attention_join", {&outs, &lses, or_null(out_given)});
  const Here here(outs);
  Tensor out = out_given ? *out_given : at::empty(outs.sizes().slice(1), outs.options().dtype(dtype));
  Tensor lse = at::empty(lses.sizes().slice(1), lses.options());
  check(attention_join(data(outs), static_cast<const float *>(data(lses)), outs_part, lse_part, static_cast<int>(n),
      B * H, static_cast<int>(D), code(outs.scalar_type()), code(dtype), data(out), static_cast<float *>(data(lse)),
      here.stream), "attention_join");
  written({or_null(out_given)});
  return {out, lse};
}

}  // namespace

#define ROCSHMEM_TEXT_OF(x) #x
#define ROCSHMEM_TEXT(x) ROCSHMEM_TEXT_OF(x)
// The version that these objects fit. Read from the file before it is loaded.
const char kBuiltFor[] = "rocshmem_b200._A for torch " ROCSHMEM_TEXT(ROCSHMEM_TORCH_VERSION);

PYBIND11_MODULE(_A, m) {
  m.doc() = "Attention operators on torch tensors";
  m.attr("built_for") = kBuiltFor;
  py::class_<Cache>(m, "Cache").def(py::init([](const Tensor &k, const Tensor &v, const OptTensor &ks,
      const OptTensor &vs) {
    Cache c{k, v, ks, vs};
    cache_args(c);
    return c;
  }));
  m.def("qk_norm_rope", &py_qk_norm_rope_any);
  m.def("kv_cache_write", &py_kv_cache_write);
  m.def("kv_cache_read", &py_kv_cache_read);
  m.def("check_paged", [](const Tensor &q, const Cache &c, const Tensor &table, const Tensor &lengths,
      std::optional<double> scale, double softcap, int64_t window) {
    check_paged(q, c, table, lengths, scale, softcap, window);
  });
  m.def("paged_attention", &py_paged_attention);
  m.def("attention_join", &py_attention_join);
}

}  // namespace kernels
}  // namespace rocshmem
