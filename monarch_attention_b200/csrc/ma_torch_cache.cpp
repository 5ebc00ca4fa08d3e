// Native halves of the rotary positions, the paged cache and the attention over it: input checks, results and
// workspaces from PyTorch's caching allocator, and the launches through the C ABI.
#include <ATen/ExpandUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>

#include "ma_torch.h"

namespace ma_torch {
namespace {

using at::Tensor;
using std::optional;

const Tensor& tensor_of(PyObject* x, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(x), name, " must be a tensor");
  return THPVariable_Unpack(x);
}
optional<Tensor> optional_of(PyObject* x, const char* name) {
  if (x == Py_None) return std::nullopt;
  return tensor_of(x, name);
}

void check_python() {
  if (PyErr_Occurred()) throw python_error();
}

// ---------------------------------------------------------------------------------------------- who writes where

// A tensor's dimensions of more than one element, the largest stride first.
struct Places {
  struct Dim {
    int64_t size, stride;
    bool operator==(const Dim& o) const { return size == o.size && stride == o.stride; }
  };
  c10::SmallVector<Dim, 4> dims;
  const char *begin, *end;  // bytes from its first element to behind its last
  int64_t item;

  explicit Places(const Tensor& t) : begin(static_cast<const char*>(t.data_ptr())), item(t.element_size()) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) > 1) dims.push_back({t.size(i), t.stride(i)});
      last += (t.size(i) - 1) * t.stride(i);
    }
    std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    end = begin + (t.numel() > 0 ? (last + 1) * item : 0);
  }
  // Each stride passes over all that the smaller ones reach, so that no two elements are in one place.  (Others may have that too; they are not taken.)
  bool distinct() const {
    if (begin == end) return true;
    int64_t reach = 0;
    for (size_t i = dims.size(); i-- > 0;) {
      if (dims[i].stride <= reach) return false;
      reach += (dims[i].size - 1) * dims[i].stride;
    }
    return true;
  }
  // Two elements of dims[i ..] are `distance` apart.
  bool differ_by(int64_t distance, size_t i = 0) const {
    if (i == dims.size()) return distance == 0;
    int64_t n = distance / dims[i].stride - (distance % dims[i].stride < 0);
    for (int64_t k = n; k <= n + 1; ++k)
      if (k > -dims[i].size && k < dims[i].size && differ_by(distance - k * dims[i].stride, i + 1)) return true;
    return false;
  }
};
// Whether an element of a is in the place of one of b, both with distinct elements; true as well where that is not seen from equal strides.
bool meet(const Places& a, const Places& b) {
  if (a.end <= b.begin || b.end <= a.begin) return false;
  const int64_t distance = b.begin - a.begin;
  return !(a.dims == b.dims) || a.item != b.item || distance % a.item != 0 || a.differ_by(distance / a.item);
}

// ---------------------------------------------------------------------------------------------- rotary positions

struct Rotary {
  Tensor turns;  // int64 on the host, dim / 2 entries
  int64_t dim, pairs;
  double magnitude;
};

Rotary rotary_of(PyObject* turns, PyObject* dim, PyObject* pairs, PyObject* magnitude) {
  Rotary r{tensor_of(turns, "rotary.turns"), PyLong_AsLongLong(dim), PyLong_AsLongLong(pairs), PyFloat_AsDouble(magnitude)};
  check_python();
  TORCH_CHECK_VALUE(r.turns.device().is_cpu() && r.turns.scalar_type() == at::kLong && r.turns.is_contiguous() && r.turns.numel() * 2 == r.dim,
                    "rotary.turns must be a contiguous int64 tensor of dim / 2 entries on the host");
  return r;
}

ma_b200_rotary rotary_struct(const Rotary& r) {
  return {(int32_t)r.dim, (int32_t)r.pairs, (float)r.magnitude, reinterpret_cast<const uint64_t*>(r.turns.data_ptr<int64_t>())};
}

void check_rotated(const Tensor& q, const optional<Tensor>& k, const optional<Tensor>& positions) {
  TORCH_CHECK_VALUE(q.dim() == 4, "query must have shape (batch, heads, tokens, width)");
  TORCH_CHECK(q.is_cuda(), "monarch_attention_b200 runs on CUDA tensors only (there is no CPU path)");
  TORCH_CHECK_VALUE(dtype_code(q.scalar_type()) >= 0, "unsupported dtype ", q.scalar_type());
  if (k.has_value()) {
    TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == q.size(0) && k->size(2) == q.size(2) && k->size(3) == q.size(3), "key shape ", k->sizes(),
                      " does not match query shape ", q.sizes(), " in batch, tokens and width");
    TORCH_CHECK_VALUE(k->device() == q.device() && k->scalar_type() == q.scalar_type(), "query and key must have the same dtype and device");
  }
  if (positions.has_value()) {
    TORCH_CHECK_VALUE(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt, "positions must be int32 or int64");
    TORCH_CHECK_VALUE(positions->device() == q.device(), "positions must be on the query's device");
    TORCH_CHECK_VALUE(positions->dim() >= 1 && positions->dim() <= 2 && positions->size(-1) == q.size(2) &&
                          (positions->dim() == 1 || positions->size(0) == q.size(0) || positions->size(0) == 1),
                      "positions must have shape (tokens) or (batch, tokens), got ", positions->sizes());
  }
}

// An uninitialised tensor of t's shape and order of strides (at::empty_like without its way through the dispatcher).
Tensor new_like(const Tensor& t) {
  const at::TensorOptions o = at::TensorOptions().dtype(t.scalar_type()).device(t.device());
  if (t.is_non_overlapping_and_dense()) return at::detail::empty_strided_cuda(t.sizes(), t.strides(), o);
  const auto strides = at::infer_dense_strides(t.sizes(), t.strides());
  if (strides.back() != 1 && t.size(-1) != 1) return at::detail::empty_cuda(t.sizes(), o);  // (features next to one another whatever is expanded)
  return at::detail::empty_strided_cuda(t.sizes(), strides, o);
}

// Rotated copies of q and k (undefined ones are left out).
std::pair<Tensor, Tensor> rotate(const Tensor& q_in, const Tensor& k_in, const Rotary& r, const optional<Tensor>& positions, bool inverse) {
  const Tensor& any = q_in.defined() ? q_in : k_in;
  const c10::cuda::CUDAGuard guard(any.device());
  const Tensor q = q_in.defined() ? unit_inner(q_in) : q_in, k = k_in.defined() ? unit_inner(k_in) : k_in;
  const Tensor q_out = q.defined() ? new_like(q) : q, k_out = k.defined() ? new_like(k) : k;
  const int64_t E = any.size(0), N = any.size(2), D = any.size(3);
  TORCH_CHECK_VALUE(r.dim <= D, "rotary dim ", r.dim, " exceeds the head width ", D);
  ma_b200_rotation p{};
  p.H = q.defined() ? (int32_t)q.size(1) : 0;
  p.Hk = k.defined() ? (int32_t)k.size(1) : 0;
  if (E == 0 || N == 0 || p.H + p.Hk == 0) return {q_out, k_out};
  TORCH_CHECK_VALUE(E <= INT32_MAX && N <= INT32_MAX, "too many batch elements or tokens");
  p.abi_version = MA_B200_ABI_VERSION;
  p.E = (int32_t)E; p.N = (int32_t)N; p.D = (int32_t)D;
  p.dtype = dtype_code(any.scalar_type());
  p.inverse = inverse;
  if (p.H > 0) { p.q = view4(q); p.q_out = view4(q_out); }
  if (p.Hk > 0) { p.k = view4(k); p.k_out = view4(k_out); }
  if (positions.has_value()) {
    p.positions = positions->data_ptr();
    p.positions_i64 = positions->scalar_type() == at::kLong;
    p.pos_stride_n = positions->stride(-1);
    p.pos_stride_e = positions->dim() == 2 && positions->size(0) > 1 ? positions->stride(0) : 0;
  }
  p.rotary = rotary_struct(r);
  raise_for_status(ma_b200_rotary_apply(&p, c10::cuda::getCurrentCUDAStream().stream()));
  return {q_out, k_out};
}

std::pair<Tensor, Tensor> rotate_any(const Tensor& q, const Tensor& k, const Rotary& r, const optional<Tensor>& positions, bool inverse);

// The rotation is linear: its gradient is the inverse rotation (times the magnitude again), itself differentiable.  A node of its own:
// a training step of a small layer is bound by the host, and the general function object with its dictionary costs it 20 us.
struct RotaryBackward : torch::autograd::Node {
  Rotary rotary;
  torch::autograd::SavedVariable positions;
  bool has_positions, inverse;

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::pair<Tensor, Tensor> d;
    const Tensor dx = grads[0], dy = grads.size() > 1 ? grads[1] : Tensor();
    if (dx.defined() || dy.defined())
      d = rotate_any(dx, dy, rotary, has_positions ? optional<Tensor>(positions.unpack()) : std::nullopt, !inverse);
    if (grads.size() > 1) return {d.first, d.second};
    return {d.first};
  }
  void release_variables() override { positions.reset_data(); }
  std::string name() const override { return "RotaryBackward"; }
};

// Rotated copies of x and (where defined) y, both of which need a gradient.
std::pair<Tensor, Tensor> rotate_with_history(const Tensor& x, const Tensor& y, const Rotary& r, const optional<Tensor>& positions, bool inverse) {
  const auto out = rotate(x.detach(), y.defined() ? y.detach() : y, r, positions, inverse);
  const std::shared_ptr<RotaryBackward> node(new RotaryBackward, torch::autograd::deleteNode);
  node->rotary = r;
  node->has_positions = positions.has_value();
  if (positions.has_value()) node->positions = torch::autograd::SavedVariable(*positions, false);
  node->inverse = inverse;
  node->set_next_edges(y.defined() ? torch::autograd::collect_next_edges(x, y) : torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(out.first, node);
  if (y.defined()) torch::autograd::set_history(out.second, node);
  return out;
}

std::pair<Tensor, Tensor> rotate_reverse(const Tensor& q, const Tensor& k, const Rotary& r, const optional<Tensor>& positions, bool inverse) {
  const bool grad = at::GradMode::is_enabled();
  const bool gq = grad && q.defined() && q.requires_grad(), gk = grad && k.defined() && k.requires_grad();
  if (!gq && !gk) return rotate(q, k, r, positions, inverse);
  if (gq && gk) return rotate_with_history(q, k, r, positions, inverse);
  // one of the two has no gradient: its result is not to hang on the other's graph
  if (gq) return {rotate_with_history(q, Tensor(), r, positions, inverse).first, k.defined() ? rotate(Tensor(), k, r, positions, inverse).second : k};
  return {q.defined() ? rotate(q, Tensor(), r, positions, inverse).first : q, rotate_with_history(k, Tensor(), r, positions, inverse).first};
}

// (Either of q and k may be undefined.)  In forward mode a result's tangent is the rotated tangent.
std::pair<Tensor, Tensor> rotate_any(const Tensor& q, const Tensor& k, const Rotary& r, const optional<Tensor>& positions, bool inverse) {
  const auto out = rotate_reverse(q, k, r, positions, inverse);
  if (!has_tangent(q) && !has_tangent(k)) return out;
  auto tangent = [](const Tensor& t) {
    Tensor d = has_tangent(t) ? t._fw_grad(0) : Tensor();
    if (d.defined() && d._is_zerotensor()) d = at::zeros(d.sizes(), d.options());  // (which has no memory)
    return d;
  };
  const Tensor dq = tangent(q), dk = tangent(k);
  const auto d = rotate_any(dq, dk, r, positions, inverse);
  if (dq.defined()) out.first._set_fw_grad(d.first, 0, false);
  if (dk.defined()) out.second._set_fw_grad(d.second, 0, false);
  return out;
}

// ---------------------------------------------------------------------------------------------- paged cache

struct Cache {
  const Tensor &k, &v, &k_scale, &v_scale;
};

ma_b200_cache cache_struct(const Cache& c, const at::Device& device) {
  TORCH_CHECK_VALUE(c.k.dim() == 4 && c.v.sizes() == c.k.sizes(), "the cache's k and v must have one shape (pages, heads, page size, width)");
  TORCH_CHECK_VALUE(c.k.scalar_type() == at::kFloat8_e4m3fn && c.v.scalar_type() == at::kFloat8_e4m3fn, "the cache's k and v must be float8_e4m3fn");
  TORCH_CHECK_VALUE(c.k.device() == device && c.v.device() == device && c.k_scale.device() == device && c.v_scale.device() == device,
                    "the cache must be on the query's or key's device");
  for (const Tensor* t : {&c.k, &c.v, &c.k_scale, &c.v_scale}) {
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !t->requires_grad(), "the cache requires a gradient: the cached operators have none (torch.no_grad())");
    check_no_tangent(*t, "the cache");
  }
  TORCH_CHECK_VALUE(c.k.stride(3) == 1 && c.v.stride(3) == 1, "the features of the cache's k and v must lie next to one another");
  for (const Tensor* s : {&c.k_scale, &c.v_scale}) {
    TORCH_CHECK_VALUE(s->scalar_type() == at::kFloat && s->dim() == 3 && s->size(0) == c.k.size(0) && s->size(1) == c.k.size(1) &&
                          s->size(2) * 16 == c.k.size(2),
                      "the cache's scales must be float32 of shape (pages, heads, page size / 16)");
    TORCH_CHECK_VALUE(s->stride(2) == 1 || s->size(2) == 1, "the scales of a page and head must lie next to one another");
  }
  TORCH_CHECK_VALUE(c.k.size(0) <= INT32_MAX && c.k.size(1) <= INT32_MAX && c.k.size(2) <= INT32_MAX && c.k.size(3) <= INT32_MAX, "the cache is too large");
  return {c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr<float>(), c.v_scale.data_ptr<float>(),
          (int32_t)c.k.size(0), (int32_t)c.k.size(1), (int32_t)c.k.size(2), (int32_t)c.k.size(3),
          c.k.stride(0), c.k.stride(1), c.k.stride(2), c.v.stride(0), c.v.stride(1), c.v.stride(2),
          c.k_scale.stride(0), c.k_scale.stride(1), c.v_scale.stride(0), c.v_scale.stride(1)};
}

ma_b200_sequences sequences_struct(const Tensor& table, const Tensor& lengths, const optional<Tensor>& counts, int64_t E, const at::Device& device) {
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == E && table.size(1) > 0 && table.size(1) <= INT32_MAX,
                    "page_table must be int32 of shape (batch, pages of a sequence)");
  TORCH_CHECK_VALUE(table.stride(1) == 1 || table.size(1) == 1, "the rows of page_table must be contiguous");
  TORCH_CHECK_VALUE(lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == E && lengths.is_contiguous(),
                    "lengths must be contiguous int32 of shape (batch)");
  TORCH_CHECK_VALUE(table.device() == device && lengths.device() == device, "page_table and lengths must be on the query's or key's device");
  if (counts.has_value())
    TORCH_CHECK_VALUE(counts->scalar_type() == at::kInt && counts->dim() == 1 && counts->size(0) == E && counts->is_contiguous() && counts->device() == device,
                      "counts must be contiguous int32 of shape (batch) on the query's or key's device");
  return {table.data_ptr<int32_t>(), table.stride(0), (int32_t)table.size(1), lengths.data_ptr<int32_t>(),
          counts.has_value() ? counts->data_ptr<int32_t>() : nullptr};
}

// Rows that the kernels can read as they are, else a copy.
Tensor aligned(const Tensor& t, size_t bytes) {
  bool fine = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
  for (int i = 0; i < 3; ++i) fine = fine && t.stride(i) % (int64_t)(bytes / t.element_size()) == 0;
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_16bit(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must have shape (batch, heads, tokens, width)");
  TORCH_CHECK(t.is_cuda(), "monarch_attention_b200 runs on CUDA tensors only (there is no CPU path)");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "unsupported dtype ", t.scalar_type(), " (bfloat16 or float16)");
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !t.requires_grad(), name, " requires a gradient: the cached operators have none (torch.no_grad())");
  check_no_tangent(t, name);
  TORCH_CHECK_VALUE(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX && t.size(2) <= INT32_MAX, name, " is too large");
}

Tensor append(const Cache& cache, const Tensor& k_in, const Tensor& v_in, const Tensor& table, const Tensor& lengths, const optional<Tensor>& counts,
              const optional<Tensor>& query, const Rotary* rotary) {
  check_16bit(k_in, "key");
  check_16bit(v_in, "value");
  TORCH_CHECK_VALUE(v_in.sizes() == k_in.sizes() && v_in.scalar_type() == k_in.scalar_type() && v_in.device() == k_in.device(),
                    "key and value must have the same shape, dtype and device");
  const c10::cuda::CUDAGuard guard(k_in.device());
  raise_for_status(ma_b200_poll_cache_status(k_in.device().index()));
  ma_b200_append p{};
  p.abi_version = MA_B200_ABI_VERSION;
  p.cache = cache_struct(cache, k_in.device());
  TORCH_CHECK_VALUE(k_in.size(1) == p.cache.heads && k_in.size(3) == p.cache.width, "key shape ", k_in.sizes(), " does not match the cache's ",
                    p.cache.heads, " heads of ", p.cache.width);
  p.sequences = sequences_struct(table, lengths, counts, k_in.size(0), k_in.device());
  for (const auto& [a, b] : {std::pair<const Tensor&, const Tensor&>(cache.k, cache.v), std::pair<const Tensor&, const Tensor&>(cache.k_scale, cache.v_scale)}) {
    const char *at = static_cast<const char*>(a.data_ptr()), *bt = static_cast<const char*>(b.data_ptr());
    if (a.is_contiguous() && b.is_contiguous() && (at + a.nbytes() <= bt || bt + b.nbytes() <= at)) continue;  // (as allocated: 0.2 us less of the host's 6.5)
    const Places x(a), y(b);
    TORCH_CHECK_VALUE(x.distinct() && y.distinct() && !meet(x, y),
                      "what the append writes must not overlap: pages, heads or tokens of the cache are over one another, or keys over values");
  }
  const size_t lane = 16;
  Tensor q, q_out;
  if (query.has_value()) {
    check_16bit(*query, "query");
    TORCH_CHECK_VALUE(query->size(0) == k_in.size(0) && query->size(2) == k_in.size(2) && query->size(3) == k_in.size(3) &&
                          query->scalar_type() == k_in.scalar_type() && query->device() == k_in.device(),
                      "query must match the key in batch, tokens, width, dtype and device");
    q = aligned(*query, lane);
    q_out = new_like(q);
    p.H = (int32_t)q.size(1);
    p.q = view4(q);
    p.q_out = view4(q_out);
  }
  if (k_in.size(0) == 0 || k_in.size(2) == 0) return q_out;
  const Tensor k = aligned(k_in, lane), v = aligned(v_in, lane);
  p.E = (int32_t)k.size(0); p.N = (int32_t)k.size(2);
  p.dtype = dtype_code(k.scalar_type());
  p.k = view4(k);
  p.v = view4(v);
  ma_b200_rotary r{};
  if (rotary != nullptr) {
    r = rotary_struct(*rotary);
    p.rotary = &r;
  }
  raise_for_status(ma_b200_cache_append(&p, c10::cuda::getCurrentCUDAStream().stream()));
  // (what a graph has saved of the pool is not what it was)
  for (const Tensor* t : {&cache.k, &cache.v, &cache.k_scale, &cache.v_scale})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return q_out;
}

Tensor attend(const Tensor& q_in, const Cache& cache, const Tensor& table, const Tensor& lengths, const optional<Tensor>& counts, bool causal, double scale,
              double softcap, int64_t window, const optional<Tensor>& out_in, bool token_major) {
  check_16bit(q_in, "query");
  const c10::cuda::CUDAGuard guard(q_in.device());
  raise_for_status(ma_b200_poll_device_status(q_in.device().index()));  // (a bounded wait of an earlier call that gave up)
  raise_for_status(ma_b200_poll_cache_status(q_in.device().index()));
  ma_b200_attend p{};
  p.abi_version = MA_B200_ABI_VERSION;
  p.cache = cache_struct(cache, q_in.device());
  TORCH_CHECK_VALUE(q_in.size(3) == p.cache.width && q_in.size(1) > 0 && p.cache.heads > 0 && q_in.size(1) % p.cache.heads == 0, "query shape ",
                    q_in.sizes(), " does not match the cache's ", p.cache.heads, " heads of ", p.cache.width);
  p.sequences = sequences_struct(table, lengths, counts, q_in.size(0), q_in.device());
  TORCH_CHECK_VALUE(window >= 0 && window <= INT32_MAX, "window must not be negative");
  // (before it becomes a number of 32 bits, where a smaller one is zero: none)
  TORCH_CHECK_VALUE(softcap == 0.0 || (softcap >= 1e-20 && softcap <= 1e30), "softcap must be 0 (none) or from 1e-20 to 1e30");
  const int64_t E = q_in.size(0), H = q_in.size(1), N = q_in.size(2), W = q_in.size(3);
  Tensor out;
  if (out_in.has_value()) {
    out = *out_in;
    TORCH_CHECK_VALUE(out.sizes() == q_in.sizes() && out.scalar_type() == q_in.scalar_type() && out.device() == q_in.device() && out.stride(3) == 1,
                      "out must have the query's shape, dtype and device and unit inner stride");
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !out.requires_grad(), "out requires a gradient");
    TORCH_CHECK_VALUE(Places(out).distinct(), "the rows of out overlap");
  } else {
    const at::TensorOptions o = at::TensorOptions().dtype(q_in.scalar_type()).device(q_in.device());
    out = token_major ? at::detail::empty_strided_cuda({E, H, N, W}, {N * H * W, W, H * W, 1}, o) : at::detail::empty_cuda({E, H, N, W}, o);
  }
  if (E == 0 || N == 0) return out;
  const Tensor q = aligned(q_in, 16);
  if (out_in.has_value()) {
    // (the query itself may take the result: a row is read by those that write it, before they do)
    bool same = out.data_ptr() == q.data_ptr();
    for (int i = 0; i < 4; ++i) same = same && (out.size(i) == 1 || out.stride(i) == q.stride(i));
    TORCH_CHECK_VALUE(same || !meet(Places(out), Places(q)), "out and query overlap in part");
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  }
  p.E = (int32_t)E; p.H = (int32_t)H; p.N = (int32_t)N;
  p.dtype = dtype_code(q.scalar_type());
  p.causal = causal;
  p.window = (int32_t)window;
  p.scale = (float)scale;
  p.softcap = (float)softcap;
  p.q = view4(q);
  p.out = view4(out);
  const size_t need = ma_b200_cache_attend_workspace_bytes(&p);
  if (need == 0) raise_for_status(MA_B200_INVALID_ARGUMENT);
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(need);
  raise_for_status(ma_b200_cache_attend(&p, ws.get(), need, c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

PyObject* wrap_or_none(Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(t));
}

}  // namespace

PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "rotary() takes 8 arguments");
  const Tensor q = tensor_of(args[0], "query");
  const optional<Tensor> k = optional_of(args[1], "key"), positions = optional_of(args[6], "positions");
  const Rotary r = rotary_of(args[2], args[3], args[4], args[5]);
  const bool inverse = PyObject_IsTrue(args[7]) == 1;
  check_python();
  std::pair<Tensor, Tensor> out;
  {
    pybind11::gil_scoped_release no_gil;
    check_rotated(q, k, positions);
    out = rotate_any(q, k.value_or(Tensor()), r, positions, inverse);
  }
  PyObject* result = PyTuple_New(2);
  if (result == nullptr) throw python_error();
  PyTuple_SET_ITEM(result, 0, wrap_or_none(out.first));
  PyTuple_SET_ITEM(result, 1, wrap_or_none(out.second));
  return result;
  END_HANDLE_TH_ERRORS
}

PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 14, "append() takes 14 arguments");
  const Cache cache{tensor_of(args[0], "cache.k"), tensor_of(args[1], "cache.v"), tensor_of(args[2], "cache.k_scale"), tensor_of(args[3], "cache.v_scale")};
  const Tensor &k = tensor_of(args[4], "key"), &v = tensor_of(args[5], "value"), &table = tensor_of(args[6], "page_table"),
               &lengths = tensor_of(args[7], "lengths");
  const optional<Tensor> counts = optional_of(args[8], "counts"), query = optional_of(args[9], "query");
  optional<Rotary> rotary;
  if (args[10] != Py_None) rotary = rotary_of(args[10], args[11], args[12], args[13]);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = append(cache, k, v, table, lengths, counts, query, rotary.has_value() ? &*rotary : nullptr);
  }
  return wrap_or_none(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* py_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 14, "attend() takes 14 arguments");
  const Tensor& q = tensor_of(args[0], "query");
  const Cache cache{tensor_of(args[1], "cache.k"), tensor_of(args[2], "cache.v"), tensor_of(args[3], "cache.k_scale"), tensor_of(args[4], "cache.v_scale")};
  const Tensor &table = tensor_of(args[5], "page_table"), &lengths = tensor_of(args[6], "lengths");
  const optional<Tensor> counts = optional_of(args[7], "counts"), out_in = optional_of(args[12], "out");
  const bool causal = PyObject_IsTrue(args[8]) == 1, token_major = PyObject_IsTrue(args[13]) == 1;
  const double scale = PyFloat_AsDouble(args[9]), softcap = PyFloat_AsDouble(args[10]);
  const int64_t window = PyLong_AsLongLong(args[11]);
  check_python();
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = attend(q, cache, table, lengths, counts, causal, scale, softcap, window, out_in, token_major);
  }
  return wrap_or_none(std::move(out));
  END_HANDLE_TH_ERRORS
}

}  // namespace ma_torch
