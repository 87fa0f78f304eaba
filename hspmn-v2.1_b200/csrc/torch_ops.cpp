// torch operators of the paged K/V cache: argument checks, outputs and workspace
// from PyTorch's allocator, and the call into the C ABI on the caller's current
// stream. They are in C++ because a decode step calls them for microseconds of
// GPU work each (through Python checks and ctypes a call took 28 to 37 us of host
// time). Registered as torch.ops.hspmn.* for CUDA tensors, for traced calls, and as
// functions of the Python module libhspmn_torch, which eager calls use: the
// dispatcher's boxing of the arguments costs 1 us more (6.9 and 7.9 us a call of
// the attention of one token).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <initializer_list>
#include <tuple>

#include "hspmn_sm100.h"

namespace {

using at::Tensor;

struct Range {
  explicit Range(const char* name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
};

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == HSPMN_OK, what, " failed: ", hspmn_strerror(rc), " (status ", rc, ")");
}

c10::Device require_cuda(std::initializer_list<const Tensor*> tensors) {
  const c10::Device dev = (*tensors.begin())->device();
  for (const Tensor* t : tensors) {
    TORCH_CHECK(t->is_cuda(), "hspmn: the sm_100a kernels need CUDA tensors (there is no CPU path); got a tensor on ",
                t->device());
    TORCH_CHECK(t->device() == dev, "hspmn: tensors on different devices (", dev, " vs ", t->device(), ")");
  }
  return dev;
}

void no_grad_needed(const char* name, std::initializer_list<const Tensor*> tensors) {
  const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    TORCH_CHECK(!(backward && t->requires_grad()), name,
                ": has no backward; call it under torch.no_grad() or detach its inputs");
    TORCH_CHECK(!(forward && t->_fw_grad(0).defined()), name, ": has no forward-mode derivative; give it the primals");
  }
}

int dtype_code(const char* name, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HSPMN_F32;
    case at::kHalf: return HSPMN_F16;
    case at::kBFloat16: return HSPMN_BF16;
    default: TORCH_CHECK_TYPE(false, name, ": unsupported dtype ", t, "; expected float32, float16 or bfloat16");
  }
}

// Tells autograd that a tensor has been written in place: a backward that saved
// what it held before then raises instead of using what it holds now. (No kernel of
// the dispatcher does it: eager calls do not pass there.) Inference tensors have no
// version.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// at::empty without the dispatcher's part of its cost.
Tensor empty_on(c10::Device dev, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, dev, std::nullopt);
}

// n elements of `whole`'s memory from element `at` on, as a tensor of its own
// (0.4 us less than an allocation).
Tensor part_of(const Tensor& whole, int64_t at, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  return t;
}

// A 1-D int32 / int64 argument of n elements, contiguous.
Tensor vector_arg(const char* name, const char* what, const Tensor& t, at::ScalarType dtype, int64_t n) {
  TORCH_CHECK_VALUE(t.scalar_type() == dtype && t.dim() == 1 && (n < 0 || t.size(0) == n), name, ": ", what, " must be ",
                    dtype, " [", n < 0 ? "*" : std::to_string(n), "], got ", t.scalar_type(), " ", t.sizes());
  return t.is_contiguous() ? t : t.contiguous();
}

// [N,H,hd] operand with dense head rows and 16-byte strides and base; copied where it is not.
Tensor rows_arg(const Tensor& t) {
  const int64_t es = t.element_size(), a = t.stride(0), b = t.stride(1);
  const bool ok = (t.size(2) <= 1 || t.stride(2) == 1) && a > 0 && b > 0 && (a * es) % 16 == 0 && (b * es) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Whether a [L,hd] table can be read as it lies: dense rows, 16-byte stride and base.
// (cos and sin share one stride, that of a table of one row included.)
bool table_ok(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) >= t.size(1) && (t.stride(0) * t.element_size()) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

void check_caches(const char* name, const Tensor& k, const Tensor& v, at::ScalarType dtype, int64_t heads, int64_t hd) {
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.size(2) == heads && k.size(3) == hd, name,
                    ": caches must both be [num_pages, page_size, ", heads, ", ", hd, "], got ", k.sizes(), " and ",
                    v.sizes());
  TORCH_CHECK_TYPE(k.scalar_type() == dtype && v.scalar_type() == dtype, name, ": the caches (", k.scalar_type(), ", ",
                   v.scalar_type(), ") must have the operands' dtype ", dtype);
  TORCH_CHECK_VALUE(hd <= 1 || (k.stride(3) == 1 && v.stride(3) == 1), name,
                    ": the caches' last dimension must be contiguous (they are used in place)");
}

// kShare: the outputs of the requests, and those of the tokens, lie in one
// allocation each (operators that are traced must give tensors that share nothing).
template <bool kShare>
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> paged_slots_(const Tensor& block_table, const Tensor& seq_lens_,
                                                                const Tensor& new_lens_, const Tensor& free_pages_,
                                                                int64_t page_size, int64_t num_tokens) {
  constexpr const char* name = "paged_slots_";
  const c10::Device dev = require_cuda({&block_table, &seq_lens_, &new_lens_, &free_pages_});
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2, name,
                    ": block_table must be int32 [R,P]");
  const int64_t R = block_table.size(0), P = block_table.size(1);
  const Tensor seq_lens = vector_arg(name, "seq_lens", seq_lens_, at::kInt, R);
  const Tensor new_lens = vector_arg(name, "new_lens", new_lens_, at::kInt, R);
  const Tensor free_pages = vector_arg(name, "free_pages", free_pages_, at::kInt, -1);
  TORCH_CHECK_VALUE((P <= 1 || block_table.stride(1) == 1) && (R <= 1 || block_table.stride(0) >= P), name,
                    ": block_table is written in place: its rows must be dense and must not overlap");
  TORCH_CHECK_VALUE(num_tokens >= 0, name, ": num_tokens=", num_tokens);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor cu, kv_lens, taken, positions, slots;
  if constexpr (kShare) {
    const int64_t r4 = (R + 4) / 4 * 4, n2 = (num_tokens + 1) / 2 * 2;  // 16-byte boundaries
    const Tensor requests = empty_on(dev, {2 * r4 + 1}, at::kInt), tokens = empty_on(dev, {n2 + num_tokens}, at::kLong);
    cu = part_of(requests, 0, R + 1), kv_lens = part_of(requests, r4, R), taken = part_of(requests, 2 * r4, 1);
    positions = part_of(tokens, 0, num_tokens), slots = part_of(tokens, n2, num_tokens);
  } else {
    cu = empty_on(dev, {R + 1}, at::kInt), kv_lens = empty_on(dev, {R}, at::kInt), taken = empty_on(dev, {1}, at::kInt);
    positions = empty_on(dev, {num_tokens}, at::kLong), slots = empty_on(dev, {num_tokens}, at::kLong);
  }
  const Range range("hspmn::paged_slots");
  check_status(
      hspmn_paged_slots(block_table.data_ptr<int32_t>(), R > 1 ? block_table.stride(0) : P,
                        seq_lens.const_data_ptr<int32_t>(), new_lens.const_data_ptr<int32_t>(),
                        free_pages.const_data_ptr<int32_t>(), free_pages.size(0), R, P, page_size, num_tokens,
                        cu.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(), positions.data_ptr<int64_t>(),
                        slots.data_ptr<int64_t>(), taken.data_ptr<int32_t>(),
                        c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
      "hspmn_paged_slots");
  written(block_table);
  return {cu, kv_lens, positions, slots, taken};
}

void rope_paged_write_(const Tensor& k_, const Tensor& v_, const std::optional<Tensor>& cos_,
                       const std::optional<Tensor>& sin_, const Tensor& positions_, const Tensor& slots_,
                       const Tensor& k_cache, const Tensor& v_cache) {
  constexpr const char* name = "rope_paged_write_";
  TORCH_CHECK_VALUE(cos_.has_value() == sin_.has_value(), name, ": cos and sin must both be given or both be None");
  const c10::Device dev = require_cuda({&k_, &v_, &positions_, &slots_, &k_cache, &v_cache});
  no_grad_needed(name, {&k_, &v_, &k_cache, &v_cache});
  TORCH_CHECK_VALUE(k_.dim() == 3 && k_.sizes() == v_.sizes(), name, ": k and v must both be [N,Hkv,hd], got ", k_.sizes(),
                    " and ", v_.sizes());
  const int64_t n = k_.size(0), heads = k_.size(1), hd = k_.size(2);
  TORCH_CHECK_TYPE(k_.scalar_type() == v_.scalar_type(), name, ": k (", k_.scalar_type(), ") and v (", v_.scalar_type(),
                   ") must share one dtype");
  const int code = dtype_code(name, k_.scalar_type());
  check_caches(name, k_cache, v_cache, k_.scalar_type(), heads, hd);
  const Tensor positions = vector_arg(name, "positions", positions_, at::kLong, n);
  const Tensor slots = vector_arg(name, "slots", slots_, at::kLong, n);
  Tensor cos, sin;
  int tab_code = code;
  if (cos_.has_value()) {
    cos = *cos_, sin = *sin_;
    require_cuda({&k_, &cos, &sin});
    no_grad_needed(name, {&cos, &sin});
    TORCH_CHECK_TYPE(cos.scalar_type() == sin.scalar_type() &&
                         (cos.scalar_type() == k_.scalar_type() || cos.scalar_type() == at::kFloat),
                     name, ": cos/sin must both have k's dtype or float32");
    TORCH_CHECK_VALUE(cos.dim() >= 2 && cos.size(-1) == hd && sin.dim() >= 2 && sin.size(-1) == hd &&
                          cos.numel() == sin.numel(),
                      name, ": cos/sin must both be [L,", hd, "], got ", cos.sizes(), " and ", sin.sizes());
    if (cos.dim() != 2) cos = cos.reshape({-1, hd});
    if (sin.dim() != 2) sin = sin.reshape({-1, hd});
    if (!table_ok(cos) || !table_ok(sin) || cos.stride(0) != sin.stride(0))
      cos = cos.clone(at::MemoryFormat::Contiguous), sin = sin.clone(at::MemoryFormat::Contiguous);
    tab_code = dtype_code(name, cos.scalar_type());
  }
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor k = rows_arg(k_), v = rows_arg(v_);
  const Range range("hspmn::rope_paged_write");
  check_status(
      hspmn_rope_paged_write(k.const_data_ptr(), k.stride(0), k.stride(1), v.const_data_ptr(), v.stride(0), v.stride(1),
                             cos.defined() ? cos.const_data_ptr() : nullptr,
                             sin.defined() ? sin.const_data_ptr() : nullptr, cos.defined() ? cos.stride(0) : 0,
                             cos.defined() ? cos.size(0) : 0, tab_code, positions.const_data_ptr<int64_t>(),
                             slots.const_data_ptr<int64_t>(), k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1),
                             k_cache.stride(2), v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1),
                             v_cache.stride(2), n, heads, hd, k_cache.size(0), k_cache.size(1), code,
                             c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
      "hspmn_rope_paged_write");
  written(k_cache);
  written(v_cache);
}

Tensor sqdk_paged_fwd(const Tensor& q_, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table_,
                      const Tensor& kv_lens_, const Tensor& cu_q_, const Tensor& positions_, double sm_scale,
                      int64_t max_q) {
  constexpr const char* name = "sqdk_paged_fwd";
  const c10::Device dev = require_cuda({&q_, &k_cache, &v_cache, &block_table_, &kv_lens_, &cu_q_, &positions_});
  no_grad_needed(name, {&q_, &k_cache, &v_cache});
  TORCH_CHECK_VALUE(q_.dim() == 3, name, ": q must be [N,H,hd], got ", q_.sizes());
  const int64_t n = q_.size(0), H = q_.size(1), hd = q_.size(2);
  TORCH_CHECK_TYPE(q_.scalar_type() == at::kBFloat16 || q_.scalar_type() == at::kHalf, name, ": q dtype ",
                   q_.scalar_type(), " unsupported (bf16 or f16)");
  TORCH_CHECK_VALUE(k_cache.dim() == 4, name, ": caches must be [num_pages, page_size, Hkv, hd], got ", k_cache.sizes());
  const int64_t Hkv = k_cache.size(2);
  check_caches(name, k_cache, v_cache, q_.scalar_type(), Hkv, hd);
  TORCH_CHECK_VALUE(Hkv > 0 && H % Hkv == 0, name, ": num_heads ", H, " is not a multiple of num_kv_heads ", Hkv);
  TORCH_CHECK_VALUE(block_table_.scalar_type() == at::kInt && block_table_.dim() == 2, name,
                    ": block_table must be int32 [R,P], got ", block_table_.scalar_type(), " ", block_table_.sizes());
  const int64_t R = block_table_.size(0), P = block_table_.size(1);
  const Tensor block_table = (P <= 1 || block_table_.stride(1) == 1) && (R <= 1 || block_table_.stride(0) >= P)
                                 ? block_table_
                                 : block_table_.contiguous();
  const Tensor kv_lens = vector_arg(name, "kv_lens", kv_lens_, at::kInt, R);
  const Tensor cu_q = vector_arg(name, "cu_q", cu_q_, at::kInt, R + 1);
  const Tensor positions = vector_arg(name, "positions", positions_, at::kLong, n);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor q = rows_arg(q_);
  Tensor o = empty_on(dev, {n, H, hd}, q.scalar_type());
  if (n == 0) return o;
  const int64_t bytes = hspmn_sqdk_paged_workspace_size(n, H, Hkv, hd, max_q);
  TORCH_CHECK(bytes >= 0, "hspmn_sqdk_paged_workspace_size: device query failed");
  Tensor ws = empty_on(dev, {bytes}, at::kByte);
  const Range range("hspmn::sqdk_paged_fwd");
  check_status(
      hspmn_sqdk_paged_fwd(q.const_data_ptr(), q.stride(0), q.stride(1), k_cache.const_data_ptr(), k_cache.stride(0),
                           k_cache.stride(1), k_cache.stride(2), v_cache.const_data_ptr(), v_cache.stride(0),
                           v_cache.stride(1), v_cache.stride(2), block_table.const_data_ptr<int32_t>(),
                           R > 1 ? block_table.stride(0) : P, kv_lens.const_data_ptr<int32_t>(),
                           cu_q.const_data_ptr<int32_t>(), positions.const_data_ptr<int64_t>(), o.data_ptr(), H * hd, hd,
                           n, R, P, k_cache.size(0), k_cache.size(1), H, Hkv, hd,
                           q.scalar_type() == at::kBFloat16 ? HSPMN_BF16 : HSPMN_F16, static_cast<float>(sm_scale),
                           max_q, ws.data_ptr(), static_cast<size_t>(bytes),
                           c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
      "hspmn_sqdk_paged_fwd");
  return o;
}

}  // namespace

// (the schemas are defined by the Python package, whether this library is loaded or not)
TORCH_LIBRARY_IMPL(hspmn, CUDA, m) {
  m.impl("paged_slots_", paged_slots_<false>);
  m.impl("rope_paged_write_", rope_paged_write_);
  m.impl("sqdk_paged_fwd", sqdk_paged_fwd);
}

// What this file was built for (found in the built file: a library that was built for
// another PyTorch must not be loaded to ask it).
extern "C" {
extern const char hspmn_torch_build_id[];
__attribute__((visibility("default"), used)) const char hspmn_torch_build_id[] = HSPMN_TORCH_BUILD_ID;
}

PYBIND11_MODULE(libhspmn_torch, m) {
  m.def("paged_slots_", paged_slots_<true>);
  m.def("rope_paged_write_", rope_paged_write_);
  m.def("sqdk_paged_fwd", sqdk_paged_fwd);
}
