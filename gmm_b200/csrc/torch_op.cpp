// torch_op.cpp -- the `hopper_gmm_fwd::gmm` PyTorch operator over the C ABI.
//
// Drop-in for the reference's op registration (reference csrc/bindings.cc:13-19)
// and host entry point (reference csrc/hopper_gmm_forward.cu:372-486): same
// schema, same argument checks and messages, CUDA dispatch key only.  The
// tensor work is delegated to libgmm_sm100.so through include/gmm_sm100.h.
//
// Differences from the reference host layer, all deliberate:
//   * D is allocated uninitialised (at::empty): sum(batch_sizes) == T means
//     every row is written by exactly one expert, so the reference's memset
//     (hopper_gmm_forward.cu:440) is dead work.
//   * No per-expert tensor views or problem-table upload: the C ABI turns the
//     host batch_sizes into a tile schedule passed with the kernel launch.
//   * fp32 with trans_b=True multiplies by B[e]^T (B given as [E, dim_out, dim]),
//     as documented for trans_b; the reference transposed such a B a second
//     time (hopper_gmm_forward.cu:442-446).
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include "gmm_sm100.h"
#include "hopper_gmm_forward.h"

namespace hpc_ops_hopper {

// Declared in include/hopper_gmm_forward.h with the reference's signature
// (reference csrc/hopper_gmm_forward.h:23-25).
at::Tensor hopper_gmm_forward(at::Tensor A, at::Tensor B, at::Tensor batch_sizes, bool transb) {
  TORCH_CHECK(A.is_cuda() && A.is_contiguous(), "A must be a contiguous CUDA tensor");
  TORCH_CHECK(B.is_cuda() && B.is_contiguous(), "B must be a contiguous CUDA tensor");
  TORCH_CHECK(A.dim() == 2, "A must be 2D");
  TORCH_CHECK(B.dim() == 3, "B must be 3D [num_experts, dim, dim_out] (forward-only build)");
  TORCH_CHECK(batch_sizes.is_cpu() && batch_sizes.dim() == 1 &&
                  batch_sizes.scalar_type() == at::kLong,
              "batch_sizes must be a 1D CPU int64 tensor");
  TORCH_CHECK(A.scalar_type() == B.scalar_type(), "A and B must have the same dtype");
  TORCH_CHECK(A.get_device() == B.get_device(), "A and B must be on the same device");

  const int device = A.get_device();
  c10::cuda::CUDAGuard guard(device);
  {
    const int rc = gmm_sm100_check_device(device);
    TORCH_CHECK(rc == GMM_OK, "hopper_gmm_forward: ", gmm_sm100_last_error());
  }

  const int64_t num_experts = batch_sizes.size(0);
  const int64_t dim = A.size(1);
  const int64_t dim_out = transb ? B.size(1) : B.size(2);
  TORCH_CHECK(B.size(0) == num_experts, "B.size(0) must equal num_experts (batch_sizes.size(0))");
  TORCH_CHECK((transb ? B.size(2) : B.size(1)) == dim, "B.", (transb ? "size(2)" : "size(1)"),
              " must equal A.size(1) (dim), got ", (transb ? B.size(2) : B.size(1)), " vs ", dim);

  int dtype;
  switch (A.scalar_type()) {
    case at::kFloat: dtype = GMM_DTYPE_F32; break;
    case at::kBFloat16: dtype = GMM_DTYPE_BF16; break;
    case at::kHalf: dtype = GMM_DTYPE_F16; break;
    default: TORCH_CHECK(false, "Unsupported dtype: only FP32 / BF16 / FP16 are supported");
  }

  auto bs = batch_sizes.contiguous();
  const int64_t* bs_ptr = bs.data_ptr<int64_t>();
  at::Tensor D = at::empty({A.size(0), dim_out}, A.options());
  const size_t ws_bytes =
      gmm_sm100_workspace_size(bs_ptr, num_experts, A.size(0), dim, dim_out, dtype, transb ? 1 : 0);
  at::Tensor ws;
  if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, A.options().dtype(at::kByte));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int rc = gmm_sm100_forward(A.data_ptr(), B.data_ptr(), bs_ptr, num_experts, A.size(0), dim,
                                   dim_out, dtype, transb ? 1 : 0, D.data_ptr(),
                                   ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream);
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return D;
}

}  // namespace hpc_ops_hopper

namespace gmm_b200 {

// Fused MoE gate/up projection + SwiGLU: B holds [gate | up] (2*I output
// columns); returns silu(A @ Bgate) * (A @ Bup), [T, I].  No reference
// counterpart (the reference's caller would run two GEMM segments with the
// activation in between).
at::Tensor gmm_swiglu(at::Tensor A, at::Tensor B, at::Tensor batch_sizes, bool transb) {
  TORCH_CHECK(A.is_cuda() && A.is_contiguous(), "A must be a contiguous CUDA tensor");
  TORCH_CHECK(B.is_cuda() && B.is_contiguous(), "B must be a contiguous CUDA tensor");
  TORCH_CHECK(A.dim() == 2, "A must be 2D");
  TORCH_CHECK(B.dim() == 3, "B must be 3D [num_experts, dim, 2*inter] (or [num_experts, 2*inter, dim])");
  TORCH_CHECK(batch_sizes.is_cpu() && batch_sizes.dim() == 1 &&
                  batch_sizes.scalar_type() == at::kLong,
              "batch_sizes must be a 1D CPU int64 tensor");
  TORCH_CHECK(A.scalar_type() == B.scalar_type(), "A and B must have the same dtype");
  TORCH_CHECK(A.scalar_type() == at::kBFloat16 || A.scalar_type() == at::kHalf,
              "gmm_swiglu supports bf16 / fp16");
  const int device = A.get_device();
  c10::cuda::CUDAGuard guard(device);
  TORCH_CHECK(gmm_sm100_check_device(device) == GMM_OK, "gmm_swiglu: ", gmm_sm100_last_error());
  const int64_t num_experts = batch_sizes.size(0);
  const int64_t dim = A.size(1);
  const int64_t dim_out = transb ? B.size(1) : B.size(2);
  TORCH_CHECK(B.size(0) == num_experts, "B.size(0) must equal num_experts (batch_sizes.size(0))");
  TORCH_CHECK((transb ? B.size(2) : B.size(1)) == dim, "B's contraction size must equal A.size(1) (dim)");
  TORCH_CHECK(dim_out % 2 == 0, "B must hold gate and up projections of equal width");
  const int dtype = A.scalar_type() == at::kBFloat16 ? GMM_DTYPE_BF16 : GMM_DTYPE_F16;
  auto bs = batch_sizes.contiguous();
  const int64_t* bs_ptr = bs.data_ptr<int64_t>();
  at::Tensor D = at::empty({A.size(0), dim_out / 2}, A.options());
  const size_t ws_bytes =
      gmm_sm100_workspace_size(bs_ptr, num_experts, A.size(0), dim, dim_out, dtype, transb ? 1 : 0);
  at::Tensor ws;
  if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, A.options().dtype(at::kByte));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int rc = gmm_sm100_forward_swiglu(A.data_ptr(), B.data_ptr(), bs_ptr, num_experts, A.size(0),
                                          dim, dim_out, dtype, transb ? 1 : 0, D.data_ptr(),
                                          ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream);
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return D;
}

// An uninitialised tensor on the current device, straight from the caching
// allocator: at::empty dispatches again, which costs a small call as much as
// its launch does.
at::Tensor device_empty(c10::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(),
                                              c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}

// ---------------------------------------------------------------- 8-bit grouped product
int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return GMM_DTYPE_F32;
    case at::kBFloat16: return GMM_DTYPE_BF16;
    case at::kHalf: return GMM_DTYPE_F16;
    default: TORCH_CHECK(false, what, " must be fp32, bf16 or fp16, got ", t);
  }
}

// What the host- and device-sized forms check alike; returns D.
at::Tensor check_int8(const at::Tensor& A, const at::Tensor& a_scale, const at::Tensor& B, const at::Tensor& b_scale,
                      int64_t num_experts, at::ScalarType out_dtype, bool swiglu) {
  TORCH_CHECK(A.is_cuda() && A.is_contiguous(), "A must be a contiguous CUDA tensor");
  TORCH_CHECK(B.is_cuda() && B.is_contiguous(), "B must be a contiguous CUDA tensor");
  TORCH_CHECK(A.scalar_type() == at::kChar && B.scalar_type() == at::kChar, "A and B must be int8");
  TORCH_CHECK(A.dim() == 2, "A must be 2D");
  TORCH_CHECK(B.dim() == 3, "B must be 3D [num_experts, dim_out, dim]");
  TORCH_CHECK(B.size(0) == num_experts, "B.size(0) must equal num_experts (batch_sizes.size(0))");
  TORCH_CHECK(B.size(2) == A.size(1), "B.size(2) must equal A.size(1) (dim), got ", B.size(2), " vs ", A.size(1));
  TORCH_CHECK(a_scale.is_cuda() && a_scale.is_contiguous() && a_scale.scalar_type() == at::kFloat &&
                  a_scale.dim() == 1 && a_scale.size(0) == A.size(0),
              "a_scale must be a contiguous CUDA fp32 tensor [num_tokens]");
  TORCH_CHECK(b_scale.is_cuda() && b_scale.is_contiguous() && b_scale.scalar_type() == at::kFloat &&
                  b_scale.dim() == 2 && b_scale.size(0) == B.size(0) && b_scale.size(1) == B.size(1),
              "b_scale must be a contiguous CUDA fp32 tensor [num_experts, dim_out]");
  TORCH_CHECK(A.get_device() == B.get_device() && A.get_device() == a_scale.get_device() &&
                  A.get_device() == b_scale.get_device(),
              "A, B and their scales must be on the same device");
  TORCH_CHECK(gmm_sm100_check_device(A.get_device()) == GMM_OK, "gmm_int8: ", gmm_sm100_last_error());
  dtype_code(out_dtype, "out_dtype");
  if (swiglu) {
    TORCH_CHECK(out_dtype != at::kFloat, "gmm_int8 with swiglu gives bf16 / fp16");
    TORCH_CHECK(B.size(1) % 2 == 0, "B must hold gate and up projections of equal width");
  }
  return device_empty({A.size(0), swiglu ? B.size(1) / 2 : B.size(1)}, out_dtype);
}

at::Tensor gmm_int8(const at::Tensor& A, const at::Tensor& a_scale, const at::Tensor& B, const at::Tensor& b_scale,
                    const at::Tensor& batch_sizes, at::ScalarType out_dtype, bool swiglu) {
  TORCH_CHECK(batch_sizes.is_cpu() && batch_sizes.dim() == 1 && batch_sizes.scalar_type() == at::kLong,
              "batch_sizes must be a 1D CPU int64 tensor");
  const c10::cuda::OptionalCUDAGuard guard(A.is_cuda() ? std::optional<c10::Device>(A.device()) : std::nullopt);
  at::Tensor D = check_int8(A, a_scale, B, b_scale, batch_sizes.size(0), out_dtype, swiglu);
  auto bs = batch_sizes.contiguous();
  const int64_t* bs_ptr = bs.data_ptr<int64_t>();
  const int64_t E = bs.size(0);
  size_t ws_bytes = 0;
  at::Tensor ws;
  if (E > 1024) {  // only a larger table needs one
    ws_bytes = gmm_sm100_int8_workspace_size(bs_ptr, E, A.size(0), A.size(1), B.size(1));
    if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, A.options().dtype(at::kByte));
  }
  const int rc = gmm_sm100_forward_int8(
      A.data_ptr<int8_t>(), a_scale.data_ptr<float>(), B.data_ptr<int8_t>(), b_scale.data_ptr<float>(), bs_ptr, E,
      A.size(0), A.size(1), B.size(1), dtype_code(out_dtype, "out_dtype"), swiglu ? 1 : 0, D.data_ptr(),
      ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, c10::cuda::getCurrentCUDAStream(A.get_device()).stream());
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return D;
}

at::Tensor gmm_int8_dev(const at::Tensor& A, const at::Tensor& a_scale, const at::Tensor& B,
                        const at::Tensor& b_scale, const at::Tensor& batch_sizes, at::ScalarType out_dtype,
                        bool swiglu) {
  TORCH_CHECK(batch_sizes.is_cuda() && batch_sizes.dim() == 1 && batch_sizes.scalar_type() == at::kInt &&
                  batch_sizes.is_contiguous(),
              "batch_sizes must be a contiguous 1D CUDA int32 tensor");
  const c10::cuda::OptionalCUDAGuard guard(A.is_cuda() ? std::optional<c10::Device>(A.device()) : std::nullopt);
  at::Tensor D = check_int8(A, a_scale, B, b_scale, batch_sizes.size(0), out_dtype, swiglu);
  TORCH_CHECK(batch_sizes.get_device() == A.get_device(), "batch_sizes must be on A's device");
  const int rc = gmm_sm100_forward_int8_dev(
      A.data_ptr<int8_t>(), a_scale.data_ptr<float>(), B.data_ptr<int8_t>(), b_scale.data_ptr<float>(),
      batch_sizes.data_ptr<int>(), batch_sizes.size(0), A.size(0), A.size(1), B.size(1),
      dtype_code(out_dtype, "out_dtype"), swiglu ? 1 : 0, D.data_ptr(),
      c10::cuda::getCurrentCUDAStream(A.get_device()).stream());
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return D;
}

std::tuple<at::Tensor, at::Tensor> quantize_rows(const at::Tensor& x, const std::optional<at::Tensor>& dst_pos,
                                                 int64_t out_rows) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a 2D CUDA tensor");
  const int dtype = dtype_code(x.scalar_type(), "x");
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(gmm_sm100_check_device(x.get_device()) == GMM_OK, "quantize_rows: ", gmm_sm100_last_error());
  const at::Tensor rows = x.contiguous();
  int64_t k = 1;
  at::Tensor pos;
  if (dst_pos) {
    TORCH_CHECK(dst_pos->is_cuda() && dst_pos->get_device() == x.get_device() && dst_pos->dim() == 2 &&
                    dst_pos->scalar_type() == at::kInt && dst_pos->size(0) == x.size(0),
                "dst_pos must be a 2D int32 tensor [num_rows, k] on x's device");
    pos = dst_pos->contiguous();
    k = pos.size(1);
  }
  TORCH_CHECK(out_rows >= 0, "out_rows must not be negative");
  at::Tensor q = device_empty({out_rows, (x.size(1) + 15) / 16 * 16}, at::kChar);
  at::Tensor scale = device_empty({out_rows}, at::kFloat);
  const int rc = gmm_sm100_quantize_rows(rows.data_ptr(), dtype, x.size(0), x.size(1),
                                         dst_pos ? pos.data_ptr<int>() : nullptr, static_cast<int>(std::min<int64_t>(k, 1 << 20)),
                                         out_rows, q.data_ptr<int8_t>(), scale.data_ptr<float>(),
                                         c10::cuda::getCurrentCUDAStream(x.get_device()).stream());
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return {q, scale};
}

// ---------------------------------------------------------------- norms around a block
using OptTensor = std::optional<at::Tensor>;

// The shape rules of the norms: x [..., dim], y alike, parameters [dim], gate
// [dim], [..., 1] or [..., dim].
struct NormArgs {
  int64_t rows = 0, dim = 0;
  int dtype = 0, weight_dtype = 0, gate_dtype = 0, gate_mode = GMM_GATE_MODE_NONE;
};

NormArgs check_norm(const OptTensor& y, const at::Tensor& x, const OptTensor& weight, const OptTensor& gate,
                    const OptTensor& next_weight) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1, "the rows must be a CUDA tensor [..., dim]");
  NormArgs n;
  n.dim = x.size(-1);
  n.rows = n.dim ? x.numel() / n.dim : 0;
  n.dtype = dtype_code(x.scalar_type(), "the rows");
  n.weight_dtype = n.gate_dtype = n.dtype;
  auto same_device = [&](const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == x.get_device(), what, " must be on the rows' device");
  };
  auto param_type = [&](const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, what,
                " must have the rows' dtype or be fp32");
    return dtype_code(t.scalar_type(), what);
  };
  if (y) {
    same_device(*y, "y");
    TORCH_CHECK(y->sizes() == x.sizes() && y->scalar_type() == x.scalar_type(),
                "y and residual must have the same shape and dtype");
    TORCH_CHECK(weight.has_value(), "a post-norm needs its weight");
  }
  TORCH_CHECK(y || next_weight, "nothing to compute: neither a block output nor a pre-norm weight");
  for (const OptTensor* w : {&weight, &next_weight}) {
    if (!w->has_value()) continue;
    same_device(**w, "a weight");
    TORCH_CHECK((*w)->dim() == 1 && (*w)->size(0) == n.dim, "a norm weight must have shape [dim] = [", n.dim, "]");
    n.weight_dtype = param_type(**w, "a norm weight");
  }
  if (weight && next_weight)
    TORCH_CHECK(weight->scalar_type() == next_weight->scalar_type(), "weight and next_weight must have one dtype");
  if (gate) {
    TORCH_CHECK(y.has_value(), "a gate needs a block output");
    same_device(*gate, "gate");
    n.gate_dtype = param_type(*gate, "gate");
    auto token = x.sizes().vec();
    token.back() = 1;
    if (gate->sizes() == x.sizes() && x.dim() > 1) n.gate_mode = GMM_GATE_MODE_FULL;
    else if (gate->dim() == 1 && gate->size(0) == n.dim) n.gate_mode = GMM_GATE_MODE_CHANNEL;
    else if (gate->sizes() == c10::IntArrayRef(token)) n.gate_mode = GMM_GATE_MODE_TOKEN;
    else TORCH_CHECK(false, "gate must have shape [dim], [..., 1] or [..., dim], got ", gate->sizes());
  }
  TORCH_CHECK(gmm_sm100_check_device(x.get_device()) == GMM_OK, "post_norm: ", gmm_sm100_last_error());
  return n;
}

void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
OptTensor dense(const OptTensor& t) { return t ? OptTensor(t->contiguous()) : t; }

// (x_new, h, stats): stats keeps r(y) and r(x_new) of every row, [2, rows];
// what was not asked for is an empty tensor.
std::tuple<at::Tensor, at::Tensor, at::Tensor> post_norm(const OptTensor& y_, const at::Tensor& x_,
                                                         const OptTensor& weight_, const OptTensor& gate_,
                                                         const OptTensor& next_weight_, int64_t gate_act,
                                                         double residual_scale, double eps, double weight_offset,
                                                         bool keep) {
  const NormArgs n = check_norm(y_, x_, weight_, gate_, next_weight_);
  const c10::cuda::CUDAGuard guard(x_.device());
  const OptTensor y = dense(y_), weight = dense(weight_), gate = dense(gate_), next_weight = dense(next_weight_);
  const at::Tensor x = x_.contiguous();
  const at::ScalarType type = x.scalar_type();
  at::Tensor x_new = y ? device_empty(x.sizes(), type) : device_empty({0}, type);
  at::Tensor h = next_weight ? device_empty(x.sizes(), type) : device_empty({0}, type);
  at::Tensor stats = keep ? device_empty({2, n.rows}, at::kFloat) : device_empty({0}, at::kFloat);
  float* ry = keep ? stats.data_ptr<float>() : nullptr;
  const int rc = gmm_sm100_post_norm(
      ptr(y), x.data_ptr(), ptr(weight), ptr(gate), ptr(next_weight), n.rows, n.dim, n.dtype, n.weight_dtype,
      n.gate_dtype, n.gate_mode, static_cast<int>(gate_act), static_cast<float>(residual_scale),
      static_cast<float>(eps), static_cast<float>(weight_offset), y ? x_new.data_ptr() : nullptr,
      next_weight ? h.data_ptr() : nullptr, ry, ry ? ry + n.rows : nullptr,
      c10::cuda::getCurrentCUDAStream(x.get_device()).stream());
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return {x_new, h, stats};
}

// (dy, dx, dweight, dgate, dnext_weight); empty where there is nothing to differentiate.
std::vector<at::Tensor> post_norm_backward(const OptTensor& y_, const at::Tensor& x_, const OptTensor& weight_,
                                           const OptTensor& gate_, const OptTensor& next_weight_,
                                           const at::Tensor& stats, const OptTensor& dx_new_, const OptTensor& dh_,
                                           int64_t gate_act, double residual_scale, double weight_offset) {
  const NormArgs n = check_norm(y_, x_, weight_, gate_, next_weight_);
  const c10::cuda::CUDAGuard guard(x_.device());
  TORCH_CHECK(dx_new_ || dh_, "post_norm_backward needs the gradient of x_new or of h");
  for (const OptTensor* g : {&dx_new_, &dh_})
    if (g->has_value())
      TORCH_CHECK((*g)->is_cuda() && (*g)->get_device() == x_.get_device() && (*g)->sizes() == x_.sizes() &&
                      (*g)->scalar_type() == x_.scalar_type(),
                  "the outputs' gradients must have the rows' shape, dtype and device");
  TORCH_CHECK(!dh_ || next_weight_, "a gradient of h needs next_weight");
  TORCH_CHECK(stats.is_cuda() && stats.get_device() == x_.get_device() && stats.is_contiguous() &&
                  stats.scalar_type() == at::kFloat && stats.numel() == 2 * n.rows,
              "stats must be the forward pass's");
  const OptTensor y = dense(y_), weight = dense(weight_), gate = dense(gate_), next_weight = dense(next_weight_),
                  dx_new = dense(dx_new_), dh = dense(dh_);
  const at::Tensor x = x_.contiguous();
  const at::ScalarType type = x.scalar_type();
  auto like = [&](const OptTensor& t, bool wanted = true) {
    return wanted && t ? device_empty(t->sizes(), t->scalar_type()) : device_empty({0}, type);
  };
  at::Tensor dx = device_empty(x.sizes(), type), dy = like(y), dw = like(weight, y.has_value()), dg = like(gate);
  // without dh the next norm's weight gets no gradient
  at::Tensor dv = next_weight && !dh ? at::zeros_like(*next_weight) : like(next_weight);
  const size_t ws_bytes = gmm_sm100_post_norm_backward_workspace_size(n.rows, n.dim);
  at::Tensor ws = device_empty({static_cast<int64_t>(ws_bytes)}, at::kByte);
  const float* ry = stats.data_ptr<float>();
  const int rc = gmm_sm100_post_norm_backward(
      ptr(y), x.data_ptr(), ptr(weight), ptr(gate), ptr(next_weight), ry, ry + n.rows, ptr(dx_new), ptr(dh), n.rows, n.dim, n.dtype, n.weight_dtype,
      n.gate_dtype, n.gate_mode, static_cast<int>(gate_act), static_cast<float>(residual_scale),
      static_cast<float>(weight_offset), y ? dy.data_ptr() : nullptr, dx.data_ptr(), y ? dw.data_ptr() : nullptr,
      gate ? dg.data_ptr() : nullptr, dh ? dv.data_ptr() : nullptr, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
      c10::cuda::getCurrentCUDAStream(x.get_device()).stream());
  TORCH_CHECK(rc == GMM_OK, gmm_sm100_last_error());
  return {dy, dx, dw, dg, dv};
}

// The operators below autograd, through the dispatcher (so that fake tensors work too).
template <typename F>
c10::TypedOperatorHandle<F> typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
const auto& post_norm_op() {
  static const auto op = typed_op<decltype(post_norm)>("hopper_gmm_fwd::post_norm");
  return op;
}
const auto& post_norm_backward_op() {
  static const auto op = typed_op<decltype(post_norm_backward)>("hopper_gmm_fwd::post_norm_backward");
  return op;
}

// The norms have no forward-mode derivative: a dual tensor's tangent would be dropped without a word.
void refuse_forward_gradients(std::initializer_list<const at::Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                "post_norm has no forward-mode derivative (torch.func.jvp, torch.autograd.forward_ad)");
}
const at::Tensor& or_undefined(const OptTensor& t) {
  static const at::Tensor none;
  return t ? *t : none;
}

// A leaf that an eager graph still holds accumulates on that graph's stream. The legacy stream takes no event of a
// captured one, and autograd meets that error on a thread where it ends the process: refused while it is an exception.
void check_captured_leaves(const torch::autograd::variable_list& inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const at::Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = accumulator ? accumulator->stream() : std::nullopt;
    TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(t.get_device()),
                "post_norm: a graph made on the default stream still holds an input of this captured backward pass; "
                "delete its outputs before the capture");
  }
}

// Gradients of post_norm: one node, whose backward is post_norm_backward.
class PostNormGrad : public torch::autograd::Function<PostNormGrad> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const OptTensor& y,
                                                const at::Tensor& x, const OptTensor& weight, const OptTensor& gate,
                                                const OptTensor& next_weight, int64_t gate_act, double residual_scale,
                                                double eps, double weight_offset) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [x_new, h, stats] =
        post_norm_op().call(y, x, weight, gate, next_weight, gate_act, residual_scale, eps, weight_offset, true);
    ctx->save_for_backward({y.value_or(at::Tensor()), x, weight.value_or(at::Tensor()), gate.value_or(at::Tensor()),
                            next_weight.value_or(at::Tensor()), stats});
    ctx->saved_data["gate_act"] = gate_act;
    ctx->saved_data["residual_scale"] = residual_scale;
    ctx->saved_data["weight_offset"] = weight_offset;
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);
    return {x_new, h, stats};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(9);
    const auto saved = ctx->get_saved_variables();
    auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const OptTensor y = opt(saved[0]), next_weight = opt(saved[4]);
    const OptTensor dx_new = y ? opt(grads[0]) : OptTensor(), dh = next_weight ? opt(grads[1]) : OptTensor();
    if (!dx_new && !dh) return out;
    check_captured_leaves(saved);
    const OptTensor weight = opt(saved[2]), gate = opt(saved[3]);
    const auto g = post_norm_backward_op().call(
        y, saved[1], weight, gate, next_weight, saved[5], dx_new, dh, ctx->saved_data["gate_act"].toInt(),
        ctx->saved_data["residual_scale"].toDouble(), ctx->saved_data["weight_offset"].toDouble());
    out[1] = g[1];
    if (y) {
      out[0] = g[0];
      out[2] = g[2];
    }
    if (gate) out[3] = g[3];
    if (next_weight) out[4] = g[4];
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> post_norm_autograd(
    const OptTensor& y, const at::Tensor& x, const OptTensor& weight, const OptTensor& gate,
    const OptTensor& next_weight, int64_t gate_act, double residual_scale, double eps, double weight_offset,
    bool keep) {
  refuse_forward_gradients(
      {&or_undefined(y), &x, &or_undefined(weight), &or_undefined(gate), &or_undefined(next_weight)});
  bool grad = x.requires_grad();
  for (const OptTensor* t : {&y, &weight, &gate, &next_weight}) grad = grad || (t->has_value() && (*t)->requires_grad());
  if (!grad || !at::GradMode::is_enabled()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return post_norm_op().call(y, x, weight, gate, next_weight, gate_act, residual_scale, eps, weight_offset, keep);
  }
  auto out = PostNormGrad::apply(y, x, weight, gate, next_weight, gate_act, residual_scale, eps, weight_offset);
  return {out[0], out[1], out[2]};
}

std::vector<at::Tensor> post_norm_backward_autograd(const OptTensor& y, const at::Tensor& x, const OptTensor& weight,
                                                    const OptTensor& gate, const OptTensor& next_weight,
                                                    const at::Tensor& stats, const OptTensor& dx_new,
                                                    const OptTensor& dh, int64_t gate_act, double residual_scale,
                                                    double weight_offset) {
  // reached with gradients on only under create_graph
  TORCH_CHECK(!at::GradMode::is_enabled(), "post_norm has no second derivative (create_graph=True)");
  refuse_forward_gradients({&or_undefined(y), &x, &or_undefined(weight), &or_undefined(gate),
                            &or_undefined(next_weight), &stats, &or_undefined(dx_new), &or_undefined(dh)});
  at::AutoDispatchBelowADInplaceOrView below;
  return post_norm_backward_op().call(y, x, weight, gate, next_weight, stats, dx_new, dh, gate_act, residual_scale,
                                      weight_offset);
}

}  // namespace gmm_b200

TORCH_LIBRARY(hopper_gmm_fwd, m) {
  m.def("gmm(Tensor A, Tensor B, Tensor batch_sizes, bool trans_b) -> Tensor");
  m.def("gmm_swiglu(Tensor A, Tensor B, Tensor batch_sizes, bool trans_b) -> Tensor");
  m.def("gmm_int8(Tensor A, Tensor a_scale, Tensor B, Tensor b_scale, Tensor batch_sizes, ScalarType out_dtype, "
        "bool swiglu) -> Tensor");
  m.def("gmm_int8_dev(Tensor A, Tensor a_scale, Tensor B, Tensor b_scale, Tensor batch_sizes, "
        "ScalarType out_dtype, bool swiglu) -> Tensor");
  m.def("quantize_rows(Tensor x, Tensor? dst_pos, int out_rows) -> (Tensor, Tensor)");
  m.def("post_norm(Tensor? y, Tensor x, Tensor? weight, Tensor? gate, Tensor? next_weight, int gate_act, "
        "float residual_scale, float eps, float weight_offset, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("post_norm_backward(Tensor? y, Tensor x, Tensor? weight, Tensor? gate, Tensor? next_weight, Tensor stats, "
        "Tensor? dx_new, Tensor? dh, int gate_act, float residual_scale, float weight_offset) "
        "-> Tensor[]");
}

TORCH_LIBRARY_IMPL(hopper_gmm_fwd, CUDA, m) {
  m.impl("gmm", &hpc_ops_hopper::hopper_gmm_forward);
  m.impl("gmm_swiglu", &gmm_b200::gmm_swiglu);
  m.impl("gmm_int8", &gmm_b200::gmm_int8);
  m.impl("gmm_int8_dev", &gmm_b200::gmm_int8_dev);
  m.impl("quantize_rows", &gmm_b200::quantize_rows);
  m.impl("post_norm", &gmm_b200::post_norm);
  m.impl("post_norm_backward", &gmm_b200::post_norm_backward);
}

TORCH_LIBRARY_IMPL(hopper_gmm_fwd, AutogradCUDA, m) {
  m.impl("post_norm", &gmm_b200::post_norm_autograd);
  m.impl("post_norm_backward", &gmm_b200::post_norm_backward_autograd);
}
