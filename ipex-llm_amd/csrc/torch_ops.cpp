// The host path from a torch tensor to a launch: allocation of the result and of the workspace, the current stream
// and the call of the C ABI, in one native call per layer.
//
// What bounds a decode-sized call is the host: a [4096 x 4096] product at one row is 3.8 us of GPU time, and the same
// steps taken in Python (module attributes, torch.empty, torch.cuda.device, current_stream, five ctypes calls) were
// 17 us of the 21 us a LowBitLinear call took.  The module is plain CPython (METH_FASTCALL, no argument parsing by
// keyword).  It holds no state but the addresses of the C ABI functions, which the ctypes binding hands over
// (`bind`), so that both always run the same library.
//
// Functions whose name says "or None" answer None for anything but the plain case (a tensor on another device, a
// dtype they do not know, a weight of another size): the Python code behind them then takes its own way and words
// the error.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/Event.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>

#include "../../include/lowbit_abi.h"

namespace {

using at::Tensor;

struct Api {
    decltype(&lowbit_last_error) last_error = nullptr;
    decltype(&lowbit_blob_bytes) blob_bytes = nullptr;
    decltype(&lowbit_tileable) tileable = nullptr;
    decltype(&lowbit_linear_scratch_bytes) linear_scratch_bytes = nullptr;
    decltype(&lowbit_linear) linear = nullptr;
    decltype(&lowbit_gated_mlp) gated_mlp = nullptr;
    decltype(&lowbit_dequantize_rows) dequantize_rows = nullptr;
    decltype(&lowbit_dequantize) dequantize = nullptr;
    decltype(&lowbit_backward_ws) backward_ws = nullptr;
    decltype(&lowbit_backward_workspace_bytes) backward_workspace_bytes = nullptr;
    decltype(&lowbit_backward_ws_applies) backward_ws_applies = nullptr;
    decltype(&lowbit_experts_workspace_bytes) experts_workspace_bytes = nullptr;
    decltype(&lowbit_experts_forward) experts_forward = nullptr;
    decltype(&lowbit_block_fp8_quantize) block_fp8_quantize = nullptr;
    decltype(&lowbit_block_fp8_quantize_weight) block_fp8_quantize_weight = nullptr;
    decltype(&lowbit_block_fp8_linear) block_fp8_linear = nullptr;
    decltype(&lowbit_block_fp8_linear_workspace_bytes) block_fp8_linear_workspace_bytes = nullptr;
    decltype(&lowbit_block_fp8_backward) block_fp8_backward = nullptr;
    decltype(&lowbit_block_fp8_backward_workspace_bytes) block_fp8_backward_workspace_bytes = nullptr;
    decltype(&lowbit_row_int8_quantize) row_int8_quantize = nullptr;
    decltype(&lowbit_row_int8_linear) row_int8_linear = nullptr;
    decltype(&lowbit_row_int8_linear_workspace_bytes) row_int8_linear_workspace_bytes = nullptr;
    decltype(&lowbit_row_int8_product) row_int8_product = nullptr;
    decltype(&lowbit_row_int8_product_workspace_bytes) row_int8_product_workspace_bytes = nullptr;
    decltype(&lowbit_row_int8_backward) row_int8_backward = nullptr;
    decltype(&lowbit_row_int8_backward_workspace_bytes) row_int8_backward_workspace_bytes = nullptr;
    decltype(&lowbit_row_int8_experts) row_int8_experts = nullptr;
    decltype(&lowbit_row_int8_experts_workspace_bytes) row_int8_experts_workspace_bytes = nullptr;
    decltype(&lowbit_row_int8_moe) row_int8_moe = nullptr;
    decltype(&lowbit_row_int8_moe_workspace_bytes) row_int8_moe_workspace_bytes = nullptr;
    decltype(&lowbit_route) route = nullptr;
    decltype(&lowbit_route_workspace_bytes) route_workspace_bytes = nullptr;
    decltype(&lowbit_route_backward) route_backward = nullptr;
    decltype(&lowbit_route_backward_workspace_bytes) route_backward_workspace_bytes = nullptr;
    decltype(&lowbit_block_fp8_experts) block_fp8_experts = nullptr;
    decltype(&lowbit_block_fp8_experts_workspace_bytes) block_fp8_experts_workspace_bytes = nullptr;
} api;

constexpr size_t WORKSPACE_CAP = (size_t)256 << 20;      // most that a product borrows for split-K partial sums

struct Failed : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char *what) {
    if (rc != 0) throw Failed(std::string(what) + " failed (" + std::to_string(rc) + "): " + api.last_error());
}

int dtype_code(at::ScalarType t) {
    switch (t) {
    case at::kHalf: return LOWBIT_DT_F16;
    case at::kBFloat16: return LOWBIT_DT_BF16;
    case at::kFloat: return LOWBIT_DT_F32;
    default: return -1;
    }
}

void *current_stream(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// a tensor of this module's calls: strided, on the GPU
bool on_gpu(const Tensor &t) { return t.device().is_cuda() && t.layout() == at::kStrided; }

// whether the result has to carry a derivative with respect to t, which no call of this module gives it
bool differentiable(const Tensor &t) {
    return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(/*level=*/0).defined();
}

// w holds the packed [N, K] weight of this format on x's device
bool is_blob(const Tensor &w, const Tensor &x, int qtype, int64_t N, int64_t K) {
    if (w.device() != x.device() || w.layout() != at::kStrided || !w.is_contiguous()) return false;
    const at::ScalarType st = w.scalar_type();
    if (st != at::kByte && !(st == at::kBFloat16 && qtype == LOWBIT_QT_NF4)) return false;
    return (size_t)w.nbytes() == api.blob_bytes(qtype, N * K) && w.nbytes() > 0;
}

// y = x * dequant(w)^T (+ bias), in x's dtype; x contiguous [.., K] with M rows, not empty
Tensor product(const Tensor &x, const Tensor &w, const Tensor &bias, int qtype, int layout, int64_t M, int64_t N, int64_t K,
               at::IntArrayRef shape) {
    c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(shape, x.options());
    const int dt = dtype_code(x.scalar_type());
    // the workspace comes from torch's caching allocator: ordered with the stream, no allocation in the steady state
    const size_t bytes = M <= 16 ? 0 : api.linear_scratch_bytes(qtype, layout, dt, M, N, K, WORKSPACE_CAP);
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    check(api.linear(x.const_data_ptr(), w.const_data_ptr(), bias.defined() ? bias.const_data_ptr() : nullptr, y.data_ptr(), qtype,
                     layout, dt, M, N, K, bytes ? ws.data_ptr() : nullptr, bytes, current_stream(x)), "lowbit_linear");
    return y;
}

// Whether a small batch of float32 rows stays float32 (use_batch_forward of low_bit_linear.py)
bool batch_stays_f32(int qtype, int64_t M, int64_t N, int64_t K) {
    if (M <= 1 || K % 128) return false;
    if (qtype != LOWBIT_QT_SYM_INT4 && qtype != LOWBIT_QT_ASYM_INT4 && qtype != LOWBIT_QT_FP8_E4M3) return false;
    return M <= 48 || (M <= 64 && K % 256 == 0 && N % 64 == 0);
}

int device_layout(int qtype, int64_t N, int64_t K) {
    return api.tileable(qtype, N, K) ? LOWBIT_LAYOUT_TILED : LOWBIT_LAYOUT_GGML;
}

at::DimVector with_last(const Tensor &x, int64_t last) {
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = last;
    return shape;
}

// LowBitLinear at inference on a GPU-resident weight; an undefined tensor when this is not the plain case
Tensor linear(const Tensor &x_in, const Tensor &w, const Tensor &bias, int qtype, int64_t N, bool conver_to_half) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || dtype_code(x_in.scalar_type()) < 0) return {};
    const int64_t K = x_in.size(-1), M = x_in.numel() / K;
    if (!is_blob(w, x_in, qtype, N, K)) return {};
    if (bias.defined() && (bias.scalar_type() != x_in.scalar_type() || bias.device() != x_in.device() || bias.numel() != N || !bias.is_contiguous() ||
                           differentiable(bias))) return {};
    const Tensor x = x_in.is_contiguous() ? x_in : x_in.contiguous();
    const int layout = device_layout(qtype, N, K);
    const auto shape = with_last(x, N);
    if (x.scalar_type() == at::kFloat && conver_to_half && M > 1 && !batch_stays_f32(qtype, M, N, K)) {
        Tensor y = product(x.to(at::kHalf), w, Tensor(), qtype, layout, M, N, K, shape).to(at::kFloat);
        if (bias.defined()) y.add_(bias);
        return y;
    }
    return product(x, w, bias, qtype, layout, M, N, K, shape);
}

// ---- training: the same product below trained parameters
//
// What bounded a small step was the host: a layer's forward and backward took some 110 us of Python, ctypes and the
// interpreter lock taken in autograd's thread, around 20 us of GPU time (77 rows on [1200 x 1024]).

// no transform (vmap, grad), trace or dispatch mode that wants to see the operators
bool nothing_watches(const Tensor &t) {
    using c10::DispatchKey;
    const c10::DispatchKeySet on = c10::impl::tls_local_dispatch_key_set().included_;
    if (on.has(DispatchKey::FuncTorchDynamicLayerFrontMode) || on.has(DispatchKey::Tracer) || on.has(DispatchKey::Functionalize) ||
        c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
    return !t.key_set().has_any(c10::DispatchKeySet({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                                     DispatchKey::Batched, DispatchKey::Functionalize}));
}

// The gradient that flows on to x.  A node and not a torch::autograd::Function: it holds the weight as MatMulLowBit's context
// does, as it is when the backward runs, past saved-tensor hooks and through repeated backwards.
struct ProductBackward : public torch::autograd::Node {
    Tensor w;
    int qtype = 0, layout = 0;
    int64_t N = 0, K = 0;
    at::ScalarType dtype = at::kHalf;
    at::DimVector x_shape;

    std::string name() const override { return "MatMulLowBitBackward"; }

    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        // (a gradient that a function above left out counts as zeros, as autograd functions in Python are given it)
        const Tensor grad = grads[0].defined() ? grads[0].to(dtype).reshape({-1, N})
                                               : at::zeros({c10::multiply_integers(x_shape) / K, N}, w.options().dtype(dtype));
        const int64_t M = grad.size(0);
        c10::DeviceGuard guard(grad.device());
        if (!is_blob(w, grad, qtype, N, K)) throw Failed("the low-bit weight is not where the forward found it");
        const int dt = dtype_code(dtype);
        void *const stream = current_stream(grad);
        const bool tracked = differentiable(grad) || !nothing_watches(grad);
        const size_t bytes = tracked ? 0 : api.backward_workspace_bytes(qtype, M, N, K);
        if (!tracked && api.backward_ws_applies(qtype, layout, dt, M, N, K, bytes)) {
            const Tensor g = grad.contiguous();
            if ((((uintptr_t)g.const_data_ptr() | (uintptr_t)w.const_data_ptr()) & 15) == 0) {
                Tensor gx = at::empty(x_shape, g.options());
                const Tensor ws = bytes ? at::empty({(int64_t)bytes}, g.options().dtype(at::kByte)) : Tensor();
                check(api.backward_ws(g.const_data_ptr(), w.const_data_ptr(), gx.data_ptr(), qtype, dt, M, N, K,
                                      bytes ? ws.data_ptr() : nullptr, bytes, stream), "lowbit_backward");
                return {gx};
            }
        }
        // (tracked: a second derivative, a tangent or a transform over the backward goes through the dense product)
        const Tensor dense = at::empty({N, K}, w.options().dtype(dtype));
        check(api.dequantize(w.const_data_ptr(), dense.data_ptr(), qtype, N, K, layout, dt, stream), "lowbit_dequantize");
        return {at::matmul(grad, dense).view(x_shape)};
    }
};

// LowBitLinear in training on a 16-bit x that wants a gradient, where the weight and bias want none; an undefined tensor when
// this is not the plain case
Tensor linear_train(const Tensor &x_in, const Tensor &w, const Tensor &bias, int qtype, int64_t N) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || !x_in.requires_grad() || !c10::GradMode::is_enabled()) return {};
    const int dt = dtype_code(x_in.scalar_type());
    const int64_t K = x_in.size(-1), M = x_in.numel() / K;
    if ((dt != LOWBIT_DT_F16 && dt != LOWBIT_DT_BF16) || !nothing_watches(x_in) || x_in._fw_grad(/*level=*/0).defined() ||
        !is_blob(w, x_in, qtype, N, K) || w.requires_grad()) return {};
    if (bias.defined() && (bias.scalar_type() != x_in.scalar_type() || bias.device() != x_in.device() || bias.numel() != N || !bias.is_contiguous() ||
                           bias.requires_grad() || differentiable(bias))) return {};
    Tensor y;
    auto node = std::shared_ptr<ProductBackward>(new ProductBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x_in));
    node->w = w;
    node->qtype = qtype;
    node->layout = device_layout(qtype, N, K);
    node->N = N;
    node->K = K;
    node->dtype = x_in.scalar_type();
    node->x_shape.assign(x_in.sizes().begin(), x_in.sizes().end());
    {
        c10::AutoGradMode no_grad(false);
        const Tensor x = x_in.detach().contiguous();
        y = product(x, w, bias, qtype, node->layout, M, N, K, with_last(x, N));
    }
    torch::autograd::set_history(y, node);
    return y;
}

// act(x Wg^T) * (x Wu^T) for 16-bit x and tiled weights; an undefined tensor when this is not the plain case
Tensor gated(const Tensor &x_in, const Tensor &wg, const Tensor &wu, int qtype, int64_t N, int act) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0) return {};
    const int dt = dtype_code(x_in.scalar_type());
    if (dt != LOWBIT_DT_F16 && dt != LOWBIT_DT_BF16) return {};
    const int64_t K = x_in.size(-1), M = x_in.numel() / K;
    if (!is_blob(wg, x_in, qtype, N, K) || !is_blob(wu, x_in, qtype, N, K) || !api.tileable(qtype, N, K)) return {};
    const Tensor x = x_in.is_contiguous() ? x_in : x_in.contiguous();
    c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(with_last(x, N), x.options());
    check(api.gated_mlp(x.const_data_ptr(), wg.const_data_ptr(), wu.const_data_ptr(), y.data_ptr(), qtype, dt, M, N, K, act,
                          current_stream(x)), "lowbit_gated_mlp");
    return y;
}

// rows ids[i] of the dequantized [N, K] table, in `dtype`; an undefined tensor when this is not the plain case
Tensor embedding(const Tensor &ids_in, const Tensor &w, int qtype, int64_t N, int64_t K, at::ScalarType dtype) {
    if (!on_gpu(ids_in) || ids_in.numel() == 0 || ids_in.scalar_type() != at::kLong || !is_blob(w, ids_in, qtype, N, K)) return {};
    const int dt = dtype_code(dtype);
    if (dt < 0) return {};
    const Tensor ids = ids_in.contiguous();
    c10::DeviceGuard guard(ids.device());
    at::DimVector shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(K);
    Tensor y = at::empty(shape, ids.options().dtype(dtype));
    check(api.dequantize_rows(w.const_data_ptr(), ids.const_data_ptr<int64_t>(), ids.numel(), y.data_ptr(), qtype, N, K,
                              device_layout(qtype, N, K), dt, current_stream(ids)), "lowbit_dequantize_rows");
    return y;
}

// a table of n weight pointers in x's device memory
bool is_table(const Tensor &t, const Tensor &x, int64_t n) {
    return t.device() == x.device() && t.layout() == at::kStrided && t.scalar_type() == at::kLong && t.numel() == n && t.is_contiguous();
}

// the experts of a mixture-of-experts block on x [tokens, hidden]; tables: one weight pointer per expert, on x's device.
// The caller has checked what the pointers lead to: gate, up [inter, hidden] and down [hidden, inter] weights of one qtype.
Tensor experts(const Tensor &x_in, const Tensor &ids_in, const Tensor &weight_in, const Tensor &gates, const Tensor &ups,
               const Tensor &downs, int qtype, int64_t hidden, int64_t inter, int act) {
    if (!on_gpu(x_in) || x_in.dim() != 2 || x_in.size(1) != hidden || ids_in.dim() != 2 || ids_in.size(0) != x_in.size(0) ||
        ids_in.numel() == 0 || !at::isIntegralType(ids_in.scalar_type(), /*includeBool=*/false) || weight_in.sizes() != ids_in.sizes() ||
        ids_in.device() != x_in.device() || weight_in.device() != x_in.device() || !is_table(gates, x_in, gates.numel()) ||
        !is_table(ups, x_in, gates.numel()) || !is_table(downs, x_in, gates.numel()) || differentiable(weight_in)) return {};
    const int dt = dtype_code(x_in.scalar_type()), wdt = dtype_code(weight_in.scalar_type());
    if ((dt != LOWBIT_DT_F16 && dt != LOWBIT_DT_BF16) || wdt < 0) return {};
    const int64_t tokens = ids_in.size(0), top_k = ids_in.size(1), n_exp = gates.numel();
    const size_t bytes = top_k > 64 || n_exp > 4096 ? 0 : api.experts_workspace_bytes(tokens, (int)top_k, (int)n_exp, hidden, inter);
    if (!bytes) return {};                               // more than the library takes
    const Tensor x = x_in.contiguous(), ids = ids_in.to(at::kLong).contiguous(), weight = weight_in.contiguous();
    c10::DeviceGuard guard(x.device());
    const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    Tensor y = at::empty({tokens, hidden}, x.options());
    check(api.experts_forward(x.const_data_ptr(), ids.const_data_ptr<int64_t>(), weight.const_data_ptr(), wdt, tokens, (int)top_k,
                              (int)n_exp, (const void *const *)gates.const_data_ptr(), (const void *const *)ups.const_data_ptr(),
                              (const void *const *)downs.const_data_ptr(), ws.data_ptr(), bytes, y.data_ptr(), qtype, dt, hidden, inter,
                              act, current_stream(x)), "lowbit_experts_forward");
    return y;
}

// ---- e4m3 operands with a scale for each block of 128

int64_t blocks(int64_t n) { return (n + 127) / 128; }

// rows as the kernels read them: contiguous, from a 16-byte boundary on
Tensor whole_rows(const Tensor &t) {
    Tensor c = t.contiguous();
    return ((uintptr_t)c.const_data_ptr() & 15) ? c.clone() : c;
}
// the same, of a tensor whose history is left behind (a detached tensor is a tensor more, half a microsecond: made only where a copy is)
Tensor whole_values(const Tensor &t) {
    return t.is_contiguous() && !((uintptr_t)t.const_data_ptr() & 15) ? t : whole_rows(t.detach());
}

// w holds e4m3 codes [.., N, K] and scale their scales, one per block of 128 x 128, on x's device
bool is_block_fp8(const Tensor &w, const Tensor &scale, const Tensor &x, int64_t matrices) {
    if (w.device() != x.device() || scale.device() != x.device() || w.layout() != at::kStrided || scale.layout() != at::kStrided ||
        w.scalar_type() != at::kFloat8_e4m3fn || scale.scalar_type() != at::kFloat || w.dim() < 2 || w.dim() != scale.dim() ||
        !w.is_contiguous() || !scale.is_contiguous() || ((uintptr_t)w.const_data_ptr() & 15)) return false;
    const int64_t d = w.dim();
    if (scale.size(d - 2) != blocks(w.size(d - 2)) || scale.size(d - 1) != blocks(w.size(d - 1)) || w.size(d - 1) % 16 || w.numel() == 0) return false;
    if (d == 3 && (w.size(0) != matrices || scale.size(0) != matrices)) return false;
    return d == (matrices ? 3 : 2) && !differentiable(w) && !differentiable(scale);
}

// codes and scales of x by row (weight false) or by 128 x 128; undefined tensors when this is not the plain case
std::pair<Tensor, Tensor> block_fp8_quantize(const Tensor &x_in, bool weight) {
    if (!on_gpu(x_in) || x_in.dim() < (weight ? 2 : 1) || x_in.numel() == 0 || x_in.size(-1) % 16 || dtype_code(x_in.scalar_type()) < 0 ||
        !nothing_watches(x_in)) return {};
    const Tensor x = whole_rows(x_in.detach());
    const int64_t K = x.size(-1), N = weight ? x.size(-2) : 1;
    c10::DeviceGuard guard(x.device());
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = blocks(K);
    if (weight) shape[shape.size() - 2] = blocks(N);
    const Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scale = at::empty(shape, x.options().dtype(at::kFloat));
    const int dt = dtype_code(x.scalar_type());
    if (weight)
        check(api.block_fp8_quantize_weight(x.const_data_ptr(), dt, x.numel() / (N * K), N, K, codes.data_ptr(), scale.data_ptr<float>(),
                                            current_stream(x)), "lowbit_block_fp8_quantize_weight");
    else
        check(api.block_fp8_quantize(x.const_data_ptr(), dt, x.numel() / K, K, codes.data_ptr(), scale.data_ptr<float>(), current_stream(x)),
              "lowbit_block_fp8_quantize");
    return {codes, scale};
}

Tensor block_fp8_product(const Tensor &x, const Tensor &w, const Tensor &scale, const Tensor &bias) {
    c10::DeviceGuard guard(x.device());
    const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
    const int dt = dtype_code(x.scalar_type());
    Tensor y = at::empty(with_last(x, N), x.options());
    const size_t bytes = api.block_fp8_linear_workspace_bytes(dt, M, N, K);
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    check(api.block_fp8_linear(x.const_data_ptr(), w.const_data_ptr(), scale.const_data_ptr<float>(), bias.defined() ? bias.const_data_ptr() : nullptr,
                               y.data_ptr(), dt, M, N, K, bytes ? ws.data_ptr() : nullptr, bytes, current_stream(x)), "lowbit_block_fp8_linear");
    return y;
}

// the weight in `dtype`, for what the kernels do not take
Tensor block_fp8_dense(const Tensor &w, const Tensor &scale, at::ScalarType dtype) {
    const Tensor rows = scale.repeat_interleave(128, 0).narrow(0, 0, w.size(0));
    return w.to(at::kFloat).mul_(rows.repeat_interleave(128, 1).narrow(1, 0, w.size(1))).to(dtype);
}

// The gradient that flows on to x, the quantization of x counting as the identity.  Holds the weight as ProductBackward does.
struct BlockFp8Backward : public torch::autograd::Node {
    Tensor w, scale;
    at::ScalarType dtype = at::kHalf, x_dtype = at::kHalf;   // what the gradient is multiplied in; x's own
    at::DimVector x_shape;

    std::string name() const override { return "BlockFp8LinearBackward"; }

    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        const int64_t N = w.size(0), K = w.size(1);
        const Tensor grad = grads[0].defined() ? grads[0].to(x_dtype).reshape({-1, N})
                                               : at::zeros({c10::multiply_integers(x_shape) / K, N}, w.options().dtype(x_dtype));
        c10::DeviceGuard guard(grad.device());
        if (grad.device() != w.device()) throw Failed("the block-scaled weight is not where the forward found it");
        if (dtype == at::kFloat || differentiable(grad) || !nothing_watches(grad))     // (float32, a second derivative, a transform: the dense product)
            return {at::matmul(grad, block_fp8_dense(w, scale, x_dtype)).view(x_shape)};
        const Tensor g = whole_rows(grad.to(dtype));
        const int64_t M = g.size(0);
        const int dt = dtype_code(dtype);
        Tensor gx = at::empty(x_shape, g.options());
        const size_t bytes = api.block_fp8_backward_workspace_bytes(dt, M, N, K);
        const Tensor ws = bytes ? at::empty({(int64_t)bytes}, g.options().dtype(at::kByte)) : Tensor();
        check(api.block_fp8_backward(g.const_data_ptr(), w.const_data_ptr(), scale.const_data_ptr<float>(), gx.data_ptr(), dt, M, N, K,
                                     bytes ? ws.data_ptr() : nullptr, bytes, current_stream(g)), "lowbit_block_fp8_backward");
        return {gx.to(x_dtype)};
    }
};

// y = Q(x) W^T (+ bias), with the gradient to x where x wants one; an undefined tensor when this is not the plain case.  grad_dt: a 16-bit
// type in which the gradient of a float32 product is multiplied, or x's own
Tensor block_fp8_linear(const Tensor &x_in, const Tensor &w, const Tensor &scale, const Tensor &bias, int grad_dt) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || dtype_code(x_in.scalar_type()) < 0 || !is_block_fp8(w, scale, x_in, 0) ||
        w.size(1) != x_in.size(-1) || !nothing_watches(x_in) || x_in._fw_grad(/*level=*/0).defined()) return {};
    if (bias.defined() && (bias.scalar_type() != x_in.scalar_type() || bias.device() != x_in.device() || bias.dim() != 1 ||
                           bias.numel() != w.size(0) || !bias.is_contiguous() || differentiable(bias))) return {};
    if (!x_in.requires_grad() || !c10::GradMode::is_enabled()) return block_fp8_product(whole_rows(x_in), w, scale, bias);
    Tensor y;
    auto node = std::shared_ptr<BlockFp8Backward>(new BlockFp8Backward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x_in));
    node->w = w;
    node->scale = scale;
    node->x_dtype = x_in.scalar_type();
    node->dtype = grad_dt == LOWBIT_DT_F16 ? at::kHalf : grad_dt == LOWBIT_DT_BF16 ? at::kBFloat16 : x_in.scalar_type();
    node->x_shape.assign(x_in.sizes().begin(), x_in.sizes().end());
    {
        c10::AutoGradMode no_grad(false);
        y = block_fp8_product(whole_rows(x_in.detach()), w, scale, bias);
    }
    torch::autograd::set_history(y, node);
    return y;
}

// the experts of a mixture-of-experts block; an undefined tensor when this is not the plain case
Tensor block_fp8_experts(const Tensor &x_in, const Tensor &ids_in, const Tensor &weight_in, const Tensor &gate_up, const Tensor &gate_up_scale,
                         const Tensor &down, const Tensor &down_scale, int act) {
    if (!on_gpu(x_in) || x_in.dim() != 2 || gate_up.dim() != 3 || ids_in.dim() != 2 || ids_in.size(0) != x_in.size(0) || ids_in.numel() == 0 ||
        !at::isIntegralType(ids_in.scalar_type(), /*includeBool=*/false) || weight_in.sizes() != ids_in.sizes() ||
        ids_in.device() != x_in.device() || weight_in.device() != x_in.device() || differentiable(weight_in) || differentiable(x_in) ||
        !nothing_watches(x_in)) return {};
    const int64_t n_exp = gate_up.size(0), hidden = x_in.size(1), inter = gate_up.size(1) / 2;
    if (!is_block_fp8(gate_up, gate_up_scale, x_in, n_exp) || !is_block_fp8(down, down_scale, x_in, n_exp) || gate_up.size(1) != 2 * inter ||
        gate_up.size(2) != hidden || down.size(1) != hidden || down.size(2) != inter) return {};
    const int dt = dtype_code(x_in.scalar_type()), wdt = dtype_code(weight_in.scalar_type());
    if ((dt != LOWBIT_DT_F16 && dt != LOWBIT_DT_BF16) || wdt < 0) return {};
    const int64_t tokens = ids_in.size(0), top_k = ids_in.size(1);
    const size_t bytes = top_k > 64 || n_exp > 4096 ? 0 : api.block_fp8_experts_workspace_bytes(tokens, (int)top_k, (int)n_exp, hidden, inter);
    if (!bytes) return {};                               // more than the library takes
    const Tensor x = whole_rows(x_in), ids = ids_in.to(at::kLong).contiguous(), weight = weight_in.contiguous();
    c10::DeviceGuard guard(x.device());
    const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    Tensor y = at::empty({tokens, hidden}, x.options());
    check(api.block_fp8_experts(x.const_data_ptr(), ids.const_data_ptr<int64_t>(), weight.const_data_ptr(), wdt, tokens, (int)top_k, (int)n_exp,
                                gate_up.const_data_ptr(), gate_up_scale.const_data_ptr<float>(), down.const_data_ptr(),
                                down_scale.const_data_ptr<float>(), ws.data_ptr(), bytes, y.data_ptr(), dt, hidden, inter, act,
                                current_stream(x)), "lowbit_block_fp8_experts");
    return y;
}

// ---- int8 operands with a scale for each row

// w holds int8 codes [.., N, K] and scale their scales [.., N], on x's device
bool holds_row_int8(const Tensor &w, const Tensor &scale, const Tensor &x, int64_t matrices) {
    if (w.device() != x.device() || scale.device() != x.device() || w.layout() != at::kStrided || scale.layout() != at::kStrided ||
        w.scalar_type() != at::kChar || scale.scalar_type() != at::kFloat || w.dim() != (matrices ? 3 : 2) || scale.dim() != w.dim() - 1 ||
        !w.is_contiguous() || !scale.is_contiguous() || ((uintptr_t)w.const_data_ptr() & 15) || w.numel() == 0 || w.size(-1) % 16) return false;
    return scale.sizes() == w.sizes().slice(0, w.dim() - 1) && (!matrices || w.size(0) == matrices) && !differentiable(scale);
}
// .. and no transform or trace is about, whose tensors have no pointers to ask for
bool is_row_int8(const Tensor &w, const Tensor &scale, const Tensor &x, int64_t matrices) {
    return nothing_watches(w) && nothing_watches(scale) && holds_row_int8(w, scale, x, matrices);
}

constexpr int64_t ROW_INT8_MOST_K = 1 << 17;

// codes and scales of x by row; undefined tensors when this is not the plain case
std::pair<Tensor, Tensor> row_int8_quantize(const Tensor &x_in) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || x_in.size(-1) % 16 || dtype_code(x_in.scalar_type()) < 0 ||
        !nothing_watches(x_in)) return {};
    const Tensor x = whole_values(x_in);
    const int64_t K = x.size(-1);
    c10::DeviceGuard guard(x.device());
    const Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar)),
                 scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    check(api.row_int8_quantize(x.const_data_ptr(), dtype_code(x.scalar_type()), x.numel() / K, K, codes.data_ptr(), scale.data_ptr<float>(),
                                current_stream(x)), "lowbit_row_int8_quantize");
    return {codes, scale};
}

// y in `dtype` of rows x (or of codes and their scales), whole as the kernels read them
Tensor row_int8_any_product(const Tensor &x, const Tensor &xs, const Tensor &w, const Tensor &scale, const Tensor &bias, at::ScalarType dtype) {
    c10::DeviceGuard guard(x.device());
    const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
    const int dt = dtype_code(dtype);
    Tensor y = at::empty(with_last(x, N), x.options().dtype(dtype));
    const size_t bytes = (xs.defined() ? api.row_int8_product_workspace_bytes : api.row_int8_linear_workspace_bytes)(dt, M, N, K);
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    const void *const b = bias.defined() ? bias.const_data_ptr() : nullptr;
    if (xs.defined())
        check(api.row_int8_product(x.const_data_ptr(), xs.const_data_ptr<float>(), w.const_data_ptr(), scale.const_data_ptr<float>(), b, y.data_ptr(), dt, M, N, K,
                                   bytes ? ws.data_ptr() : nullptr, bytes, current_stream(x)), "lowbit_row_int8_product");
    else
        check(api.row_int8_linear(x.const_data_ptr(), w.const_data_ptr(), scale.const_data_ptr<float>(), b, y.data_ptr(), dt, M, N, K,
                                  bytes ? ws.data_ptr() : nullptr, bytes, current_stream(x)), "lowbit_row_int8_linear");
    return y;
}

// a bias that the kernels add themselves
bool plain_bias(const Tensor &bias, const Tensor &x, at::ScalarType dtype, int64_t N) {
    return !bias.defined() || (bias.scalar_type() == dtype && bias.device() == x.device() && bias.dim() == 1 && bias.numel() == N &&
                               bias.is_contiguous() && !differentiable(bias) && nothing_watches(bias));
}

// how often a tensor was changed in place (inference tensors do not count that)
static int64_t changes(const Tensor &t) { return t.is_inference() ? 0 : (int64_t)t._version(); }

// The gradient that flows on to x, the quantization of x counting as the identity.  Holds the weight as ProductBackward does.
struct RowInt8Backward : public torch::autograd::Node {
    Tensor w, scale;
    int64_t N = 0, K = 0, w_changes = 0, scale_changes = 0;  // of the forward
    at::ScalarType x_dtype = at::kHalf;
    at::DimVector x_shape;

    std::string name() const override { return "RowInt8LinearBackward"; }

    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        const Tensor grad = grads[0].defined() ? grads[0].to(x_dtype).reshape({-1, N})
                                               : at::zeros({c10::multiply_integers(x_shape) / K, N}, w.options().dtype(x_dtype));
        c10::DeviceGuard guard(grad.device());
        // (a tensor's data may have been replaced, also by some of another size, which counts no change)
        if (!holds_row_int8(w, scale, grad, 0) || w.size(0) != N || w.size(1) != K) throw Failed("the int8 weight is not what the forward found");
        if (changes(w) != w_changes || changes(scale) != scale_changes)
            throw Failed("the int8 weight or its scales have been modified by an inplace operation since the forward");
        if (differentiable(grad) || !nothing_watches(grad))  // (a second derivative, a transform: the dense product)
            return {at::matmul(grad.to(at::kFloat), w.to(at::kFloat).mul_(scale.unsqueeze(-1))).to(x_dtype).view(x_shape)};
        const Tensor g = whole_rows(grad);
        const int64_t M = g.size(0);
        const int dt = dtype_code(x_dtype);
        Tensor gx = at::empty(x_shape, g.options());
        const size_t bytes = api.row_int8_backward_workspace_bytes(dt, M, N, K);
        const Tensor ws = bytes ? at::empty({(int64_t)bytes}, g.options().dtype(at::kByte)) : Tensor();
        check(api.row_int8_backward(g.const_data_ptr(), w.const_data_ptr(), scale.const_data_ptr<float>(), gx.data_ptr(), dt, M, N, K,
                                    bytes ? ws.data_ptr() : nullptr, bytes, current_stream(g)), "lowbit_row_int8_backward");
        return {gx};
    }
};

// y = Q(x) W^T (+ bias), with the gradient to x where x wants one; an undefined tensor when this is not the plain case
Tensor row_int8_linear(const Tensor &x_in, const Tensor &w, const Tensor &scale, const Tensor &bias) {
    if (!on_gpu(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || dtype_code(x_in.scalar_type()) < 0 || !is_row_int8(w, scale, x_in, 0) ||
        w.size(1) != x_in.size(-1) || w.size(1) > ROW_INT8_MOST_K || !nothing_watches(x_in) || x_in._fw_grad(/*level=*/0).defined() ||
        !plain_bias(bias, x_in, x_in.scalar_type(), w.size(0))) return {};
    if (!x_in.requires_grad() || !c10::GradMode::is_enabled()) return row_int8_any_product(whole_rows(x_in), Tensor(), w, scale, bias, x_in.scalar_type());
    Tensor y;
    auto node = std::shared_ptr<RowInt8Backward>(new RowInt8Backward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x_in));
    node->w = w;
    node->scale = scale;
    node->N = w.size(0);
    node->K = w.size(1);
    node->w_changes = changes(w);
    node->scale_changes = changes(scale);
    node->x_dtype = x_in.scalar_type();
    node->x_shape.assign(x_in.sizes().begin(), x_in.sizes().end());
    {
        c10::AutoGradMode no_grad(false);
        y = row_int8_any_product(whole_values(x_in), Tensor(), w, scale, bias, x_in.scalar_type());
    }
    torch::autograd::set_history(y, node);
    return y;
}

// the same product of codes and their scales, in the type of dtype code `dt`; an undefined tensor when this is not the plain case
Tensor row_int8_product(const Tensor &codes, const Tensor &xs, const Tensor &w, const Tensor &scale, const Tensor &bias, int dt) {
    const at::ScalarType dtype = dt == LOWBIT_DT_F16 ? at::kHalf : dt == LOWBIT_DT_BF16 ? at::kBFloat16 : at::kFloat;
    if (!on_gpu(codes) || codes.scalar_type() != at::kChar || codes.dim() < 1 || codes.numel() == 0 || !is_row_int8(w, scale, codes, 0) ||
        w.size(1) != codes.size(-1) || w.size(1) > ROW_INT8_MOST_K || xs.device() != codes.device() || xs.scalar_type() != at::kFloat ||
        xs.sizes() != codes.sizes().slice(0, codes.dim() - 1) || differentiable(xs) || !nothing_watches(codes) || !nothing_watches(xs) ||
        !plain_bias(bias, codes, dtype, w.size(0))) return {};
    return row_int8_any_product(whole_rows(codes), xs.contiguous(), w, scale, bias, dtype);
}

// codes and scales of E experts that fit together: gate_up [E, 2 I, H], down [E, H, I]
bool are_row_int8_experts(const Tensor &x, const Tensor &gate_up, const Tensor &gate_up_scale, const Tensor &down, const Tensor &down_scale) {
    if (gate_up.dim() != 3 || down.dim() != 3 || gate_up.size(1) % 2) return false;
    const int64_t n_exp = gate_up.size(0), hidden = x.size(1), inter = gate_up.size(1) / 2;
    return is_row_int8(gate_up, gate_up_scale, x, n_exp) && is_row_int8(down, down_scale, x, n_exp) && gate_up.size(2) == hidden &&
           down.size(1) == hidden && down.size(2) == inter;
}

// the experts of a mixture-of-experts block; an undefined tensor when this is not the plain case
Tensor row_int8_experts(const Tensor &x_in, const Tensor &ids_in, const Tensor &weight_in, const Tensor &gate_up, const Tensor &gate_up_scale,
                        const Tensor &down, const Tensor &down_scale, int act) {
    if (!on_gpu(x_in) || x_in.dim() != 2 || ids_in.dim() != 2 || ids_in.size(0) != x_in.size(0) || ids_in.numel() == 0 ||
        !at::isIntegralType(ids_in.scalar_type(), /*includeBool=*/false) || weight_in.sizes() != ids_in.sizes() ||
        ids_in.device() != x_in.device() || weight_in.device() != x_in.device() || differentiable(weight_in) || differentiable(x_in) ||
        !nothing_watches(x_in) || !nothing_watches(ids_in) || !nothing_watches(weight_in) ||
        !are_row_int8_experts(x_in, gate_up, gate_up_scale, down, down_scale)) return {};
    const int64_t n_exp = gate_up.size(0), hidden = x_in.size(1), inter = gate_up.size(1) / 2;
    const int dt = dtype_code(x_in.scalar_type()), wdt = dtype_code(weight_in.scalar_type());
    if (dt < 0 || wdt < 0) return {};
    const int64_t tokens = ids_in.size(0), top_k = ids_in.size(1);
    const size_t bytes = top_k > 64 || n_exp > 4096 ? 0 : api.row_int8_experts_workspace_bytes(tokens, (int)top_k, (int)n_exp, hidden, inter);
    if (!bytes) return {};                               // more than the library takes
    c10::DeviceGuard guard(x_in.device());
    const Tensor x = whole_rows(x_in), ids = ids_in.to(at::kLong).contiguous(), weight = weight_in.contiguous(), gs = whole_rows(gate_up_scale),
                 ds = whole_rows(down_scale);
    const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    Tensor y = at::empty({tokens, hidden}, x.options());
    check(api.row_int8_experts(x.const_data_ptr(), ids.const_data_ptr<int64_t>(), weight.const_data_ptr(), wdt, tokens, (int)top_k, (int)n_exp,
                               gate_up.const_data_ptr(), gs.const_data_ptr<float>(), down.const_data_ptr(), ds.const_data_ptr<float>(), ws.data_ptr(), bytes,
                               y.data_ptr(), dt, hidden, inter, act, current_stream(x)), "lowbit_row_int8_experts");
    return y;
}

// ---- the router of a mixture-of-experts block

struct RouteRule {
    int64_t top_k;
    bool sigmoid, renormalize;
    double factor;
};

// operands of a router on one GPU, of types and sizes that the library takes
bool plain_route(const Tensor &x, const Tensor &router, const Tensor &bias, const RouteRule &rule) {
    if (!on_gpu(x) || x.dim() != 2 || x.numel() == 0 || dtype_code(x.scalar_type()) < 0 || router.device() != x.device() || router.layout() != at::kStrided ||
        router.dim() != 2 || router.numel() == 0 || dtype_code(router.scalar_type()) < 0 || router.size(1) != x.size(1) || !nothing_watches(x) ||
        !nothing_watches(router) || x._fw_grad(/*level=*/0).defined() || router._fw_grad(/*level=*/0).defined()) return false;
    if (bias.defined() && (bias.device() != x.device() || bias.dim() != 1 || bias.size(0) != router.size(0) || bias.scalar_type() != at::kFloat ||
                           !nothing_watches(bias))) return false;
    return rule.top_k >= 1 && rule.top_k <= 64 && rule.top_k <= router.size(0) && x.size(0) <= 1 << 21 && router.size(0) <= 1024 && x.size(1) % 8 == 0 &&
           x.size(1) <= 1 << 20;                             // (what the library takes)
}

struct RouteBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable x_saved, router_saved, ids_saved;         // (the ids are the caller's too, who may change them)
    Tensor logits;
    int64_t hidden = 0;
    RouteRule rule{};

    std::string name() const override { return "MoeRouteBackward"; }
    void release_variables() override {
        x_saved.reset_data();
        router_saved.reset_data();
        ids_saved.reset_data();
        logits.reset();
    }

    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        const Tensor x = x_saved.unpack(), router = router_saved.unpack(), ids = ids_saved.unpack();
        // (a tensor's data may have been replaced, also by some of another size, which counts no change)
        if (x.sizes() != at::IntArrayRef({logits.size(0), hidden}) || router.sizes() != at::IntArrayRef({logits.size(1), hidden}) ||
            x.device() != logits.device() || router.device() != x.device() || dtype_code(x.scalar_type()) < 0 || dtype_code(router.scalar_type()) < 0)
            throw Failed("the router's operands are not what the forward found");
        if (ids.sizes() != at::IntArrayRef({logits.size(0), rule.top_k}) || ids.scalar_type() != at::kLong || ids.device() != x.device() || !ids.is_contiguous())
            throw Failed("the indices of the router are not what the forward found");
        const int64_t T = x.size(0), H = x.size(1), E = router.size(0);
        c10::DeviceGuard guard(x.device());
        const Tensor grad = grads[0].defined() ? grads[0] : at::zeros(ids.sizes(), logits.options().dtype(at::kFloat));
        const bool want_x = task_should_compute_output(0), want_r = task_should_compute_output(1);
        if (!want_x && !want_r) return {Tensor(), Tensor()};
        if (differentiable(grad) || !nothing_watches(grad) || c10::GradMode::is_enabled()) {
            // A second derivative, a transform: the gradient's formula (route.hip) in torch operators on the caller's operands, so that what they were made
            // from and their hooks come in where the engine walks on from here.
            const Tensor xd = x.to(at::kDouble), rd = router.to(at::kDouble), z = at::matmul(xd, rd.t()), s = rule.sigmoid ? z.sigmoid() : z.softmax(-1);
            const Tensor chosen = ids.clamp(0, E - 1);       // (numbers written past the version count, by .data: none out of range)
            Tensor dc = grad.to(at::kDouble) * rule.factor;
            if (rule.renormalize) {
                const Tensor c = s.gather(1, chosen), sum = c.sum(-1, true);
                dc = (dc - (dc * (c / sum)).sum(-1, true)) / sum;
            }
            const Tensor ds = at::zeros_like(s).scatter(1, chosen, dc), dz = rule.sigmoid ? ds * s * (1 - s) : s * (ds - (ds * s).sum(-1, true));
            return {want_x ? at::matmul(dz, rd).to(x.scalar_type()) : Tensor(), want_r ? at::matmul(dz.t(), xd).to(router.scalar_type()) : Tensor()};
        }
        const Tensor xr = whole_values(x), rr = whole_values(router), g = grad.to(at::kFloat).contiguous();
        Tensor gx = want_x ? at::empty(xr.sizes(), xr.options()) : Tensor(), gr = want_r ? at::empty(rr.sizes(), rr.options()) : Tensor();
        const size_t bytes = api.route_backward_workspace_bytes(T, (int)E, H);
        const Tensor ws = at::empty({(int64_t)bytes}, xr.options().dtype(at::kByte));
        check(api.route_backward(g.const_data_ptr<float>(), logits.const_data_ptr<double>(), ids.const_data_ptr<int64_t>(), xr.const_data_ptr(),
                                 dtype_code(xr.scalar_type()), rr.const_data_ptr(), dtype_code(rr.scalar_type()), T, (int)E, H, (int)rule.top_k, rule.sigmoid,
                                 rule.renormalize, (float)rule.factor, want_x ? gx.data_ptr() : nullptr, want_r ? gr.data_ptr() : nullptr, ws.data_ptr(), bytes,
                                 current_stream(xr)), "lowbit_route_backward");
        return {gx, gr};
    }
};

// (weights [T, top_k], indices [T, top_k]); undefined tensors when this is not the plain case
std::pair<Tensor, Tensor> route(const Tensor &x_in, const Tensor &router_in, const Tensor &bias_in, const RouteRule &rule) {
    if (!plain_route(x_in, router_in, bias_in, rule)) return {};
    c10::DeviceGuard guard(x_in.device());
    const bool wants = c10::GradMode::is_enabled() && (x_in.requires_grad() || router_in.requires_grad());
    const int64_t T = x_in.size(0), H = x_in.size(1), E = router_in.size(0);
    Tensor w, ids, logits;
    {
        c10::AutoGradMode no_grad(false);
        const Tensor x = whole_values(x_in), router = whole_values(router_in), bias = bias_in.defined() ? bias_in.detach().contiguous() : Tensor();
        w = at::empty({T, rule.top_k}, x.options().dtype(at::kFloat));
        ids = at::empty({T, rule.top_k}, x.options().dtype(at::kLong));
        if (wants) logits = at::empty({T, E}, x.options().dtype(at::kDouble));
        const size_t bytes = api.route_workspace_bytes(T, (int)E, H);
        const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
        check(api.route(x.const_data_ptr(), dtype_code(x.scalar_type()), router.const_data_ptr(), dtype_code(router.scalar_type()),
                        bias.defined() ? bias.const_data_ptr<float>() : nullptr, T, (int)E, H, (int)rule.top_k, rule.sigmoid, rule.renormalize,
                        (float)rule.factor, w.data_ptr<float>(), ids.data_ptr<int64_t>(), wants ? logits.data_ptr<double>() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes,
                        current_stream(x)), "lowbit_route");
    }
    if (wants) {
        auto node = std::shared_ptr<RouteBackward>(new RouteBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, router_in));
        node->x_saved = torch::autograd::SavedVariable(x_in, /*is_output=*/false);
        node->router_saved = torch::autograd::SavedVariable(router_in, /*is_output=*/false);
        node->ids_saved = torch::autograd::SavedVariable(ids, /*is_output=*/false);
        node->logits = logits;
        node->hidden = H;
        node->rule = rule;
        torch::autograd::set_history(w, node);
    }
    return {w, ids};
}

// router and experts in one call; an undefined tensor when this is not the plain case
Tensor row_int8_moe(const Tensor &x_in, const Tensor &router_in, const Tensor &bias_in, const RouteRule &rule, const Tensor &gate_up, const Tensor &gate_up_scale,
                    const Tensor &down, const Tensor &down_scale, int act) {
    if (!plain_route(x_in, router_in, bias_in, rule) || differentiable(x_in) || differentiable(router_in) ||
        !are_row_int8_experts(x_in, gate_up, gate_up_scale, down, down_scale) || router_in.size(0) != gate_up.size(0)) return {};
    const int64_t T = x_in.size(0), H = x_in.size(1), E = router_in.size(0), I = gate_up.size(1) / 2;
    const size_t bytes = api.row_int8_moe_workspace_bytes(T, (int)rule.top_k, (int)E, H, I);
    if (!bytes) return {};                               // more than the library takes
    c10::DeviceGuard guard(x_in.device());
    const Tensor x = whole_rows(x_in), router = whole_rows(router_in), bias = bias_in.defined() ? bias_in.contiguous() : Tensor(),
                 gs = whole_rows(gate_up_scale), ds = whole_rows(down_scale);
    const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    Tensor y = at::empty({T, H}, x.options());
    check(api.row_int8_moe(x.const_data_ptr(), router.const_data_ptr(), dtype_code(router.scalar_type()), bias.defined() ? bias.const_data_ptr<float>() : nullptr,
                           T, (int)rule.top_k, (int)E, rule.sigmoid, rule.renormalize, (float)rule.factor, gate_up.const_data_ptr(), gs.const_data_ptr<float>(),
                           down.const_data_ptr(), ds.const_data_ptr<float>(), ws.data_ptr(), bytes, y.data_ptr(), dtype_code(x.scalar_type()), H, I, act,
                           current_stream(x)), "lowbit_row_int8_moe");
    return y;
}

// ---- large copies between pageable host memory and the GPU, through two pinned buffers
//
// A pageable copy by the runtime ran at 29 GB/s up and, into memory the process has not touched yet, 7.5 GB/s down
// (the bus: 57).  Here a chunk crosses the bus while all cores copy the one before or after it between pageable and
// pinned memory: [11008 x 4096] float16 up 3.2 -> 2.0 ms, its sym_int4 blob down 1.5 (fresh memory: 3.4) -> 0.6 ms.  The buffers are torch's
// (its caching allocator for pinned memory: kept between calls, at most two chunks per call in flight, safe with
// several threads and streams).  Smaller tensors are left to Tensor.to.
constexpr int64_t COPY_CHUNK = (int64_t)4 << 20;

struct Staging {
    c10::Stream stream;
    Tensor buffer[2];
    c10::Event done[2] = {c10::Event(c10::DeviceType::CUDA), c10::Event(c10::DeviceType::CUDA)};
    explicit Staging(c10::Device device) : stream(c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getStream(device)) {
        for (Tensor &b : buffer) b = at::empty({COPY_CHUNK}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
    }
};

Tensor as_bytes(const Tensor &t) {                       // the storage of a contiguous tensor as uint8 [nbytes]
    return at::empty({0}, t.options().dtype(at::kByte)).set_(t.storage(), t.storage_offset() * (int64_t)t.itemsize(), {(int64_t)t.nbytes()}, {1});
}

bool copies_in_chunks(const Tensor &t, bool gpu) {
    return t.layout() == at::kStrided && (gpu ? t.device().is_cuda() : t.device().is_cpu() && !t.is_pinned()) && t.is_contiguous() &&
           (int64_t)t.nbytes() > COPY_CHUNK && !t.requires_grad();
}

Tensor upload(const Tensor &host, c10::DeviceIndex index) {
    if (!copies_in_chunks(host, false)) return {};
    const c10::Device device(c10::DeviceType::CUDA, index);
    c10::DeviceGuard guard(device);
    at::AutoDispatchBelowADInplaceOrView no_views;
    Staging s(device);
    Tensor out = at::empty(host.sizes(), host.options().device(device));
    const Tensor from = as_bytes(host), to = as_bytes(out);
    const int64_t n = from.numel();
    for (int64_t at = 0, i = 0; at < n; at += COPY_CHUNK, i++) {
        const int64_t len = std::min(COPY_CHUNK, n - at);
        const Tensor pinned = s.buffer[i & 1].narrow(0, 0, len);
        if (i >= 2) s.done[i & 1].synchronize();         // the buffer's last chunk has left it
        pinned.copy_(from.narrow(0, at, len));
        to.narrow(0, at, len).copy_(pinned, true);
        s.done[i & 1].record(s.stream);
    }
    for (int64_t i = 0; i < std::min<int64_t>(2, (n + COPY_CHUNK - 1) / COPY_CHUNK); i++) s.done[i].synchronize();
    return out;
}

Tensor download(const Tensor &dev) {
    if (!copies_in_chunks(dev, true)) return {};
    c10::DeviceGuard guard(dev.device());
    at::AutoDispatchBelowADInplaceOrView no_views;
    Staging s(dev.device());
    Tensor out = at::empty(dev.sizes(), dev.options().device(c10::kCPU));
    const Tensor from = as_bytes(dev), to = as_bytes(out);
    const int64_t n = from.numel(), chunks = (n + COPY_CHUNK - 1) / COPY_CHUNK;
    auto length = [&](int64_t i) { return std::min(COPY_CHUNK, n - i * COPY_CHUNK); };
    for (int64_t i = 0; i <= chunks; i++) {
        if (i < chunks) {
            s.buffer[i & 1].narrow(0, 0, length(i)).copy_(from.narrow(0, i * COPY_CHUNK, length(i)), true);
            s.done[i & 1].record(s.stream);
        }
        if (i == 0) continue;
        s.done[(i - 1) & 1].synchronize();               // chunk i - 1 has arrived, chunk i is on its way
        to.narrow(0, (i - 1) * COPY_CHUNK, length(i - 1)).copy_(s.buffer[(i - 1) & 1].narrow(0, 0, length(i - 1)));
    }
    return out;
}

// ------------------------------------------------------------------ CPython side

// Arguments by position.  A tensor argument is a torch.Tensor or a Parameter (subclass): anything else, and a value
// of the wrong kind, raises TypeError.
struct Args {
    PyObject *const *a;
    Py_ssize_t n;
    const Tensor &tensor(Py_ssize_t i) const {
        if (!THPVariable_Check(a[i])) throw std::invalid_argument("a tensor is expected");
        return THPVariable_Unpack(a[i]);
    }
    Tensor optional(Py_ssize_t i) const { return a[i] == Py_None ? Tensor() : tensor(i); }
    int64_t integer(Py_ssize_t i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); throw std::invalid_argument("an integer is expected"); }
        return v;
    }
    double number(Py_ssize_t i) const {
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); throw std::invalid_argument("a number is expected"); }
        return v;
    }
    bool truth(Py_ssize_t i) const { return PyObject_IsTrue(a[i]) == 1; }
};

// Runs fn (returning a Tensor) without the GIL and wraps the result, None for an undefined one.
template <typename Fn> PyObject *answer(const char *name, Py_ssize_t got, Py_ssize_t want, Fn &&fn) {
    HANDLE_TH_ERRORS
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, got);
        return nullptr;
    }
    try {
        Tensor y = fn();
        if (!y.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(y));
    } catch (const std::invalid_argument &e) {
        PyErr_Format(PyExc_TypeError, "%s: %s", name, e.what());
    } catch (const Failed &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

// The same for fn returning two tensors: a tuple, or None where they are undefined.
template <typename Fn> PyObject *answer_pair(const char *name, Py_ssize_t got, Py_ssize_t want, Fn &&fn) {
    std::pair<Tensor, Tensor> both;
    PyObject *first = answer(name, got, want, [&] {
        both = fn();
        return both.first;
    });
    if (!first || first == Py_None) return first;
    HANDLE_TH_ERRORS
    PyObject *second = THPVariable_Wrap(std::move(both.second));
    if (!second) {
        Py_DECREF(first);
        return nullptr;
    }
    PyObject *tuple = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return tuple;
    END_HANDLE_TH_ERRORS
}

struct NoGil {
    PyThreadState *state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

PyObject *py_bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 1 || !PyDict_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "bind takes a dict of function addresses");
        return nullptr;
    }
#define BIND(name)                                                                                 \
    do {                                                                                           \
        PyObject *v = PyDict_GetItemString(args[0], "lowbit_" #name);                              \
        void *p = v ? PyLong_AsVoidPtr(v) : nullptr;                                               \
        if (!p) {                                                                                  \
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "lowbit_" #name);               \
            return nullptr;                                                                        \
        }                                                                                          \
        api.name = (decltype(api.name))p;                                                          \
    } while (0)
    BIND(last_error); BIND(blob_bytes); BIND(tileable); BIND(linear_scratch_bytes); BIND(linear);
    BIND(gated_mlp); BIND(dequantize_rows); BIND(dequantize); BIND(backward_ws); BIND(backward_workspace_bytes); BIND(backward_ws_applies); BIND(experts_workspace_bytes); BIND(experts_forward);
    BIND(block_fp8_quantize); BIND(block_fp8_quantize_weight); BIND(block_fp8_linear); BIND(block_fp8_linear_workspace_bytes);
    BIND(row_int8_quantize); BIND(row_int8_linear); BIND(row_int8_linear_workspace_bytes); BIND(row_int8_product);
    BIND(row_int8_experts); BIND(row_int8_experts_workspace_bytes); BIND(row_int8_moe); BIND(row_int8_moe_workspace_bytes);
    BIND(route); BIND(route_workspace_bytes); BIND(route_backward); BIND(route_backward_workspace_bytes);
    BIND(row_int8_product_workspace_bytes); BIND(row_int8_backward); BIND(row_int8_backward_workspace_bytes);
    BIND(block_fp8_backward); BIND(block_fp8_backward_workspace_bytes); BIND(block_fp8_experts); BIND(block_fp8_experts_workspace_bytes);
#undef BIND
    Py_RETURN_NONE;
}

// product(x [M, K] contiguous, w, qtype, layout, N) -> [M, N] in x's dtype; the caller has checked the arguments
PyObject *py_product(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("product", n, 5, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &w = a.tensor(1);
        const int qtype = (int)a.integer(2), layout = (int)a.integer(3);
        const int64_t N = a.integer(4), M = x.size(0), K = x.size(1);
        NoGil free;
        return product(x, w, Tensor(), qtype, layout, M, N, K, {M, N});
    });
}

// linear(x, weight, bias or None, qtype, out_len, conver_to_half) -> y or None
PyObject *py_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("linear", n, 6, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &w = a.tensor(1);
        const Tensor bias = a.optional(2);
        const int qtype = (int)a.integer(3);
        const int64_t N = a.integer(4);
        const bool half = a.truth(5);
        NoGil free;
        return linear(x, w, bias, qtype, N, half);
    });
}

// linear_train(x, weight, bias or None, qtype, out_len) -> y or None
PyObject *py_linear_train(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("linear_train", n, 5, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &w = a.tensor(1);
        const Tensor bias = a.optional(2);
        const int qtype = (int)a.integer(3);
        const int64_t N = a.integer(4);
        NoGil free;
        return linear_train(x, w, bias, qtype, N);
    });
}

// gated(x, w_gate, w_up, qtype, out_len, act) -> y or None
PyObject *py_gated(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("gated", n, 6, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &wg = a.tensor(1), &wu = a.tensor(2);
        const int qtype = (int)a.integer(3), act = (int)a.integer(5);
        const int64_t N = a.integer(4);
        NoGil free;
        return gated(x, wg, wu, qtype, N, act);
    });
}

// embedding(ids, weight, qtype, num_embeddings, embedding_dim, tensor of the result's dtype) -> rows or None
PyObject *py_embedding(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("embedding", n, 6, [&] {
        const Args a{args, n};
        const Tensor &ids = a.tensor(0), &w = a.tensor(1);
        const int qtype = (int)a.integer(2);
        const int64_t N = a.integer(3), K = a.integer(4);
        const at::ScalarType dtype = a.tensor(5).scalar_type();
        NoGil free;
        return embedding(ids, w, qtype, N, K, dtype);
    });
}

// experts(x, ids, weights, gates, ups, downs, qtype, hidden, inter, act) -> y or None
PyObject *py_experts(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("experts", n, 10, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &ids = a.tensor(1), &weight = a.tensor(2), &g = a.tensor(3), &u = a.tensor(4), &d = a.tensor(5);
        const int qtype = (int)a.integer(6), act = (int)a.integer(9);
        const int64_t hidden = a.integer(7), inter = a.integer(8);
        NoGil free;
        return experts(x, ids, weight, g, u, d, qtype, hidden, inter, act);
    });
}

// block_fp8_quantize(x, weight) -> (codes, scale) or None
PyObject *py_block_fp8_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer_pair("block_fp8_quantize", n, 2, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0);
        const bool weight = a.truth(1);
        NoGil free;
        return block_fp8_quantize(x, weight);
    });
}

// block_fp8_linear(x, weight, scale, bias or None, dtype code of the gradient's product) -> y or None
PyObject *py_block_fp8_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("block_fp8_linear", n, 5, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &w = a.tensor(1), &scale = a.tensor(2);
        const Tensor bias = a.optional(3);
        const int grad_dt = (int)a.integer(4);
        NoGil free;
        return block_fp8_linear(x, w, scale, bias, grad_dt);
    });
}

// block_fp8_experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, act) -> y or None
PyObject *py_block_fp8_experts(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("block_fp8_experts", n, 8, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &ids = a.tensor(1), &weight = a.tensor(2);
        const Tensor &gu = a.tensor(3), &gus = a.tensor(4), &d = a.tensor(5), &ds = a.tensor(6);
        const int act = (int)a.integer(7);
        NoGil free;
        return block_fp8_experts(x, ids, weight, gu, gus, d, ds, act);
    });
}

// row_int8_quantize(x) -> (codes, scale) or None
PyObject *py_row_int8_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer_pair("row_int8_quantize", n, 1, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0);
        NoGil free;
        return row_int8_quantize(x);
    });
}

// row_int8_linear(x, weight, scale, bias or None) -> y or None
PyObject *py_row_int8_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("row_int8_linear", n, 4, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &w = a.tensor(1), &scale = a.tensor(2);
        const Tensor bias = a.optional(3);
        NoGil free;
        return row_int8_linear(x, w, scale, bias);
    });
}

// row_int8_product(codes, scale of the rows, weight, scale, bias or None, dtype code) -> y or None
PyObject *py_row_int8_product(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("row_int8_product", n, 6, [&] {
        const Args a{args, n};
        const Tensor &codes = a.tensor(0), &xs = a.tensor(1), &w = a.tensor(2), &scale = a.tensor(3);
        const Tensor bias = a.optional(4);
        const int dt = (int)a.integer(5);
        NoGil free;
        return row_int8_product(codes, xs, w, scale, bias, dt);
    });
}

// row_int8_experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, act) -> y or None
PyObject *py_row_int8_experts(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("row_int8_experts", n, 8, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &ids = a.tensor(1), &weight = a.tensor(2);
        const Tensor &gu = a.tensor(3), &gus = a.tensor(4), &d = a.tensor(5), &ds = a.tensor(6);
        const int act = (int)a.integer(7);
        NoGil free;
        return row_int8_experts(x, ids, weight, gu, gus, d, ds, act);
    });
}

RouteRule rule_of(const Args &a, Py_ssize_t first) { return {a.integer(first), a.truth(first + 1), a.truth(first + 2), a.number(first + 3)}; }

// route(x, router, bias or None, top_k, sigmoid, renormalize, factor) -> (weights, indices) or None
PyObject *py_route(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer_pair("route", n, 7, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &router = a.tensor(1);
        const Tensor bias = a.optional(2);
        const RouteRule rule = rule_of(a, 3);
        NoGil free;
        return route(x, router, bias, rule);
    });
}

// row_int8_moe(x, router, bias or None, top_k, sigmoid, renormalize, factor, gate_up, gate_up_scale, down, down_scale, act) -> y or None
PyObject *py_row_int8_moe(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("row_int8_moe", n, 12, [&] {
        const Args a{args, n};
        const Tensor &x = a.tensor(0), &router = a.tensor(1);
        const Tensor bias = a.optional(2);
        const RouteRule rule = rule_of(a, 3);
        const Tensor &gu = a.tensor(7), &gus = a.tensor(8), &d = a.tensor(9), &ds = a.tensor(10);
        const int act = (int)a.integer(11);
        NoGil free;
        return row_int8_moe(x, router, bias, rule, gu, gus, d, ds, act);
    });
}

// upload(host tensor, device index) -> the tensor on that GPU, or None; complete when it returns
PyObject *py_upload(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("upload", n, 2, [&] {
        const Args a{args, n};
        const Tensor &t = a.tensor(0);
        const auto index = (c10::DeviceIndex)a.integer(1);
        NoGil free;
        return upload(t, index);
    });
}

// download(tensor on a GPU) -> the tensor in host memory, or None
PyObject *py_download(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return answer("download", n, 1, [&] {
        const Args a{args, n};
        const Tensor &t = a.tensor(0);
        NoGil free;
        return download(t);
    });
}

// holds(parameter dicts, addresses): whether every dict's "weight" is a tensor whose data lies at the address (bytes of
// unsigned 64-bit numbers).  What ExpertWeights.check asks of each expert, 180 times for 60 experts: 0.3 us each in Python.
PyObject *py_holds(PyObject *, PyObject *const *args, Py_ssize_t n) {
    static PyObject *const weight = PyUnicode_InternFromString("weight");
    if (n != 2 || !PyTuple_Check(args[0]) || !PyBytes_Check(args[1]) ||
        PyBytes_GET_SIZE(args[1]) != PyTuple_GET_SIZE(args[0]) * (Py_ssize_t)sizeof(uint64_t)) {
        PyErr_SetString(PyExc_TypeError, "holds takes a tuple of dicts and as many addresses");
        return nullptr;
    }
    const uint64_t *want = (const uint64_t *)PyBytes_AS_STRING(args[1]);
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[0]); i++) {
        PyObject *d = PyTuple_GET_ITEM(args[0], i);
        PyObject *w = PyDict_Check(d) ? PyDict_GetItem(d, weight) : nullptr;
        if (!w || !THPVariable_Check(w)) Py_RETURN_FALSE;
        const Tensor &t = THPVariable_Unpack(w);
        if (!t.has_storage() || (uint64_t)(uintptr_t)t.const_data_ptr() != want[i]) Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(product), METHOD(linear), METHOD(linear_train), METHOD(gated), METHOD(embedding), METHOD(experts), METHOD(block_fp8_quantize),
                         METHOD(block_fp8_linear), METHOD(block_fp8_experts), METHOD(row_int8_quantize), METHOD(row_int8_linear), METHOD(row_int8_product),
                         METHOD(row_int8_experts), METHOD(route), METHOD(row_int8_moe),
                         METHOD(upload),
                         METHOD(download), METHOD(holds),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lowbit_torch", "native host path of the low-bit layers", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_lowbit_torch(void) { return PyModule_Create(&module); }
