"""Linear layers and experts whose two operands are 8-bit integers with a scale for each row.

The reference multiplies 8-bit weights by 16-bit activations (transformers/low_bit_linear.py:657-668), and so does LowBitLinear with
sym_int8, one scale per 32 weights.  Checkpoints made for products in 8-bit integers hold something else: row-major int8 codes `weight`
[N, K] and `weight_scale` [N] or [N, 1], what a row's codes are multiplied by, made for activations that are quantized too, with one scale
for each token.  Both operands then go through the int8 matrix pipes, whose sums are exact (csrc/row_int8.h has the formulas).  RowInt8Linear
and RowInt8Experts stand beside LowBitLinear and LowBitExperts; the conversion pass puts them in place of a checkpoint's layers, whose codes
they keep, or of dense layers with `optimize_model(model, "sym_int8", row_int8=True)`.

Weights are frozen, as in LowBitLinear.  The gradient flows on to the activations, whose quantization counts as the identity.
"""
import torch

import ipex_llm.ggml.model.llama.llama_cpp as ggml
from ipex_llm.transformers.native_ops import ops
from ipex_llm.utils.common import invalidInputError

MOST_K = 1 << 17                                             # of a row, so that sums of 127 * 127 fit 32 bits
_ACCEL = "cuda"
_FLOATS = {torch.float16: ggml.DT_F16, torch.bfloat16: ggml.DT_BF16, torch.float32: ggml.DT_F32}


def _check_gpu(x, what):
    invalidInputError(isinstance(x, torch.Tensor) and x.device.type == _ACCEL, f"{what} needs a tensor on an MI355X: "
                                                                               "the kernels have no CPU implementation")


def _check_input(x, what):
    _check_gpu(x, what)
    invalidInputError(x.dtype in _FLOATS, f"{what}: unsupported dtype {x.dtype}")


def _check_weight(w, scale, x, what, dim=2):
    invalidInputError(isinstance(w, torch.Tensor) and isinstance(scale, torch.Tensor) and w.device == x.device
                      and scale.device == x.device, f"{what}: the weight and its scales must be on x's GPU")
    invalidInputError(w.dtype == torch.int8 and scale.dtype == torch.float32, f"{what}: codes are int8, scales float32")
    invalidInputError(w.dim() == dim and w.numel() > 0 and scale.shape == w.shape[:-1],
                      f"{what}: a weight {tuple(w.shape)} has one scale for each row, not {tuple(scale.shape)}")
    invalidInputError(w.shape[-1] % 16 == 0 and w.shape[-1] <= MOST_K, f"{what}: in_features must be a multiple of 16, at most {MOST_K}")
    invalidInputError(w.is_contiguous() and scale.is_contiguous() and w.data_ptr() % 16 == 0,
                      f"{what}: weights and scales must be contiguous, codes from a 16-byte boundary on")
    invalidInputError(not (torch.is_grad_enabled() and scale.requires_grad), f"{what}: weights and scales are frozen")


def _check_bias(bias, n, x, what):
    invalidInputError(bias is None or (isinstance(bias, torch.Tensor) and bias.device == x.device and bias.shape == (n,)
                                       and bias.is_floating_point()), f"{what}: the bias must be [{n}] on x's GPU")


def _differentiable(t):
    return (t.requires_grad and torch.is_grad_enabled()) or torch.autograd.forward_ad.unpack_dual(t).tangent is not None


def row_int8_quantize(x: torch.Tensor):
    """(codes, scale) of x [.., K], activations by token or a weight by output channel: int8 codes in x's shape and float32 scales [..], one
    for each row.  scale = a / 127 and code = x * 127 / a to the nearest, ties to even, a the row's largest magnitude (2^-100 at least); a row
    that holds a NaN or an infinity has the scale NaN and codes of zero."""
    both = ops.row_int8_quantize(x) if isinstance(x, torch.Tensor) else None
    if both is not None:
        return both
    what = "row_int8_quantize"
    _check_input(x, what)
    invalidInputError(x.dim() >= 1 and x.shape[-1] % 16 == 0, f"{what}: rows must be a multiple of 16 long")
    if x.numel() == 0:
        return torch.empty(x.shape, dtype=torch.int8, device=x.device), torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    return _quantize_steps(x.detach())


def _quantize_steps(x):
    """The quantizer as torch operators, for a transform, a trace or a dispatch mode, which want to see them."""
    a = x.abs().amax(-1, keepdim=True).float().clamp(min=2.0 ** -100)
    bad = ~a.isfinite()
    codes = torch.round(x.double() * 127 / a.double()).masked_fill(bad, 0).to(torch.int8)
    # (by a tensor: a division by a number is a product with its reciprocal on the GPU, a unit off)
    return codes, (a / torch.full_like(a, 127.0)).masked_fill(bad, float("nan")).squeeze(-1)


def row_int8_dequantize(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.float32):
    """What row_int8_quantize made, as numbers; on any device."""
    invalidInputError(codes.dtype == torch.int8 and codes.dim() >= 1 and scale.shape == codes.shape[:-1],
                      "row_int8_dequantize: codes and scales do not fit together")
    return (codes.float() * scale.unsqueeze(-1)).to(dtype)


def row_int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor = None):
    """y = Q(x) W^T (+ bias) in x's dtype: x [.., K] is quantized by row, W = (weight, weight_scale) int8 [N, K] and float32 [N].

    The sums are whole numbers, exact; the two scales and the bias meet them in float32, and the result is rounded once.  Where x wants a gradient
    it is grad W, grad not quantized."""
    y = ops.row_int8_linear(x, weight, weight_scale, bias)
    if y is not None:
        return y
    what = "row_int8_linear"
    _check_input(x, what)
    _check_weight(weight, weight_scale, x, what)
    n, k = weight.shape
    invalidInputError(x.dim() >= 1 and x.shape[-1] == k, f"{what}: x has rows of {x.shape[-1] if x.dim() else 0} values, the weight of {k}")
    _check_bias(bias, n, x, what)
    if x.numel() == 0:
        return x.new_empty((*x.shape[:-1], n)) + x.sum() * 0
    if bias is not None and bias.dtype == x.dtype:           # strided, or one that wants a gradient itself
        fixed = bias.detach().contiguous()
        y = ops.row_int8_linear(x, weight, weight_scale, fixed)
        if y is not None:
            # (a zero that carries the gradient; an infinity among the bias would make it a NaN)
            return y + (bias - fixed).nan_to_num() if _differentiable(bias) else y
    elif bias is not None:                                   # of another dtype: added before the result is rounded
        y = ops.row_int8_linear(x.float(), weight, weight_scale, None)
        if y is not None:
            return (y + bias).to(x.dtype)
    # a tangent, a transform or a dispatch mode wants to see the operators
    with torch.no_grad():
        values = row_int8_dequantize(*_quantize_steps(x))
        dense = row_int8_dequantize(weight, weight_scale)
    xf = x.float()
    y = torch.matmul(xf + (values - xf).detach(), dense.t())
    return (y if bias is None else y + bias).to(x.dtype)


def row_int8_product(codes: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor = None,
                     dtype=torch.bfloat16):
    """row_int8_linear of rows that row_int8_quantize has quantized already, codes [.., K] and scale [..], in `dtype`: for activations that meet
    several weights.  No gradient flows on."""
    what = "row_int8_product"
    invalidInputError(dtype in _FLOATS, f"{what}: unsupported dtype {dtype}")
    y = ops.row_int8_product(codes, scale, weight, weight_scale, bias, _FLOATS[dtype])
    if y is not None:
        return y
    _check_gpu(codes, what)
    _check_weight(weight, weight_scale, codes, what)
    n, k = weight.shape
    invalidInputError(codes.dtype == torch.int8 and codes.dim() >= 1 and codes.shape[-1] == k and isinstance(scale, torch.Tensor)
                      and scale.dtype == torch.float32 and scale.device == codes.device and scale.shape == codes.shape[:-1],
                      f"{what}: int8 codes [.., {k}] and a float32 scale for each row of them")
    _check_bias(bias, n, codes, what)
    invalidInputError(not _differentiable(scale), f"{what}: no gradient flows through the codes and scales (row_int8_linear's does)")
    if codes.numel() == 0:
        return torch.empty((*codes.shape[:-1], n), dtype=dtype, device=codes.device)
    if bias is not None:                                     # of another dtype, strided, or one that wants a gradient
        y = ops.row_int8_product(codes, scale, weight, weight_scale, None, ggml.DT_F32)
        if y is not None:
            return (y + bias).to(dtype)
    y = torch.matmul(codes.float(), weight.float().t()) * scale.unsqueeze(-1) * weight_scale
    return (y if bias is None else y + bias).to(dtype)
