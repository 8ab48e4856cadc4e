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
import torch.nn.functional as F
from torch import nn

import ipex_llm.ggml.model.llama.llama_cpp as ggml
from ipex_llm.transformers.block_fp8 import _frozen, _gated, _KeepsFormat
from ipex_llm.transformers.native_ops import ops
from ipex_llm.utils.common import invalidInputError

MOST_K = 1 << 17                                             # of a row, so that sums of 127 * 128 fit 32 bits
_ACCEL = "cuda"
_FLOATS = {torch.float16: ggml.DT_F16, torch.bfloat16: ggml.DT_BF16, torch.float32: ggml.DT_F32}


def _check_gpu(x, what):
    invalidInputError(isinstance(x, torch.Tensor) and x.device.type == _ACCEL, f"{what} needs a tensor on an MI355X: "
                                                                               "the kernels have no CPU implementation")


def _check_input(x, what):
    _check_gpu(x, what)
    invalidInputError(x.dtype in _FLOATS, f"{what}: unsupported dtype {x.dtype}")


def _as_the_kernels_read(w, scale):
    try:
        start = w.data_ptr()
    except RuntimeError:                                     # (a transform's or a trace's tensor, which has no storage and meets torch operators)
        return True
    return w.is_contiguous() and scale.is_contiguous() and start % 16 == 0


def _check_weight(w, scale, x, what, dim=2):
    invalidInputError(isinstance(w, torch.Tensor) and isinstance(scale, torch.Tensor) and w.device == x.device
                      and scale.device == x.device, f"{what}: the weight and its scales must be on x's GPU")
    invalidInputError(w.dtype == torch.int8 and scale.dtype == torch.float32, f"{what}: codes are int8, scales float32")
    invalidInputError(w.dim() == dim and w.numel() > 0 and scale.shape == w.shape[:-1],
                      f"{what}: a weight {tuple(w.shape)} has one scale for each row, not {tuple(scale.shape)}")
    invalidInputError(w.shape[-1] % 16 == 0 and w.shape[-1] <= MOST_K, f"{what}: in_features must be a multiple of 16, at most {MOST_K}")
    invalidInputError(_as_the_kernels_read(w, scale),
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
        y = x.new_empty((*x.shape[:-1], n)) + x.sum()        # (carries the gradients)
        return y if bias is None else y + bias[:0].sum().to(x.dtype)
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


def _expert_loop(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, gate):
    """Expert by expert, h = gate(g | u), with what the native call keeps in float32 (g, u, h, the pairs' results and their sum) kept so too, and
    one rounding."""
    (tokens, top_k), n_exp = top_k_index.shape, gate_up.shape[0]
    expert = top_k_index.reshape(-1).long()
    expert = expert.masked_fill((expert < 0) | (expert >= n_exp), n_exp)
    order = expert.argsort(stable=True)
    counts = torch.bincount(expert, minlength=n_exp + 1).tolist()
    rows, ys = x.float()[torch.div(order, top_k, rounding_mode="floor")].split(counts), []
    for e in range(n_exp):
        if counts[e]:
            gu = row_int8_linear(rows[e], gate_up[e], gate_up_scale[e])
            ys.append(row_int8_linear(gate(gu), down[e], down_scale[e]))
    if not ys:
        return torch.zeros_like(x) + (x[:0].sum() + top_k_weights[:0].sum().to(x.dtype))       # (zeros that carry the gradients)
    order = order[:len(order) - counts[n_exp]]
    y = torch.cat(ys) * top_k_weights.reshape(-1)[order].float().unsqueeze(-1)
    return y.new_zeros((tokens * top_k, x.shape[1])).index_copy(0, order, y).view(tokens, top_k, -1).sum(1).to(x.dtype)


_ACTS = {0: F.silu, 1: lambda g: F.gelu(g, approximate="tanh")}


def _check_experts(x, gate_up, gate_up_scale, down, down_scale, what):
    _check_input(x, what)
    _check_weight(gate_up, gate_up_scale, x, what, 3)
    _check_weight(down, down_scale, x, what, 3)
    n_exp, two_i, hidden = gate_up.shape
    invalidInputError(two_i % 2 == 0 and tuple(down.shape) == (n_exp, hidden, two_i // 2),
                      f"{what}: gate_up [E, 2 I, H] and down [E, H, I] do not fit together")
    invalidInputError(x.dim() == 2 and x.shape[1] == hidden, f"{what}: x must be [tokens, {hidden}]")


def row_int8_experts(x: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor, gate_up: torch.Tensor,
                     gate_up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor, act: int = 0):
    """The experts of a mixture-of-experts block: out[t] = sum_j p[t, j] (Q(act(g) u) down[e]^T), (g | u) = Q(x[t]) gate_up[e]^T,
    e = top_k_index[t, j], p = top_k_weights.

    x [T, H]; top_k_index, top_k_weights [T, k]; gate_up [E, 2 I, H] (gate rows first) and down [E, H, I] codes with their scales [E, 2 I] and
    [E, H]; act 0 = SiLU, 1 = GELU (tanh form).  An index that names no expert counts nothing.  act(g) u, the pairs' results and their sum are float32,
    rounded once.  One native call; x or weights that want a gradient, and more than 64 experts per token, 4096 experts or 2^21 pairs, run
    expert by expert through row_int8_linear."""
    invalidInputError(act in _ACTS, "row_int8_experts: act is 0 (SiLU) or 1 (GELU, tanh form)")
    y = ops.row_int8_experts(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, act)
    if y is not None:
        return y
    what = "row_int8_experts"
    _check_experts(x, gate_up, gate_up_scale, down, down_scale, what)
    invalidInputError(top_k_index.dim() == 2 and top_k_index.shape == top_k_weights.shape and top_k_index.shape[0] == x.shape[0]
                      and not top_k_index.is_floating_point() and top_k_index.dtype != torch.bool
                      and top_k_index.device == x.device and top_k_weights.device == x.device,
                      f"{what}: whole indices and weights [tokens, k] on x's GPU")
    return _expert_loop(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, _gated(_ACTS[act]))


def row_int8_moe(x: torch.Tensor, router: torch.Tensor, top_k: int, gate_up: torch.Tensor, gate_up_scale: torch.Tensor, down: torch.Tensor,
                 down_scale: torch.Tensor, bias: torch.Tensor = None, score: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                 act: int = 0):
    """A whole mixture-of-experts layer, moe.moe_route and row_int8_experts in one native call: x [T, H], router [E, H] (bias, score, renormalize
    and scale are the router's), the experts' codes and scales as in row_int8_experts.  Where x or the router want a gradient it is the two calls."""
    from ipex_llm.transformers.moe import _SCORES, _check_route, moe_route
    what = "row_int8_moe"
    invalidInputError(act in _ACTS, f"{what}: act is 0 (SiLU) or 1 (GELU, tanh form)")
    invalidInputError(score in _SCORES, f"{what}: score is 'softmax' or 'sigmoid', not {score!r}")
    fixed = bias.float() if isinstance(bias, torch.Tensor) and bias.is_floating_point() else bias
    y = ops.row_int8_moe(x, router, fixed, top_k, _SCORES[score], renormalize, float(scale), gate_up, gate_up_scale, down, down_scale, act)
    if y is not None:
        return y
    _check_experts(x, gate_up, gate_up_scale, down, down_scale, what)
    _check_route(x, router, top_k, bias, score, what)
    invalidInputError(router.shape[0] == gate_up.shape[0], f"{what}: the router has {router.shape[0]} rows for {gate_up.shape[0]} experts")
    if x.numel() == 0:
        return x + router[:0].sum().to(x.dtype)              # (carries the gradients)
    weights, index = moe_route(x, router, top_k, bias, score, renormalize, scale)
    return row_int8_experts(x, index, weights, gate_up, gate_up_scale, down, down_scale, act)


def _pack_weight(w, shape_only=False):
    """Codes and scales of a dense weight on any device; a host weight is quantized on the GPU."""
    if shape_only or w.device.type == "meta":
        return torch.empty(w.shape, dtype=torch.int8, device=w.device), torch.empty(w.shape[:-1], dtype=torch.float32, device=w.device)
    from ipex_llm.transformers.low_bit_linear import _require_gpu, _to_gpu
    if w.device.type == _ACCEL:
        return row_int8_quantize(w.detach())
    _require_gpu("row_int8_quantize")
    codes, scale = row_int8_quantize(_to_gpu(w.detach().contiguous()))
    return codes.to(w.device), scale.to(w.device)


def _taken(module, name, shape_only):
    """(codes, scale) of a module's weight: its own where it holds `<name>_scale`, [.., N] or [.., N, 1]; else the dense weight's."""
    w, scale = getattr(module, name).data, getattr(module, name + "_scale", None)
    if scale is None:
        return _pack_weight(w, shape_only)
    scale = scale.data.to(torch.float32)
    scale = scale.squeeze(-1) if scale.dim() == w.dim() and scale.shape[-1] == 1 else scale
    invalidInputError(w.dtype == torch.int8 and scale.shape == w.shape[:-1],
                      f"row-scaled int8 {name} {tuple(w.shape)} has one scale for each row, not {tuple(scale.shape)}")
    # (the kernels load sixteen codes at once: a view that starts between two such groups is copied)
    w = w.contiguous()
    return (w.clone() if w.device.type != "meta" and w.data_ptr() % 16 else w), scale.contiguous()


class RowInt8Linear(_KeepsFormat, nn.Linear):
    """nn.Linear with an int8 weight and a scale for each of its rows (`weight`, `weight_scale`) and activations quantized by row in the call."""

    _FORMAT = ("weight", "weight_scale")

    def __init__(self, input_features, output_features, bias=True, mp_group=None, optimize_lm_head=False):
        with torch.device("meta"):
            super().__init__(input_features, output_features, bias)
        invalidInputError(input_features % 16 == 0 and input_features <= MOST_K,
                          f"RowInt8Linear needs in_features to be a multiple of 16, at most {MOST_K}")
        self.weight = _frozen(torch.empty((output_features, input_features), dtype=torch.int8))
        self.weight_scale = _frozen(torch.empty(output_features, dtype=torch.float32))
        if bias:
            self.bias = _frozen(torch.zeros(output_features))
        self.in_len, self.out_len = input_features, output_features
        self.weight_shape = (output_features, input_features)
        self.mp_group = mp_group
        self.compute_dtype = None                        # only for training
        self.optimize_lm_head = optimize_lm_head

    @classmethod
    def from_linear(cls, linear, convert_shape_only=False, mp_group=None, optimize_lm_head=False):
        """From an nn.Linear: a dense one is quantized; one that holds `weight_scale` keeps its codes and scales."""
        w, scale = _taken(linear, "weight", convert_shape_only)
        with torch.device("meta"):
            new = cls(w.shape[1], w.shape[0], False, mp_group, optimize_lm_head)
        new.weight, new.weight_scale = _frozen(w), _frozen(scale)
        new.bias = None if linear.bias is None else _frozen(linear.bias.data)
        return new.train(linear.training)

    def forward(self, x: torch.Tensor):
        invalidInputError(self.mp_group is None, "mp_group (tensor parallel all-reduce) is outside this single-GPU build")
        if self.optimize_lm_head:
            from ipex_llm.transformers.low_bit_linear import reshape_lm_head_input
            x = reshape_lm_head_input(x)
        given = x.dtype
        if self.training and not torch.is_inference_mode_enabled() and self.compute_dtype is not None:
            x = x.to(self.compute_dtype)
        # (in x's type for this call only: the bias stays as it was given)
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        y = row_int8_linear(x, self.weight, self.weight_scale, bias)
        return y if y.dtype == given else y.to(given)

    def dequantize(self, dtype=torch.float32):
        return row_int8_dequantize(self.weight.data, self.weight_scale.data, dtype)


class RowInt8Experts(_KeepsFormat):
    """The experts of a sparse mixture-of-experts block in row-scaled int8: takes the place of a module that holds `gate_up_proj` [E, 2 I, H]
    and `down_proj` [E, H, I] (moe.LowBitExperts has the call)."""

    _FORMAT = ("gate_up_proj", "gate_up_proj_scale", "down_proj", "down_proj_scale")

    def __init__(self, num_experts, hidden_dim, intermediate_dim, act_fn):
        super().__init__()
        invalidInputError(hidden_dim % 16 == 0 and intermediate_dim % 16 == 0 and max(hidden_dim, intermediate_dim) <= MOST_K,
                          f"RowInt8Experts needs hidden_dim and intermediate_dim to be multiples of 16, at most {MOST_K}")
        self.num_experts, self.hidden_dim, self.intermediate_dim, self.act_fn = num_experts, hidden_dim, intermediate_dim, act_fn
        self.own_gate = None                             # h of (g | u), where it is not act_fn(g) * u (moe.gate_of)
        for name, n, k in (("gate_up_proj", 2 * intermediate_dim, hidden_dim), ("down_proj", hidden_dim, intermediate_dim)):
            setattr(self, name, _frozen(torch.empty((num_experts, n, k), dtype=torch.int8)))
            setattr(self, name + "_scale", _frozen(torch.empty((num_experts, n), dtype=torch.float32)))

    @classmethod
    def from_fused(cls, module, convert_shape_only=False):
        """From a module with dense or row-scaled `gate_up_proj` and `down_proj` and an `act_fn`, or a gate of its own, which is kept."""
        n_exp, two_i, hidden = module.gate_up_proj.shape
        invalidInputError(tuple(module.down_proj.shape) == (n_exp, hidden, two_i // 2), "gate_up_proj / down_proj shapes do not fit together")
        from ipex_llm.transformers.moe import gate_of
        known, gate = gate_of(module)
        invalidInputError(known, "the experts' gate depends on tensors of the module, which its row-scaled form does not have")
        with torch.device("meta"):
            new = cls(n_exp, hidden, two_i // 2, module.act_fn)
        new.own_gate = gate
        for name in ("gate_up_proj", "down_proj"):
            w, scale = _taken(module, name, convert_shape_only)
            setattr(new, name, _frozen(w))
            setattr(new, name + "_scale", _frozen(scale))
        return new.train(module.training)

    def forward(self, hidden_states, top_k_index, top_k_weights):
        from ipex_llm.transformers.moe import activation_code
        if top_k_index.shape[0] == 0:
            return torch.zeros_like(hidden_states) + (hidden_states[:0].sum() + top_k_weights[:0].sum().to(hidden_states.dtype))
        weights = (self.gate_up_proj, self.gate_up_proj_scale, self.down_proj, self.down_proj_scale)
        act = activation_code(self.act_fn)
        if act is None or self.own_gate is not None:
            return _expert_loop(hidden_states, top_k_index, top_k_weights, *weights, self.own_gate or _gated(self.act_fn))
        return row_int8_experts(hidden_states, top_k_index, top_k_weights, *weights, act)
