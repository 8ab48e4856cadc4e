"""Linear layers and experts whose two operands are e4m3 with a scale for each block of 128.

The reference multiplies fp8 weights by 16-bit activations (transformers/low_bit_linear.py:657-668), and so does LowBitLinear
with fp8_e4m3, one scale per 128 weights of a row.  Block-scaled checkpoints hold something else: row-major e4m3 codes `weight`
[N, K] and `weight_scale_inv` [ceil(N / 128), ceil(K / 128)], what a 128 x 128 block's codes are multiplied by, made for
activations that are quantized too, by row with one scale for each 128 values.  Both operands then go through the fp8 matrix pipes
(csrc/block_fp8.h has the formulas).  BlockFP8Linear and BlockFP8Experts stand beside LowBitLinear and LowBitExperts; the
conversion pass puts them in place of a checkpoint's block-scaled layers, whose codes they keep, or of dense layers with
`optimize_model(model, "fp8_e4m3", block_fp8=True)`.

Weights are frozen, as in LowBitLinear.  The gradient flows on to the activations, whose quantization counts as the identity.
"""
import torch
import torch.nn.functional as F
from torch import nn

import ipex_llm.ggml.model.llama.llama_cpp as ggml
from ipex_llm.transformers.native_ops import ops
from ipex_llm.utils.common import invalidInputError

E4M3 = torch.float8_e4m3fn
BLOCK = 128
_ACCEL = "cuda"
_FLOATS = {torch.float16: ggml.DT_F16, torch.bfloat16: ggml.DT_BF16, torch.float32: ggml.DT_F32}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _check_input(x, what):
    invalidInputError(isinstance(x, torch.Tensor) and x.device.type == _ACCEL, f"{what} needs a tensor on an MI355X: "
                                                                               "the kernels have no CPU implementation")
    invalidInputError(x.dtype in _FLOATS, f"{what}: unsupported dtype {x.dtype}")


def _check_weight(w, scale, x, what, dim=2):
    invalidInputError(isinstance(w, torch.Tensor) and isinstance(scale, torch.Tensor) and w.device == x.device
                      and scale.device == x.device, f"{what}: the weight and its scales must be on x's GPU")
    invalidInputError(w.dtype == E4M3 and scale.dtype == torch.float32, f"{what}: codes are float8_e4m3fn, scales float32")
    invalidInputError(w.dim() == dim and scale.dim() == dim and w.numel() > 0 and w.shape[:-2] == scale.shape[:-2]
                      and tuple(scale.shape[-2:]) == (_blocks(w.shape[-2]), _blocks(w.shape[-1])),
                      f"{what}: a weight {tuple(w.shape)} has one scale for each block of 128 x 128, not {tuple(scale.shape)}")
    invalidInputError(w.shape[-1] % 16 == 0, f"{what}: in_features must be a multiple of 16")
    invalidInputError(w.is_contiguous() and scale.is_contiguous() and w.data_ptr() % 16 == 0,
                      f"{what}: weights and scales must be contiguous, codes from a 16-byte boundary on")
    invalidInputError(not (torch.is_grad_enabled() and (w.requires_grad or scale.requires_grad)), f"{what}: weights and scales are frozen")


def _differentiable(t):
    return (t.requires_grad and torch.is_grad_enabled()) or torch.autograd.forward_ad.unpack_dual(t).tangent is not None


def _quantized(x, weight, what):
    _check_input(x, what)
    invalidInputError(x.dim() >= (2 if weight else 1) and x.shape[-1] % 16 == 0, f"{what}: rows must be a multiple of 16 long")
    if x.numel() == 0:
        shape = list(x.shape)
        shape[-1] = _blocks(shape[-1])
        if weight:
            shape[-2] = _blocks(shape[-2])
        return torch.empty(x.shape, dtype=E4M3, device=x.device), torch.empty(shape, dtype=torch.float32, device=x.device)
    both = ops.block_fp8_quantize(x, weight)
    return _quantize_steps(x.detach(), weight) if both is None else both


def _spread(scale, shape, weight):
    """One scale for each value of [.., R, K]."""
    s = scale.repeat_interleave(BLOCK, dim=-1)[..., :shape[-1]]
    return s.repeat_interleave(BLOCK, dim=-2)[..., :shape[-2], :] if weight else s


def _quantize_steps(x, weight):
    """The quantizers as torch operators, for a transform, a trace or a dispatch mode, which want to see them.  The quotient is rounded from
    float64 to float32 and then to a code, as the kernels do."""
    pad = F.pad(x.abs(), (0, -x.shape[-1] % BLOCK, 0, -x.shape[-2] % BLOCK) if weight else (0, -x.shape[-1] % BLOCK))
    a = pad.unflatten(-1, (-1, BLOCK)).amax(-1)
    a = (a.unflatten(-2, (-1, BLOCK)).amax(-2) if weight else a).float().clamp(min=2.0 ** -100)
    # (by a tensor: a division by a number is a product with its reciprocal on the GPU, a unit off)
    return (x.double() * 448 / _spread(a, x.shape, weight).double()).float().to(E4M3), a / torch.full_like(a, 448.0)


def block_fp8_quantize(x: torch.Tensor):
    """(codes, scale) of activations x [.., K]: e4m3 codes in x's shape and float32 scales [.., ceil(K / 128)], one for each 128 values
    of a row.  scale = a / 448 and code = e4m3(x * 448 / a), a the block's largest magnitude (2^-100 at least)."""
    return _quantized(x, False, "block_fp8_quantize")


def block_fp8_quantize_weight(w: torch.Tensor):
    """(codes, scale) of one weight [N, K] or several [.., N, K]: scales [.., ceil(N / 128), ceil(K / 128)], one for each 128 x 128."""
    return _quantized(w, True, "block_fp8_quantize_weight")


def block_fp8_dequantize(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.float32):
    """What block_fp8_quantize (scale [.., R, ceil(K / 128)]) or block_fp8_quantize_weight made, as numbers; on any device."""
    invalidInputError(codes.dtype == E4M3 and codes.dim() == scale.dim() and scale.shape[-1] == _blocks(codes.shape[-1]),
                      "block_fp8_dequantize: codes and scales do not fit together")
    weight = codes.dim() > 1 and scale.shape[-2] != codes.shape[-2]
    invalidInputError(not weight or scale.shape[-2] == _blocks(codes.shape[-2]), "block_fp8_dequantize: codes and scales do not fit together")
    return (codes.float() * _spread(scale, codes.shape, weight)).to(dtype)


def block_fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor = None):
    """y = Q(x) W^T (+ bias) in x's dtype: x [.., K] is quantized by row, W = (weight, weight_scale) [N, K] in blocks of 128 x 128.

    float16 and bfloat16: sums in float32 of products on the fp8 matrix pipes, which drop what lies 13 bits below the largest of a few
    neighbouring products (1e-5 to 5e-5 of the norm of activations times weights; where large terms cancel, of the terms); float32: exact
    products, which 16-bit rows have as `block_fp8_linear(x.float(), ..).to(x.dtype)`.  The result, with its bias, is rounded once.  Where
    x wants a gradient it is grad W, grad not quantized."""
    y = ops.block_fp8_linear(x, weight, weight_scale, bias, -1)
    if y is not None:
        return y
    what = "block_fp8_linear"
    _check_input(x, what)
    _check_weight(weight, weight_scale, x, what)
    n, k = weight.shape
    invalidInputError(x.dim() >= 1 and x.shape[-1] == k, f"{what}: x has rows of {x.shape[-1] if x.dim() else 0} values, the weight of {k}")
    invalidInputError(bias is None or (bias.device == x.device and bias.shape == (n,)), f"{what}: the bias must be [{n}] on x's GPU")
    if x.numel() == 0:
        return x.new_empty((*x.shape[:-1], n)) + x.sum() * 0
    if bias is not None and bias.dtype == x.dtype:           # strided, or one that wants a gradient itself
        fixed = bias.detach().contiguous()
        y = ops.block_fp8_linear(x, weight, weight_scale, fixed, -1)
        if y is not None:
            # (a zero that carries the gradient; an infinity among the bias would make it a NaN)
            return y + (bias - fixed).nan_to_num() if _differentiable(bias) else y
    elif bias is not None:                                   # of another dtype: added before the result is rounded
        y = ops.block_fp8_linear(x.float(), weight, weight_scale, None, _FLOATS[x.dtype])
        if y is not None:
            return (y + bias).to(x.dtype)
    # a tangent, a transform or a dispatch mode wants to see the operators
    with torch.no_grad():
        values = block_fp8_dequantize(*_quantize_steps(x, False))
        dense = block_fp8_dequantize(weight, weight_scale)
    xf = x.float()
    y = torch.matmul(xf + (values - xf).detach(), dense.t())
    return (y if bias is None else y + bias).to(x.dtype)


def _exact_product(x, weight, scale, grad_dtype):
    """The product of float32 rows; where they want a gradient, it is multiplied in `grad_dtype`."""
    y = ops.block_fp8_linear(x, weight, scale, None, _FLOATS[grad_dtype])
    return block_fp8_linear(x, weight, scale) if y is None else y


def _expert_loop(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, gate):
    """Expert by expert, h = gate(g | u), with what the native call keeps in float32 (g, u, h, the pairs' results and their sum) kept so too, and
    one rounding.  Where a gradient is wanted below 16-bit rows, the products of the backward take it in their type."""
    (tokens, top_k), n_exp = top_k_index.shape, gate_up.shape[0]
    expert = top_k_index.reshape(-1).long()
    expert = expert.masked_fill((expert < 0) | (expert >= n_exp), n_exp)
    order = expert.argsort(stable=True)
    counts = torch.bincount(expert, minlength=n_exp + 1).tolist()
    rows, ys = x.float()[torch.div(order, top_k, rounding_mode="floor")].split(counts), []
    for e in range(n_exp):
        if counts[e]:
            gu = _exact_product(rows[e], gate_up[e], gate_up_scale[e], x.dtype)
            ys.append(_exact_product(gate(gu), down[e], down_scale[e], x.dtype))
    if not ys:
        return torch.zeros_like(x)
    order = order[:len(order) - counts[n_exp]]
    y = torch.cat(ys) * top_k_weights.reshape(-1)[order].float().unsqueeze(-1)
    return y.new_zeros((tokens * top_k, x.shape[1])).index_copy(0, order, y).view(tokens, top_k, -1).sum(1).to(x.dtype)


def _gated(act_fn):
    def gate(gu):
        g, u = gu.chunk(2, dim=-1)
        return act_fn(g) * u
    return gate


_ACTS = {0: F.silu, 1: lambda g: F.gelu(g, approximate="tanh")}


def block_fp8_experts(x: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor, gate_up: torch.Tensor,
                      gate_up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor, act: int = 0):
    """The experts of a mixture-of-experts block: out[t] = sum_j p[t, j] (Q(act(g) u) down[e]^T), (g | u) = Q(x[t]) gate_up[e]^T,
    e = top_k_index[t, j], p = top_k_weights.

    x [T, H]; top_k_index, top_k_weights [T, k]; gate_up [E, 2 I, H] (gate rows first) and down [E, H, I] codes with their scales, I a
    multiple of 128; act 0 = SiLU, 1 = GELU (tanh form).  An index that names no expert counts nothing.  act(g) u, the pairs' results and
    their sum are float32, rounded once.  One native call in float16 and bfloat16; float32, x or weights that want a gradient, and more
    than 64 experts per token, 4096 experts or 2^21 pairs, run expert by expert through block_fp8_linear."""
    invalidInputError(act in _ACTS, "block_fp8_experts: act is 0 (SiLU) or 1 (GELU, tanh form)")
    y = ops.block_fp8_experts(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, act)
    if y is not None:
        return y
    what = "block_fp8_experts"
    _check_input(x, what)
    _check_weight(gate_up, gate_up_scale, x, what, 3)
    _check_weight(down, down_scale, x, what, 3)
    n_exp, two_i, hidden = gate_up.shape
    invalidInputError(two_i % 256 == 0 and tuple(down.shape) == (n_exp, hidden, two_i // 2),
                      f"{what}: gate_up [E, 2 I, H] and down [E, H, I] do not fit together (I a multiple of 128)")
    invalidInputError(x.dim() == 2 and x.shape[1] == hidden, f"{what}: x must be [tokens, {hidden}]")
    invalidInputError(top_k_index.dim() == 2 and top_k_index.shape == top_k_weights.shape and top_k_index.shape[0] == x.shape[0]
                      and not top_k_index.is_floating_point() and top_k_index.dtype != torch.bool
                      and top_k_index.device == x.device and top_k_weights.device == x.device,
                      f"{what}: whole indices and weights [tokens, k] on x's GPU")
    return _expert_loop(x, top_k_index, top_k_weights, gate_up, gate_up_scale, down, down_scale, _gated(_ACTS[act]))


class _KeepsFormat(nn.Module):
    """Codes stay e4m3 and scales float32 whatever dtype the rest of a model is moved to."""

    _FORMAT = ()

    def _apply(self, fn, recurse=True):
        keep = {id(self._parameters[n]) for n in self._FORMAT if self._parameters.get(n) is not None}

        def moved(t):
            out = fn(t)
            return t.to(out.device) if id(t) in keep and out.dtype != t.dtype else out
        return super()._apply(moved, recurse)


def _frozen(t):
    return nn.Parameter(t, requires_grad=False)


def _pack_weight(w, shape_only=False):
    """Codes and scales of a dense weight on any device; a host weight is quantized on the GPU."""
    if shape_only or w.device.type == "meta":
        return (torch.empty(w.shape, dtype=E4M3, device=w.device),
                torch.empty((*w.shape[:-2], _blocks(w.shape[-2]), _blocks(w.shape[-1])), dtype=torch.float32, device=w.device))
    from ipex_llm.transformers.low_bit_linear import _require_gpu, _to_gpu
    if w.device.type == _ACCEL:
        return block_fp8_quantize_weight(w.detach())
    _require_gpu("block_fp8_quantize_weight")
    codes, scale = block_fp8_quantize_weight(_to_gpu(w.detach().contiguous()))
    return codes.to(w.device), scale.to(w.device)


class BlockFP8Linear(_KeepsFormat, nn.Linear):
    """nn.Linear with a block-scaled e4m3 weight (`weight`, `weight_scale_inv`) and activations quantized in the call."""

    _FORMAT = ("weight", "weight_scale_inv")

    def __init__(self, input_features, output_features, bias=True, mp_group=None, optimize_lm_head=False):
        with torch.device("meta"):
            super().__init__(input_features, output_features, bias)
        invalidInputError(input_features % 16 == 0, "BlockFP8Linear needs in_features to be a multiple of 16")
        self.weight = _frozen(torch.empty((output_features, input_features), dtype=E4M3))
        self.weight_scale_inv = _frozen(torch.empty((_blocks(output_features), _blocks(input_features)), dtype=torch.float32))
        if bias:
            self.bias = _frozen(torch.zeros(output_features))
        self.in_len, self.out_len = input_features, output_features
        self.weight_shape = (output_features, input_features)
        self.mp_group = mp_group
        self.compute_dtype = None                        # only for training
        self.optimize_lm_head = optimize_lm_head

    @classmethod
    def from_linear(cls, linear, convert_shape_only=False, mp_group=None, optimize_lm_head=False):
        """From an nn.Linear: a dense one is quantized; one that holds `weight_scale_inv` keeps its codes and scales."""
        w, scale = linear.weight.data, getattr(linear, "weight_scale_inv", None)
        if scale is None:
            w, scale = _pack_weight(w, convert_shape_only)
        else:
            scale = scale.data.to(torch.float32)
            invalidInputError(w.dtype == E4M3 and tuple(scale.shape) == (_blocks(w.shape[0]), _blocks(w.shape[1])),
                              f"a block-scaled weight {tuple(w.shape)} has one scale for each block of 128 x 128, not {tuple(scale.shape)}")
        with torch.device("meta"):
            new = cls(w.shape[1], w.shape[0], False, mp_group, optimize_lm_head)
        new.weight, new.weight_scale_inv = _frozen(w.contiguous()), _frozen(scale.contiguous())
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
        if self.bias is not None and self.bias.dtype != x.dtype:
            self.bias.data = self.bias.data.to(x.dtype)
        y = block_fp8_linear(x, self.weight, self.weight_scale_inv, self.bias)
        return y if y.dtype == given else y.to(given)

    def dequantize(self, dtype=torch.float32):
        return block_fp8_dequantize(self.weight.data, self.weight_scale_inv.data, dtype)


class BlockFP8Experts(_KeepsFormat):
    """The experts of a sparse mixture-of-experts block with block-scaled weights: takes the place of a module that holds
    `gate_up_proj` [E, 2 I, H] and `down_proj` [E, H, I] (moe.LowBitExperts has the call)."""

    _FORMAT = ("gate_up_proj", "gate_up_proj_scale_inv", "down_proj", "down_proj_scale_inv")

    def __init__(self, num_experts, hidden_dim, intermediate_dim, act_fn):
        super().__init__()
        invalidInputError(hidden_dim % 16 == 0 and intermediate_dim % BLOCK == 0,
                          "BlockFP8Experts needs hidden_dim to be a multiple of 16 and intermediate_dim of 128")
        self.num_experts, self.hidden_dim, self.intermediate_dim, self.act_fn = num_experts, hidden_dim, intermediate_dim, act_fn
        self.own_gate = None                             # h of (g | u), where it is not act_fn(g) * u (moe.gate_of)
        for name, n, k in (("gate_up_proj", 2 * intermediate_dim, hidden_dim), ("down_proj", hidden_dim, intermediate_dim)):
            setattr(self, name, _frozen(torch.empty((num_experts, n, k), dtype=E4M3)))
            setattr(self, name + "_scale_inv", _frozen(torch.empty((num_experts, _blocks(n), _blocks(k)), dtype=torch.float32)))

    @classmethod
    def from_fused(cls, module, convert_shape_only=False):
        """From a module with dense or block-scaled `gate_up_proj` and `down_proj` and an `act_fn`, or a gate of its own, which is kept."""
        n_exp, two_i, hidden = module.gate_up_proj.shape
        invalidInputError(tuple(module.down_proj.shape) == (n_exp, hidden, two_i // 2), "gate_up_proj / down_proj shapes do not fit together")
        from ipex_llm.transformers.moe import gate_of
        known, gate = gate_of(module)
        invalidInputError(known, "the experts' gate depends on tensors of the module, which its block-scaled form does not have")
        with torch.device("meta"):
            new = cls(n_exp, hidden, two_i // 2, module.act_fn)
        new.own_gate = gate
        for name in ("gate_up_proj", "down_proj"):
            w, scale = getattr(module, name).data, getattr(module, name + "_scale_inv", None)
            if scale is None:
                w, scale = _pack_weight(w, convert_shape_only)
            else:
                scale = scale.data.to(torch.float32)
            invalidInputError(w.dtype == E4M3 and tuple(scale.shape) == (n_exp, _blocks(w.shape[1]), _blocks(w.shape[2])),
                              f"{name}: one scale for each block of 128 x 128 of each expert, not {tuple(scale.shape)}")
            setattr(new, name, _frozen(w.contiguous()))
            setattr(new, name + "_scale_inv", _frozen(scale.contiguous()))
        return new.train(module.training)

    def forward(self, hidden_states, top_k_index, top_k_weights):
        from ipex_llm.transformers.moe import activation_code
        if top_k_index.shape[0] == 0:
            return torch.zeros_like(hidden_states)
        weights = (self.gate_up_proj, self.gate_up_proj_scale_inv, self.down_proj, self.down_proj_scale_inv)
        act = activation_code(self.act_fn)
        if act is None or self.own_gate is not None:
            return _expert_loop(hidden_states, top_k_index, top_k_weights, *weights, self.own_gate or _gated(self.act_fn))
        return block_fp8_experts(hidden_states, top_k_index, top_k_weights, *weights, act)
