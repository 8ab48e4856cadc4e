"""Products of two 8-bit floating point operands with a scale for each block of 128, as cases that can be timed.

A weight [N, K] is held as e4m3 codes with one float32 scale for each 128 x 128 block; the rows of the activations are
quantized in the call, with one scale for each 128 values of a row.  Both are x = code * scale with
scale = a / 448 and code = e4m3(x * 448 / a), rounded to the nearest, a the block's largest magnitude (2^-100 at least).

Operators:
  linear    y = Q(x) W^T (+ bias)
  train     the same below trained parameters: y, and the gradient grad W that flows on to x
  experts   the experts of a mixture-of-experts block: out_t = sum_j p_tj (Q(act(g) u) D_e^T) with (g | u) = Q(x_t) G_e^T, e = ids_tj
  quantize  codes and scales of a weight (blocks of 128 x 128) or of activations (blocks of 1 x 128)
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
E4M3 = torch.float8_e4m3fn
MOST_FLOPS = 3.8e12                                    # just below the largest listed case
MOST_BYTES = 1.5e9                                     # weights of one drawn case


def listed():
    return [
        # one user: the output projection of one new token, where the launch counts
        dict(name="decode_linear", kind="linear", dtype="bfloat16", m=1, n=4096, k=4096, bias=False),
        # a serving batch of a few dozen sequences through a projection with a bias
        dict(name="serve_batch40", kind="linear", dtype="bfloat16", m=40, n=11008, k=4096, bias=True),
        # a model loaded without a 16-bit dtype: a short prompt, odd rows of the weight, a row length that ends inside a block
        dict(name="ragged_prompt", kind="linear", dtype="float32", m=333, n=3211, k=2112, bias=False),
        # a prompt through the widest layer of a 7B model
        dict(name="prefill_2048", kind="linear", dtype="bfloat16", m=2048, n=11008, k=4096, bias=False),
        # prompts of several users through the widest layer of a 70B model
        dict(name="prefill_8192", kind="linear", dtype="bfloat16", m=8192, n=28672, k=8192, bias=False),
        # adapter finetuning: a step's rows through the down projection of a 7B model
        dict(name="train_2048", kind="train", dtype="bfloat16", m=2048, n=4096, k=11008, bias=False),
        # adapter finetuning of a small model, a batch of no round length
        dict(name="train_77", kind="train", dtype="float16", m=77, n=1200, k=1024, bias=True),
        # one new token through two of eight wide experts
        dict(name="experts_token", kind="experts", dtype="bfloat16", tokens=1, top_k=2, experts=8, hidden=4096, inter=14336),
        # a prompt through the same block
        dict(name="experts_prompt", kind="experts", dtype="bfloat16", tokens=512, top_k=2, experts=8, hidden=4096, inter=14336),
        # many small experts, which get some thirty rows each
        dict(name="experts_small", kind="experts", dtype="float16", tokens=300, top_k=6, experts=64, hidden=2048, inter=1408),
        # loading a checkpoint: the largest weight of a 70B model
        dict(name="quantize_weight", kind="quantize", dtype="bfloat16", m=28672, n=8192, rows=False),
        # the activations of a short prompt, kept for several products
        dict(name="quantize_rows", kind="quantize", dtype="float32", m=333, n=4096, rows=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _length(rng, low, high):
    """A row length: whole blocks mostly, sometimes one that ends inside a block."""
    k = _log(rng, low, high)
    return max(16, k // 16 * 16) if rng.random() < 0.25 else max(128, k // 128 * 128)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "train", "experts", "experts", "quantize"))
    while True:
        if kind in ("linear", "train"):
            types = ("bfloat16", "float16", "float32") if kind == "linear" else ("bfloat16", "float16")
            case = dict(kind=kind, dtype=rng.choice(types), m=_log(rng, 1 if kind == "linear" else 16, 8192),
                        n=_log(rng, 64, 28672), k=_length(rng, 128, 16384), bias=rng.random() < 0.3)
            if rng.random() < 0.6:
                case["n"] = max(64, case["n"] // 64 * 64)
            weights, flops = case["n"] * case["k"], 2 * case["m"] * case["n"] * case["k"]
            flops *= 2 if kind == "train" else 1
        elif kind == "experts":
            experts = rng.choice((4, 8, 10, 16, 60, 64))
            case = dict(kind=kind, dtype=rng.choice(("bfloat16", "float16")), tokens=_log(rng, 1, 4096),
                        top_k=rng.randint(1, min(8, experts // 2)), experts=experts, hidden=_length(rng, 512, 8192),
                        inter=max(256, _log(rng, 256, 14336) // 128 * 128))
            per = 3 * case["hidden"] * case["inter"]
            weights, flops = experts * per, 2 * case["tokens"] * case["top_k"] * per
        else:
            rows = rng.random() < 0.5
            case = dict(kind=kind, dtype=rng.choice(("bfloat16", "float16", "float32")),
                        m=_log(rng, 1 if rows else 64, 28672), n=_length(rng, 128, 16384), rows=rows)
            weights, flops = case["m"] * case["n"] * 4, 0
        if weights <= MOST_BYTES and flops <= MOST_FLOPS:
            return case


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "quantize":
        m, n = case["m"], case["n"]
        blocks = m * -(-n // 128) if case["rows"] else -(-m // 128) * -(-n // 128)
        return {"bytes": m * n * (size + 1) + 4 * blocks, "flops": 0}
    if case["kind"] == "experts":
        t, top, e, h, i = case["tokens"], case["top_k"], case["experts"], case["hidden"], case["inter"]
        used = e * (1 - (1 - top / e) ** t)                # experts that some token goes to, as a mean
        return {"bytes": used * 3 * h * i * (1 + 4 / 128 ** 2) + t * (2 * h * size + top * 12), "flops": 6 * t * top * h * i}
    m, n, k = case["m"], case["n"], case["k"]
    both = 2 if case["kind"] == "train" else 1
    return {"bytes": n * k * (1 + 4 / 128 ** 2) + both * (m * k + m * n) * size + (n * size if case["bias"] else 0), "flops": both * 2 * m * n * k}


# ---- the plain forms

def _spread(scale, shape, rows):
    """One scale for each value: [.., R, C] of the scales of 128-blocks."""
    s = scale.repeat_interleave(128, dim=-1)[..., :shape[-1]]
    return s if rows else s.repeat_interleave(128, dim=-2)[..., :shape[-2], :]


def _largest(x, rows):
    """The largest magnitude of each block."""
    pad = torch.nn.functional.pad(x.abs(), (0, -x.shape[-1] % 128, 0, 0 if rows else -x.shape[-2] % 128))
    a = pad.unflatten(-1, (-1, 128)).amax(-1)
    return a if rows else a.unflatten(-2, (-1, 128)).amax(-2)


def _quantize(x, rows):
    """Codes and scales.  The quotient is taken in 64 bits: next to the border of two codes 32 would decide by their own roundings."""
    a = _largest(x, rows).float().clamp(min=2.0 ** -100)
    q = x.double() * 448 / _spread(a, x.shape, rows).double()
    return q.float().to(E4M3), a / 448


def _values(codes, scale, rows):
    return codes.float() * _spread(scale, codes.shape, rows)


def _linear(x, w, scale, bias):
    y = _values(*_quantize(x, True), True) @ _values(w, scale, False).t()
    return y if bias is None else y + bias.float()


def _experts(s):
    x, ids, p = s["x"], s["ids"], s["p"]
    tokens, top = ids.shape
    counts = torch.bincount(ids.reshape(-1), minlength=s["gate_up"].shape[0])
    used = counts.nonzero().squeeze(1)
    most = int(counts.max())
    order = ids.reshape(-1).argsort(stable=True)
    place = torch.arange(tokens * top, device=x.device) - (counts.cumsum(0) - counts)[ids.reshape(-1)[order]]
    slot = torch.empty_like(order)
    slot[order] = torch.searchsorted(used, ids.reshape(-1)[order]) * most + place     # of each pair, in [used experts, most]
    pad = torch.zeros((used.numel() * most, x.shape[1]), device=x.device)
    pad[slot] = _values(*_quantize(x, True), True).repeat_interleave(top, dim=0)
    gu = torch.bmm(pad.view(used.numel(), most, -1), _values(s["gate_up"][used], s["gate_up_scale"][used], False).transpose(1, 2).contiguous())
    g, u = gu.chunk(2, dim=-1)
    h = _values(*_quantize(g / (1 + torch.exp(-g)) * u, True), True)
    y = torch.bmm(h, _values(s["down"][used], s["down_scale"][used], False).transpose(1, 2).contiguous())
    y = y.reshape(used.numel() * most, -1)[slot].view(tokens, top, -1)
    return (y * p.float().unsqueeze(-1)).sum(1).to(x.dtype)


# ---- inputs

def _activations(gen, shape, dtype):
    """N(0, 1) with a few channels of large magnitude, as the residual stream of a language model has them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.randint(0, shape[-1], (max(1, shape[-1] // 512),), generator=gen, device="cuda")
    x[..., loud] *= 20
    return x.to(dtype)


def _weight(gen, shape):
    w = torch.randn(shape, generator=gen, device="cuda") * 0.02
    a = _largest(w, False).clamp(min=2.0 ** -100)
    return (w * 448 / _spread(a, shape, False)).to(E4M3), a / 448


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"kind": kind}
    if kind == "quantize":
        s["rows"] = case["rows"]
        x = _activations(gen, (case["m"], case["n"]), dtype) if case["rows"] else \
            (torch.randn((case["m"], case["n"]), generator=gen, device="cuda") * 0.02).to(dtype)
        s["x"] = x
    elif kind == "experts":
        e, h, i = case["experts"], case["hidden"], case["inter"]
        s["x"] = _activations(gen, (case["tokens"], h), dtype)
        logits = torch.randn((case["tokens"], e), generator=gen, device="cuda") + torch.randn(e, generator=gen, device="cuda") * 0.3
        p, s["ids"] = torch.softmax(logits, dim=-1).topk(case["top_k"], dim=-1)
        s["p"] = (p / p.sum(-1, keepdim=True)).to(dtype)
        s["gate_up"], s["gate_up_scale"] = (torch.empty((e, 2 * i, h), dtype=E4M3, device="cuda"),
                                            torch.empty((e, 2 * i // 128, -(-h // 128)), device="cuda"))
        s["down"], s["down_scale"] = (torch.empty((e, h, i), dtype=E4M3, device="cuda"),
                                      torch.empty((e, -(-h // 128), i // 128), device="cuda"))
        for j in range(e):
            s["gate_up"][j], s["gate_up_scale"][j] = _weight(gen, (2 * i, h))
            s["down"][j], s["down_scale"][j] = _weight(gen, (h, i))
    else:
        s["x"] = _activations(gen, (case["m"], case["k"]), dtype)
        s["w"], s["scale"] = _weight(gen, (case["n"], case["k"]))
        s["bias"] = torch.randn(case["n"], generator=gen, device="cuda").to(dtype) if case["bias"] else None
        if kind == "train":
            s["x"].requires_grad_()
            s["grad"] = (torch.randn((case["m"], case["n"]), generator=gen, device="cuda") * 0.01).to(dtype)
    return s


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        if s["kind"] == "quantize":
            return _quantize(s["x"], s["rows"])
        if s["kind"] == "experts":
            return _experts(s)
        y = _linear(s["x"], s["w"], s["scale"], s["bias"]).to(s["x"].dtype)
        if s["kind"] == "linear":
            return y
        return y, (s["grad"].float() @ _values(s["w"], s["scale"], False)).to(s["x"].dtype)


def _run_own(s):
    calls = getattr(_run_own, "calls", None)
    if calls is None:                                      # a user's program imports the package once
        sys.path.insert(0, os.path.abspath("ipex-llm_amd"))    # it lives beside this folder, in the working directory
        import ipex_llm.transformers.block_fp8 as calls
        _run_own.calls = calls
    if s["kind"] == "quantize":
        return calls.block_fp8_quantize(s["x"]) if s["rows"] else calls.block_fp8_quantize_weight(s["x"])
    if s["kind"] == "experts":
        return calls.block_fp8_experts(s["x"], s["ids"], s["p"], s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"])
    y = calls.block_fp8_linear(s["x"], s["w"], s["scale"], s["bias"])
    if s["kind"] == "linear":
        return y
    return y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]


# ---- the definition in 64 bits

def _blockwise64(x, high):
    """The codes of x as numbers and the scales of its blocks of `high` x 128, which may end short."""
    x = x.detach().double()
    r, c = x.shape
    codes, scales = torch.zeros_like(x), []
    for j in range(0, c, 128):
        part = x[:, j:j + 128]
        rows = torch.cat([part, part.new_zeros((-r % high, part.shape[1]))]).reshape(-1, high * part.shape[1])
        a = rows.abs().max(dim=1).values.clamp(min=2.0 ** -100)
        q = part * 448 / a.repeat_interleave(high)[:r, None]
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)   # 3 bits behind the leading one
        codes[:, j:j + 128] = torch.round(q / step) * step
        scales.append(a / 448)
    return codes, torch.stack(scales, dim=1)


def _dense64(codes, scale, high):
    codes = codes.detach().double()
    for j in range(scale.shape[1]):
        codes[:, 128 * j:128 * (j + 1)] *= scale[:, j].double().repeat_interleave(high)[:codes.shape[0], None]
    return codes


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return _blockwise64(s["x"], 1 if case["rows"] else 128)
    x = _dense64(*_blockwise64(s["x"], 1), 1)
    if case["kind"] == "experts":
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            t, j = torch.where(s["ids"] == e)
            if t.numel():
                gu = x[t] @ _dense64(s["gate_up"][e], s["gate_up_scale"][e], 128).t()
                g, u = gu[:, :case["inter"]], gu[:, case["inter"]:]
                h = _dense64(*_blockwise64(g * torch.sigmoid(g) * u, 1), 1)
                out.index_add_(0, t, h @ _dense64(s["down"][e], s["down_scale"][e], 128).t() * s["p"][t, j].double()[:, None])
        return out
    w = _dense64(s["w"], s["scale"], 128)
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y if case["kind"] == "linear" else (y, s["grad"].double() @ w)
