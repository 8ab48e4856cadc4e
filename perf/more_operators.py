"""Products of 8-bit integers with a scale for each token and channel, and mixture-of-experts layers from the router on, as cases that can
be timed.

A weight [N, K] is held as int8 codes with one float32 scale for each row; the rows of the activations are quantized in the call.  Both are
x = code * scale with scale = a / 127 and code = x * 127 / a, rounded to the nearest, ties to even, a the row's largest magnitude (2^-100 at
least).

Operators:
  linear    y = Q(x) W^T (+ bias)
  train     the same below trained parameters: y, and the gradient grad W that flows on to x
  quantize  codes and scales of rows
  route     the experts of each token and their weights: z = x R^T, s = softmax(z) or sigmoid(z), the top_k largest z (s + bias with a
            bias), weights s of those, renormalized or not, times a factor; with `train` the gradients of x and R for given ones of the weights
  layer     out_t = sum_j p_tj (Q(act(g) u) D_e^T) with (g | u) = Q(x_t) G_e^T and (p, e) from route
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
MOST_FLOPS = 3.8e12                                    # just below the largest listed case
MOST_BYTES = 1.5e9                                     # weights of one drawn case
MOST_ROUTE = 2.0e10                                    # operations of one drawn router


def listed():
    return [
        # one user: the output projection of one new token, where the launch counts
        dict(name="decode_linear", kind="linear", dtype="bfloat16", m=1, n=4096, k=4096, bias=False),
        # a serving batch of a few dozen sequences through a projection with a bias
        dict(name="serve_batch48", kind="linear", dtype="float16", m=48, n=11008, k=4096, bias=True),
        # a model loaded without a 16-bit dtype: a prompt, odd rows of the weight, a row length of no round number
        dict(name="ragged_prompt", kind="linear", dtype="float32", m=777, n=3211, k=2128, bias=False),
        # prompts of several users through the widest layer of a 70B model
        dict(name="prefill_8192", kind="linear", dtype="bfloat16", m=8192, n=28672, k=8192, bias=False),
        # adapter finetuning: a step's rows through the down projection of a 7B model
        dict(name="train_2048", kind="train", dtype="bfloat16", m=2048, n=4096, k=11008, bias=False),
        # adapter finetuning of a small model in float32, a batch of no round length
        dict(name="train_77", kind="train", dtype="float32", m=77, n=1203, k=1024, bias=True),
        # converting a checkpoint: the largest weight of a 70B model
        dict(name="quantize_weight", kind="quantize", dtype="bfloat16", m=28672, n=8192),
        # the activations of a serving batch, kept for several products
        dict(name="quantize_rows", kind="quantize", dtype="float16", m=48, n=11008),
        # a long prompt's tokens dealt to many experts
        dict(name="route_prompt", kind="route", dtype="bfloat16", tokens=4096, hidden=2048, experts=64, top_k=6, score="softmax", bias=False,
             renormalize=True, train=False),
        # finetuning with the router: a step's tokens, scores by sigmoid with a correction of the choice
        dict(name="route_train", kind="route", dtype="bfloat16", tokens=1000, hidden=4096, experts=60, top_k=4, score="sigmoid", bias=True,
             renormalize=True, train=True),
        # one new token through two of eight wide experts, the router included
        dict(name="layer_token", kind="layer", dtype="bfloat16", tokens=1, hidden=4096, inter=14336, experts=8, top_k=2, score="softmax",
             bias=False, renormalize=True),
        # a prompt through a layer of many small experts
        dict(name="layer_prompt", kind="layer", dtype="float16", tokens=500, hidden=2048, inter=1408, experts=64, top_k=6, score="softmax",
             bias=False, renormalize=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _length(rng, low, high):
    """A row length: a multiple of 128 mostly, sometimes one of 16."""
    k = _log(rng, low, high)
    return max(16, k // 16 * 16) if rng.random() < 0.3 else max(128, k // 128 * 128)


def _router(rng, tokens, hidden):
    experts = rng.choice((4, 8, 10, 16, 60, 64, 128, 160, 256))
    return dict(tokens=tokens, hidden=hidden, experts=experts, top_k=rng.randint(1, min(8, experts // 2)),
                score=rng.choice(("softmax", "softmax", "sigmoid")), bias=rng.random() < 0.3, renormalize=rng.random() < 0.7)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "train", "quantize", "route", "route", "layer", "layer", "layer"))
    types = ("bfloat16", "bfloat16", "float16") + (("float32",) if kind != "layer" else ())
    while True:
        case = dict(kind=kind, dtype=rng.choice(types))
        if kind in ("linear", "train"):
            case |= dict(m=_log(rng, 1 if kind == "linear" else 16, 8192), n=_log(rng, 64, 28672), k=_length(rng, 128, 16384), bias=rng.random() < 0.3)
            if rng.random() < 0.6:
                case["n"] = max(64, case["n"] // 64 * 64)
            weights, flops = case["n"] * case["k"], 2 * case["m"] * case["n"] * case["k"] * (2 if kind == "train" else 1)
        elif kind == "quantize":
            case |= dict(m=_log(rng, 1, 28672), n=_length(rng, 128, 16384))
            weights, flops = case["m"] * case["n"] * 4, 0
        elif kind == "route":
            case |= _router(rng, _log(rng, 1, 8192), _length(rng, 512, 8192)) | dict(train=rng.random() < 0.4)
            weights, flops = case["experts"] * case["hidden"] * 4, 2 * case["tokens"] * case["experts"] * case["hidden"] * (3 if case["train"] else 1)
            if flops > MOST_ROUTE:
                continue
        else:
            case |= _router(rng, _log(rng, 1, 4096), _length(rng, 512, 8192))
            case["inter"] = _length(rng, 256, 14336)
            per = 3 * case["hidden"] * case["inter"]
            weights, flops = case["experts"] * per, 2 * case["tokens"] * case["top_k"] * per
        if weights <= MOST_BYTES and flops <= MOST_FLOPS:
            return case


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "quantize":
        return {"bytes": case["m"] * case["n"] * (size + 1) + 4 * case["m"], "flops": 0}
    if case["kind"] in ("route", "layer"):
        t, top, e, h = case["tokens"], case["top_k"], case["experts"], case["hidden"]
        routing = {"bytes": (t + e) * h * size, "flops": 2 * t * e * h}
        if case["kind"] == "route":
            if not case["train"]:
                return {"bytes": routing["bytes"] + t * top * 12, "flops": routing["flops"]}
            return {"bytes": 2 * routing["bytes"] + t * top * 16, "flops": 3 * routing["flops"]}       # (gradients as large as x and the router)
        used = e * (1 - (1 - top / e) ** t)            # experts that some token goes to, as a mean
        return {"bytes": routing["bytes"] + used * (3 * h * case["inter"] + 4 * (2 * case["inter"] + h)) + t * h * size,
                "flops": routing["flops"] + 6 * t * top * h * case["inter"]}
    m, n, k = case["m"], case["n"], case["k"]
    both = 2 if case["kind"] == "train" else 1
    return {"bytes": n * (k + 4) + both * (m * k + m * n) * size + (n * size if case["bias"] else 0), "flops": both * 2 * m * n * k}


# ---- the plain forms

def _quantize(x):
    """Codes as numbers, and scales.  The quotient is taken in 64 bits: next to the border of two codes 32 would decide by their own roundings."""
    a = x.abs().amax(-1, keepdim=True).float().clamp(min=2.0 ** -100)
    return torch.round(x.double() * 127 / a.double()).float(), a / torch.full_like(a, 127.0)


def _values(codes, scale):
    return codes.float() * scale


def _linear(x, w, scale, bias):
    codes, xs = _quantize(x)
    y = (codes @ w.float().t()) * xs * scale
    return y if bias is None else y + bias.float()


def _route(s):
    """Weights and indices, and what the gradients need: the scores of all experts and of the chosen ones, and the sum that divides those."""
    z = s["x"].double() @ s["router"].double().t()             # (64 bits: which of two near experts is taken)
    score = 1 / (1 + torch.exp(-z))
    if s["score"] == "softmax":
        score = torch.exp(z - z.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    order = torch.sort(z if s["choice"] is None else score + s["choice"].double(), dim=-1, descending=True, stable=True).indices[:, :s["top_k"]]
    chosen = score.gather(1, order)
    total = chosen.sum(-1, keepdim=True) if s["renormalize"] else torch.ones_like(chosen[:, :1])
    return chosen / total, order, score, total


def _route_train(s):
    w, order, score, total = _route(s)
    g = s["grad"].double()
    if s["renormalize"]:
        g = (g - (g * w).sum(-1, keepdim=True)) / total
    ds = torch.zeros_like(score).scatter(1, order, g)
    if s["score"] == "softmax":
        dz = score * (ds - (ds * score).sum(-1, keepdim=True))
    else:
        dz = ds * score * (1 - score)
    dtype = s["x"].dtype
    return w.float(), order, (dz @ s["router"].double()).to(dtype), (dz.t() @ s["x"].double()).to(dtype)


def _layer(s):
    x = s["x"]
    p, ids = _route(s)[:2]
    tokens, top = ids.shape
    counts = torch.bincount(ids.reshape(-1), minlength=s["gate_up"].shape[0])
    used = counts.nonzero().squeeze(1)
    most = int(counts.max())
    order = ids.reshape(-1).argsort(stable=True)
    place = torch.arange(tokens * top, device=x.device) - (counts.cumsum(0) - counts)[ids.reshape(-1)[order]]
    slot = torch.empty_like(order)
    slot[order] = torch.searchsorted(used, ids.reshape(-1)[order]) * most + place     # of each pair, in [used experts, most]
    pad = torch.zeros((used.numel() * most, x.shape[1]), device=x.device)
    pad[slot] = _values(*_quantize(x)).repeat_interleave(top, dim=0)
    gu = torch.bmm(pad.view(used.numel(), most, -1), _values(s["gate_up"][used], s["gate_up_scale"][used].unsqueeze(-1)).transpose(1, 2).contiguous())
    g, u = gu.chunk(2, dim=-1)
    h = _values(*_quantize(g / (1 + torch.exp(-g)) * u))
    y = torch.bmm(h, _values(s["down"][used], s["down_scale"][used].unsqueeze(-1)).transpose(1, 2).contiguous())
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
    a = w.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    return torch.round(w * 127 / a).to(torch.int8), (a / 127).squeeze(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"kind": kind}
    if kind == "quantize":
        s["x"] = _activations(gen, (case["m"], case["n"]), dtype)
    elif kind in ("route", "layer"):
        e, h = case["experts"], case["hidden"]
        s |= {"top_k": case["top_k"], "score": case["score"], "renormalize": case["renormalize"]}
        s["x"] = _activations(gen, (case["tokens"], h), dtype)
        s["router"] = (torch.randn((e, h), generator=gen, device="cuda") * (0.8 / h ** 0.5)).to(dtype)
        s["choice"] = torch.randn(e, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        s["train"] = case.get("train", False)
        if s["train"]:
            s["x"].requires_grad_()
            s["router"].requires_grad_()
            s["grad"] = torch.randn((case["tokens"], case["top_k"]), generator=gen, device="cuda") * 0.01
        if kind == "layer":
            i = case["inter"]
            s["gate_up"], s["gate_up_scale"] = torch.empty((e, 2 * i, h), dtype=torch.int8, device="cuda"), torch.empty((e, 2 * i), device="cuda")
            s["down"], s["down_scale"] = torch.empty((e, h, i), dtype=torch.int8, device="cuda"), torch.empty((e, h), device="cuda")
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
            codes, scale = _quantize(s["x"])
            return codes.to(torch.int8), scale.squeeze(-1)
        if s["kind"] == "route":
            if s["train"]:
                return _route_train(s)
            w, order = _route(s)[:2]
            return w.float(), order
        if s["kind"] == "layer":
            return _layer(s)
        y = _linear(s["x"], s["w"], s["scale"], s["bias"]).to(s["x"].dtype)
        if s["kind"] == "linear":
            return y
        return y, ((s["grad"].float() * s["scale"]) @ s["w"].float()).to(s["x"].dtype)


def _run_own(s):
    calls = getattr(_run_own, "calls", None)
    if calls is None:                                      # a user's program imports the package once
        sys.path.insert(0, os.path.abspath("ipex-llm_amd"))    # it lives beside this folder, in the working directory
        import ipex_llm.transformers.moe as moe
        import ipex_llm.transformers.row_int8 as row_int8
        calls = _run_own.calls = (row_int8, moe)
    row_int8, moe = calls
    if s["kind"] == "quantize":
        return row_int8.row_int8_quantize(s["x"])
    if s["kind"] == "route":
        w, order = moe.moe_route(s["x"], s["router"], s["top_k"], bias=s["choice"], score=s["score"], renormalize=s["renormalize"])
        return (w.detach(), order, *torch.autograd.grad(w, (s["x"], s["router"]), s["grad"])) if s["train"] else (w, order)
    if s["kind"] == "layer":
        return row_int8.row_int8_moe(s["x"], s["router"], s["top_k"], s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"],
                                     bias=s["choice"], score=s["score"], renormalize=s["renormalize"])
    y = row_int8.row_int8_linear(s["x"], s["w"], s["scale"], s["bias"])
    if s["kind"] == "linear":
        return y
    return y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]


# ---- the definition in 64 bits

def _rows64(x):
    """What the codes of x's rows stand for."""
    x = x.detach().double()
    most = torch.maximum(x.max(-1, keepdim=True).values, -x.min(-1, keepdim=True).values).clamp(min=2.0 ** -100)
    return torch.round(x / most * 127), most / 127


def _dense64(codes, scale):
    return codes.detach().double() * scale.detach().double().unsqueeze(-1)


def _gates64(case, s):
    """For each token the weights of all experts (zero where it is not sent), the chosen ones in order, and d weights / d logits by autograd."""
    z = (s["x"].detach().double() @ s["router"].detach().double().t()).requires_grad_()
    score = torch.softmax(z, -1) if case["score"] == "softmax" else torch.sigmoid(z)
    by = (z if s["choice"] is None else score + s["choice"].double()).detach()
    order = torch.argsort(by, dim=-1, descending=True, stable=True)[:, :case["top_k"]]
    w = torch.gather(score, 1, order)
    return (w / w.sum(-1, keepdim=True) if case["renormalize"] else w), order, z


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return None, _rows64(s["x"])[1].squeeze(-1)
    if case["kind"] == "route":
        w, order, z = _gates64(case, s)
        if not case["train"]:
            return w.detach(), order
        dz = torch.autograd.grad(w, z, s["grad"].double())[0]
        return w.detach(), order, dz @ s["router"].detach().double(), dz.t() @ s["x"].detach().double()
    codes, scale = _rows64(s["x"])
    x = codes * scale
    if case["kind"] == "layer":
        p, ids, _ = _gates64(case, s)
        p, out = p.detach(), torch.zeros_like(x)
        for e in range(case["experts"]):
            t, j = torch.where(ids == e)
            if t.numel():
                gu = x[t] @ _dense64(s["gate_up"][e], s["gate_up_scale"][e]).t()
                g, u = gu[:, :case["inter"]], gu[:, case["inter"]:]
                hc, hs = _rows64(g * torch.sigmoid(g) * u)
                out.index_add_(0, t, (hc * hs) @ _dense64(s["down"][e], s["down_scale"][e]).t() * p[t, j][:, None])
        return out
    w = _dense64(s["w"], s["scale"])
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y if case["kind"] == "linear" else (y, s["grad"].double() @ w)
