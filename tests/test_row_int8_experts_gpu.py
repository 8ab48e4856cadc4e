"""Row-scaled int8 experts and whole mixture-of-experts layers against 64 bits on the host."""
import pytest
import torch

import row_int8_util as u
from ipex_llm.transformers import moe, row_int8 as ri

pytestmark = pytest.mark.gpu
ALL = [torch.float16, torch.bfloat16, torch.float32]
IDS = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
# tokens, top_k, experts, hidden, inter: pair by pair, sorted, sizes that end inside a block, one expert, experts without tokens
SIZES = [(1, 1, 1, 16, 16), (1, 2, 8, 128, 128), (1, 8, 8, 400, 272), (2, 2, 16, 256, 400), (3, 4, 4, 272, 144), (1, 3, 8, 4112, 1040), (40, 2, 5, 512, 256),
         (130, 3, 4, 144, 400), (300, 2, 70, 256, 128), (17, 5, 3, 384, 16), (600, 1, 2, 640, 512), (70, 2, 4, 16, 1040), (1700, 2, 600, 16, 32),
         (2000, 4, 20, 128, 144), (64, 6, 64, 528, 208), (3226, 6, 222, 160, 16),
         (3672, 5, 254, 16, 112), (3947, 5, 114, 16, 208), (5417, 6, 173, 144, 16), (3000, 2, 2100, 16, 16), (900, 2, 2100, 16, 16), (4096, 1, 2048, 16, 16), (4100, 1, 3, 16, 16)]


def ids(v):
    return IDS.get(v) if isinstance(v, torch.dtype) else None


def gen(seed):
    return torch.Generator().manual_seed(seed)


def experts(g, n_exp, hidden, inter):
    gate_up, gs = u.weight(g, 2 * inter, hidden, (n_exp,), std=0.5 / hidden ** 0.5 * 4)
    down, ds = u.weight(g, hidden, inter, (n_exp,))
    return gate_up, gs, down, ds


def plain(x, index, p, gate_up, gs, down, ds, act=0):
    """(results, how far each may be off by codes of h next to a border): the oracle in float64.

    h in float32: three scales and sums of two, g and u, each 2^-24; exp2 and reciprocal 2^-23 each, the exponent's rounding 2^-24 times 2 |g|, at
    most 2 * 16 where silu is not g or 0 already: 2^-18 in all at most.  A code of up to 127 then lies 127 * 2^-18 = 4.8e-4 from the true quotient at
    most; of I values evenly spread between borders up to 1e-3 I = L change sides in the mean, by one step each, and more than N = L + 6 sqrt(L) + 6 in
    one row of 10^9 (the tail of their number's distribution).  Each moves a row by a column of `down` times a step of h; N of them, of either sign, by
    2 sqrt(N) of the largest column at most: all of one sign up to four, and twice the root of their squares beyond."""
    x, p = x.double(), p.double()
    codes, xs = u.quantize(x.float())
    out, slack = torch.zeros_like(x), torch.zeros(x.shape[0], dtype=torch.float64)
    for e in range(gate_up.shape[0]):
        t, j = torch.where(index == e)
        if t.numel():
            gu = u.sums(codes[t], gate_up[e]) * xs[t].double().unsqueeze(-1) * gs[e].double()
            g, v = gu.chunk(2, dim=-1)
            a = g * torch.sigmoid(g) if act == 0 else torch.nn.functional.gelu(g, approximate="tanh")
            h = a * v
            top = h.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
            hc = torch.round(h * 127 / top)
            y = (hc @ down[e].double().t()) * (top / 127) * ds[e].double() * p[t, j].unsqueeze(-1)
            out.index_add_(0, t, y)
            mean = 1e-3 * h.shape[1]
            column = (down[e].double() * ds[e].double().unsqueeze(-1)).norm(dim=0).amax()
            slack.index_add_(0, t, 2 * (mean + 6 * mean ** 0.5 + 6) ** 0.5 * column * (top[:, 0] / 127) * p[t, j])
    return out, slack


def check(got, want, slack, dtype):
    """The result: half a unit of its type, of the smallest numbers half of those; sums and scales in float32; codes that changed sides."""
    off = (got.cpu().double() - want).norm(dim=1)
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -20) * want.norm(dim=1) + slack + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 * want.shape[1] ** 0.5
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max()
    if dtype == torch.float32:                               # rows of which no code changed sides
        assert (off <= 2.0 ** -19 * want.norm(dim=1)).double().mean() >= 0.5


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", SIZES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_experts(dtype, tokens, top_k, n_exp, hidden, inter):
    g = gen(tokens + hidden)
    x = torch.randn((tokens, hidden), generator=g).to(dtype)
    weights = experts(g, n_exp, hidden, inter)
    index = torch.randint(0, n_exp, (tokens, top_k), generator=g)         # (the same expert twice, too)
    p = torch.rand((tokens, top_k), generator=g)
    dev = [w.cuda() for w in weights]
    for act in (0, 1):
        y = ri.row_int8_experts(x.cuda(), index.cuda(), p.cuda(), *dev, act)
        assert y.dtype == dtype and y.shape == x.shape
        check(y, *plain(x, index, p, *weights, act), dtype)
    y = ri.row_int8_experts(x.cuda(), index.int().cuda(), p.to(dtype).cuda(), *dev)
    check(y, *plain(x, index, p.to(dtype), *weights), dtype)


def test_every_form_is_run():
    from gpu_util import ggml
    plans = [ggml.lowbit_row_int8_experts_plan(*s) for s in SIZES]
    assert {p[0] for p in plans} == {0, 32, 64, 128, 192}
    assert {p[1:3] for p in plans} == {(0, 0), (64, 64), (64, 128), (128, 256), (256, 256)}
    assert {p[3] for p in plans if p[0]} == {0, 1}
    assert {ggml.lowbit_row_int8_experts_waves(*s) for s in SIZES} == {0, 8, 16}


@pytest.mark.parametrize("tokens", [1, 3, 50])
def test_ids_that_name_no_expert(tokens):
    g = gen(tokens)
    x = torch.randn((tokens, 256), generator=g).bfloat16()
    weights = experts(g, 6, 256, 128)
    index = torch.randint(-1, 8, (tokens, 4), generator=g)
    index[0] = torch.tensor([-1, 6, 1 << 40, -(1 << 40)])
    p = torch.rand((tokens, 4), generator=g)
    y = ri.row_int8_experts(x.cuda(), index.cuda(), p.cuda(), *[w.cuda() for w in weights])
    check(y, *plain(x, index, p, *weights), torch.bfloat16)
    assert not y[0].any()


@pytest.mark.parametrize("tokens", [1, 4, 60])
def test_rows_with_a_nan_stay_their_own(tokens):
    """A token with a NaN has NaN results; a zero one zeros; an expert with a NaN scale spoils its tokens only."""
    g = gen(tokens)
    x = torch.randn((tokens, 256), generator=g).bfloat16()
    weights = experts(g, 8, 256, 128)
    index = torch.stack([torch.randperm(7, generator=g)[:2] for _ in range(tokens)])
    p = torch.rand((tokens, 2), generator=g)
    x[0, 7] = float("nan")
    if tokens > 1:
        x[1] = 0
    weights[1][7, 3] = float("nan")
    index[-1, 0] = 7 if tokens > 2 else index[-1, 0]
    y = ri.row_int8_experts(x.cuda(), index.cuda(), p.cuda(), *[w.cuda() for w in weights]).cpu()
    assert y[0].isnan().all()
    if tokens > 2:
        assert y[-1].isnan().all() and y[1:-1].isfinite().all() and not y[1].any()


def test_more_tokens_than_the_workspace_holds_at_once():
    """Above 2 GiB of h, codes and results the tokens go in parts: each as if by itself."""
    g = gen(9)
    tokens, top_k, n_exp, hidden, inter = 60000, 2, 3, 16, 4096
    x = torch.randn((tokens, hidden), generator=g).bfloat16().cuda()
    dev = [w.cuda() for w in experts(g, n_exp, hidden, inter)]
    index = torch.randint(0, n_exp, (tokens, top_k), generator=g).cuda()
    p = torch.rand((tokens, top_k), generator=g).cuda()
    y = ri.row_int8_experts(x, index, p, *dev)
    parts = [ri.row_int8_experts(x[a:a + 20000], index[a:a + 20000], p[a:a + 20000], *dev) for a in range(0, tokens, 20000)]
    assert torch.equal(y, torch.cat(parts))


@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_gradients_of_experts(dtype, tokens):
    """x's and the weights' gradients against autograd in float64 with the quantizations as the identity."""
    g = gen(tokens)
    n_exp, hidden, inter, top_k = 4, 144, 64, 2
    x = torch.randn((tokens, hidden), generator=g).to(dtype)
    weights = experts(g, n_exp, hidden, inter)
    index = torch.randint(0, n_exp, (tokens, top_k), generator=g)
    p = torch.rand((tokens, top_k), generator=g)
    grad = torch.randn((tokens, hidden), generator=g).to(dtype)
    xd, pd = x.cuda().requires_grad_(), p.cuda().requires_grad_()
    y = ri.row_int8_experts(xd, index.cuda(), pd, *[w.cuda() for w in weights])
    check(y.detach(), *plain(x, index, p, *weights), dtype)
    gx, gp = torch.autograd.grad(y, (xd, pd), grad.cuda())

    xo, po = x.double().requires_grad_(), p.double().requires_grad_()
    gate_up, gs, down, ds = (w.double() for w in weights)

    def through(v):                                          # quantized forward, identity backward
        top = v.detach().abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
        return v + (torch.round(v.detach() * 127 / top) * top / 127 - v.detach())
    xq, out = through(xo), torch.zeros((tokens, hidden), dtype=torch.float64)
    for e in range(n_exp):
        t, j = torch.where(index == e)
        if t.numel():
            a, b = (xq[t] @ (gate_up[e] * gs[e].unsqueeze(-1)).t()).chunk(2, dim=-1)
            out = out.index_add(0, t, through(torch.nn.functional.silu(a) * b) @ (down[e] * ds[e].unsqueeze(-1)).t() * po[t, j].unsqueeze(-1))
    wx, wp = torch.autograd.grad(out, (xo, po), grad.double())
    # sums of products in float32 throughout; a code of h that changes sides moves gp by its share of the result (see plain)
    assert (gx.cpu().double() - wx).norm() <= (torch.finfo(dtype).eps / 2 + 2e-6) * wx.norm()
    assert (gp.cpu().double() - wp).norm() <= 2e-3 * wp.norm()


# ---------------------------------------------------------------- whole layers

@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", SIZES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_layer_is_router_and_experts(dtype, tokens, top_k, n_exp, hidden, inter):
    g = gen(tokens * 3 + hidden)
    x = torch.randn((tokens, hidden), generator=g).to(dtype)
    weights = experts(g, n_exp, hidden, inter)
    router = (torch.randn((n_exp, hidden), generator=g) / hidden ** 0.5).to(dtype)
    bias = torch.randn(n_exp, generator=g) * 0.1
    top_k = min(top_k, n_exp)
    dev = [w.cuda() for w in weights]
    if n_exp > 1024:
        pytest.skip("more experts than the router takes")
    for b, score, renormalize, scale in ((None, "softmax", True, 1.0), (bias, "sigmoid", True, 2.5), (None, "softmax", False, 1.0)):
        bd = None if b is None else b.cuda()
        y = ri.row_int8_moe(x.cuda(), router.cuda(), top_k, *dev, bias=bd, score=score, renormalize=renormalize, scale=scale)
        w, index = moe.moe_route(x.cuda(), router.cuda(), top_k, bd, score, renormalize, scale)
        assert torch.equal(y, ri.row_int8_experts(x.cuda(), index, w, *dev))
        z = x.double() @ router.double().t()
        s = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)
        order = torch.sort(z if b is None else s + b.double(), dim=-1, descending=True, stable=True).indices[:, :top_k]
        p = s.gather(1, order)
        p = (p / p.sum(-1, keepdim=True) if renormalize else p) * scale
        assert torch.equal(index.cpu(), order)
        check(y, *plain(x, order, p, *weights), dtype)


def test_layer_gradients_flow_through_router_and_experts():
    g = gen(3)
    x = torch.randn((20, 64), generator=g)
    dev = [w.cuda() for w in experts(g, 4, 64, 32)]
    router = torch.randn((4, 64), generator=g) / 8
    xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
    y = ri.row_int8_moe(xd, rd, 2, *dev)
    gx, gr = torch.autograd.grad(y.square().sum(), (xd, rd))
    w, index = moe.moe_route(xd, rd, 2)
    y2 = ri.row_int8_experts(xd, index, w, *dev)
    wx, wr = torch.autograd.grad(y2.square().sum(), (xd, rd))
    assert torch.equal(y, y2) and torch.equal(gx, wx) and torch.equal(gr, wr) and gr.any()


@pytest.mark.parametrize("tokens", [1, 5, 100])
def test_layer_in_a_graph(tokens):
    """Replays with other inputs against the eager call, two graphs in turn, with eager work between them."""
    g = gen(tokens)
    dev = [w.cuda() for w in experts(g, 8, 256, 144)]
    router = (torch.randn((8, 256), generator=g) / 16).bfloat16().cuda()
    x = [torch.randn((tokens, 256), generator=g).bfloat16().cuda() for _ in range(2)]
    for v in x:
        ri.row_int8_moe(v, router, 2, *dev)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for v in x:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ri.row_int8_moe(v, router, 2, *dev))
        graphs.append(graph)
    for step in range(4):
        for v in x:
            v.copy_(torch.randn((tokens, 256), generator=g).bfloat16())
        want = [ri.row_int8_moe(v, router, 2, *dev) for v in x]
        for graph in graphs if step % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert torch.equal(out, ref)


def test_refusals():
    g = gen(1)
    gate_up, gs, down, ds = (w.cuda() for w in experts(g, 4, 64, 32))
    x = torch.randn((3, 64), generator=g).cuda()
    index, p = torch.zeros((3, 2), dtype=torch.int64, device="cuda"), torch.ones((3, 2), device="cuda")
    router = torch.zeros((4, 64), device="cuda")
    for call, why in ((lambda: ri.row_int8_experts(x, index, p, gate_up, gs, down, ds, act=2), "act is 0"),
                      (lambda: ri.row_int8_experts(x, index.float(), p, gate_up, gs, down, ds), "whole indices"),
                      (lambda: ri.row_int8_experts(x, index, p[:, :1], gate_up, gs, down, ds), "whole indices"),
                      (lambda: ri.row_int8_experts(x, index, p, gate_up[:, :32], gs[:, :32], down, ds), "contiguous|fit together"),
                      (lambda: ri.row_int8_experts(x, index, p, gate_up, gs[:, :63], down, ds), "one scale for each row"),
                      (lambda: ri.row_int8_experts(x[:, :32], index, p, gate_up, gs, down, ds), r"x must be \[tokens, 64\]"),
                      (lambda: ri.row_int8_experts(x.double(), index, p, gate_up, gs, down, ds), "unsupported dtype"),
                      (lambda: ri.row_int8_experts(x, index, p, gate_up.float(), gs, down, ds), "codes are int8"),
                      (lambda: ri.row_int8_moe(x, router[:3], 2, gate_up, gs, down, ds), "3 rows for 4 experts"),
                      (lambda: ri.row_int8_moe(x, router, 5, gate_up, gs, down, ds), "top_k"),
                      (lambda: ri.row_int8_moe(x, router, 2, gate_up, gs, down, ds, score="relu"), "score"),
                      (lambda: ri.row_int8_moe(x.cpu(), router, 2, gate_up, gs, down, ds), "no CPU implementation")):
        with pytest.raises(RuntimeError, match=why):
            call()
    assert ri.row_int8_experts(x[:0], index[:0], p[:0], gate_up, gs, down, ds).shape == (0, 64)
    assert ri.row_int8_moe(x[:0], router, 2, gate_up, gs, down, ds).shape == (0, 64)
    assert not ri.row_int8_experts(x, index[:, :0], p[:, :0], gate_up, gs, down, ds).any()
