"""The router of a mixture-of-experts block against 64 bits on the host."""
import math

import pytest
import torch

from ipex_llm.transformers import moe

pytestmark = pytest.mark.gpu
ALL = [torch.float16, torch.bfloat16, torch.float32]
IDS = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
RULES = [("softmax", True, False), ("softmax", False, False), ("softmax", True, True), ("sigmoid", True, True), ("sigmoid", False, False)]


def ids(v):
    return IDS.get(v) if isinstance(v, torch.dtype) else None


def gen(seed):
    return torch.Generator().manual_seed(seed)


def plain(x, router, top_k, bias=None, score="softmax", renormalize=True, scale=1.0):
    z = x.double() @ router.double().t()
    s = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)
    by = z if bias is None else s + bias.double()
    index = torch.sort(by.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k]
    w = s.gather(1, index)
    return (w / w.sum(-1, keepdim=True) if renormalize else w) * scale, index


def operands(t, e, h, dtype, rdtype, seed=0):
    g = gen(t * 31 + e + seed)
    x = torch.randn((t, h), generator=g)
    x[:, torch.randint(0, h, (1 + h // 512,), generator=g)] *= 20
    return x.to(dtype), (torch.randn((e, h), generator=g) * (0.8 / h ** 0.5)).to(rdtype), torch.randn(e, generator=g) * 0.1


SIZES = [(1, 1, 8, 1), (1, 8, 4096, 2), (1, 64, 2048, 6), (3, 60, 1032, 4), (16, 16, 520, 16), (17, 33, 64, 3), (70, 130, 1024, 8), (300, 256, 2048, 8),
         (1000, 60, 512, 4), (5, 1000, 256, 64), (33, 512, 40, 7), (2050, 8, 72, 2), (300, 20, 16384, 2)]


@pytest.mark.parametrize("t,e,h,k", SIZES)
@pytest.mark.parametrize("score,renormalize,biased", RULES)
def test_route(score, renormalize, biased, t, e, h, k):
    for dtype, rdtype in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32), (torch.float32, torch.float16)):
        x, router, bias = operands(t, e, h, dtype, rdtype)
        bias = bias if biased else None
        w, index = moe.moe_route(x.cuda(), router.cuda(), k, None if bias is None else bias.cuda(), score, renormalize, 1.5)
        want, order = plain(x, router, k, bias, score, renormalize, 1.5)
        assert w.dtype == torch.float32 and index.dtype == torch.int64 and w.shape == index.shape == (t, k)
        assert torch.equal(index.cpu(), order)
        # float64 throughout, rounded once to float32
        assert ((w.cpu().double() - want).abs() <= 2.0 ** -23 * want).all()


def test_ties_go_to_the_lowest_index():
    """Whole numbers, so that the sums are exact and experts with equal rows tie."""
    g = gen(1)
    x = torch.randint(-3, 4, (40, 64), generator=g).float()
    rows = torch.randint(-2, 3, (5, 64), generator=g).float()
    router = rows[torch.randint(0, 5, (200,), generator=g)]
    for dtype in ALL:
        w, index = moe.moe_route(x.to(dtype).cuda(), router.to(dtype).cuda(), 60)
        want, order = plain(x, router, 60)
        assert torch.equal(index.cpu(), order)
        w, index = moe.moe_route(torch.zeros_like(x).to(dtype).cuda(), router.to(dtype).cuda(), 7)
        assert torch.equal(index.cpu(), torch.arange(7).expand(40, 7)) and torch.equal(w.cpu(), torch.full((40, 7), 1 / 7))


def test_not_a_number_and_infinity():
    x, router, _ = operands(6, 70, 64, torch.float32, torch.float32)
    x[1, 3] = math.nan
    router[40] = math.nan
    x[2] = 0
    router[5, 0], x[3, 0] = math.inf, 1.0
    w, index = (v.cpu() for v in moe.moe_route(x.cuda(), router.cuda(), 3))
    assert index[1].tolist() == [0, 1, 2]                    # all logits NaN
    assert index[3].tolist()[:2] == [40, 5] or index[3].tolist()[:2] == [5, 40]
    assert (index[[0, 4, 5], 0] == 40).sum() + (index[[0, 4, 5], 0] == 5).sum() == 3
    assert w.isnan().all()
    # far apart: one expert has all the weight, the others' scores are the smallest numbers and no tie
    big = torch.zeros((1, 8))
    big[0, 0] = 1.0
    r = torch.zeros((4, 8))
    r[:, 0] = torch.tensor([-2000.0, 0.0, 2000.0, -1000.0])
    w, index = (v.cpu() for v in moe.moe_route(big.cuda(), r.cuda(), 4))
    assert index.tolist() == [[2, 1, 3, 0]] and w.tolist() == [[1.0, 0.0, 0.0, 0.0]]
    w, index = (v.cpu() for v in moe.moe_route(big.cuda(), r.cuda(), 4, score="sigmoid"))
    assert index.tolist() == [[2, 1, 3, 0]] and abs(w[0, 0] - 2 / 3) < 1e-7


def back_tolerance(dtype):
    """Of the 2-norm.  The gradient of the logits rounded to float32, 2^-24; sums in float32: up to 128 instructions one after the other in a wave,
    whose roundings add up in squares, sqrt(128) * 2^-24 = 7e-7 at most, and some ten sums of waves and parts; the result half a unit of its type."""
    return 2.0 ** -24 + 1e-6 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("t,e,h,k", [(1, 1, 8, 1), (1, 8, 64, 2), (5, 33, 520, 3), (40, 64, 1032, 6), (300, 130, 256, 8), (1000, 60, 512, 4), (4100, 16, 136, 2), (70, 1000, 72, 9)])
@pytest.mark.parametrize("score,renormalize,biased", RULES)
def test_gradients(score, renormalize, biased, t, e, h, k):
    for dtype, rdtype in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)):
        x, router, bias = operands(t, e, h, dtype, rdtype, 1)
        bias = bias if biased else None
        g = torch.randn((t, k), generator=gen(5)) * torch.exp2(torch.randint(-6, 3, (t, 1), generator=gen(6)).float())
        xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
        w, index = moe.moe_route(xd, rd, k, None if bias is None else bias.cuda(), score, renormalize, 0.5)
        assert w.requires_grad and not index.requires_grad
        gx, gr = torch.autograd.grad(w, (xd, rd), g.cuda(), retain_graph=True)
        xo, ro = x.double().requires_grad_(), router.double().requires_grad_()
        want, order = plain(xo, ro, k, bias, score, renormalize, 0.5)
        assert torch.equal(index.cpu(), order)
        wx, wr = torch.autograd.grad(want, (xo, ro), g.double())
        assert gx.dtype == dtype and gr.dtype == rdtype
        # what the formula takes apart, in 64 bits, by its own size: d z is a difference of such terms
        for got, ref in ((gx, wx), (gr, wr)):
            off = (got.cpu().double() - ref).norm()
            assert off <= back_tolerance(got.dtype) * ref.norm() + 1e-12 * g.norm(), (off / ref.norm(), got.dtype)
        only, = torch.autograd.grad(w, rd, g.cuda(), retain_graph=True)
        assert torch.equal(only, gr)
        only, = torch.autograd.grad(w, xd, g.cuda())
        assert torch.equal(only, gx)


def test_gradients_against_differences():
    x, router, bias = operands(3, 6, 16, torch.float32, torch.float32)
    g = torch.randn((3, 2), generator=gen(2)).double()
    for score, renormalize, biased in RULES:
        b = bias.cuda() if biased else None
        xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
        w, index = moe.moe_route(xd, rd, 2, b, score, renormalize)
        gx, gr = torch.autograd.grad(w, (xd, rd), g.float().cuda())
        step = 2.0 ** -8
        for a, grad, at in ((x, gx, (1, 3)), (router, gr, (4, 7)), (router, gr, (int(index[0, 0]), 2))):
            ends = []
            for sign in (1, -1):
                moved = a.clone()
                moved[at] += sign * step
                w1, i1 = moe.moe_route((moved if a is x else x).cuda(), (moved if a is router else router).cuda(), 2, b, score, renormalize)
                assert torch.equal(i1, index)
                ends.append((w1.cpu().double() * g).sum())
            # third derivatives of the scores are below 1, times |x|^3 and |router|^3; float32 weights of at most 1: 2^-24 over the step
            size = (router if a is x else x).double().abs().amax() ** 3
            assert abs((ends[0] - ends[1]) / (2 * step) - grad.cpu().double()[at]) <= step ** 2 * size * g.abs().sum() + 2.0 ** -24 / step * g.abs().sum()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_one_expert_has_a_weight_that_nothing_changes(score):
    """top_k = 1, renormalized: the weight is the scale whatever x and the router are, and their gradients are zeros."""
    x, router, _ = operands(50, 33, 264, torch.bfloat16, torch.bfloat16)
    xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
    w, index = moe.moe_route(xd, rd, 1, score=score, scale=2.5)
    assert torch.equal(index.cpu(), (x.double() @ router.double().t()).argmax(-1, keepdim=True)) and (w == 2.5).all()
    gx, gr = torch.autograd.grad(w, (xd, rd), torch.randn((50, 1), generator=torch.Generator().manual_seed(1)).cuda())
    assert not gx.any() and not gr.any()


@pytest.mark.parametrize("e,h", [(1, 8), (4, 1024), (8, 4096), (8, 7160), (13, 2056), (16, 4088), (17, 520), (33, 1016), (64, 512), (64, 1016)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("biased", [False, True])
def test_small_routers_choose_as_larger_calls_do(biased, dtype, e, h):
    """One launch for a few tokens, two for many: sums in float64 in another order, off by some 2^-50, so that the choice is the same and the weights differ by
    a unit of float32 at most."""
    from gpu_util import ggml
    k = min(3, e)
    x, router, bias = operands(2500, e, h, dtype, dtype)
    x, router, bias = x.cuda(), router.cuda(), bias.cuda() if biased else None
    assert ggml._lib.lowbit_route_workspace_bytes(7, e, h) == 0 < ggml._lib.lowbit_route_workspace_bytes(2500, e, h)
    for score in ("softmax", "sigmoid"):
        w, index = moe.moe_route(x, router, k, bias, score)
        for rows in (slice(0, 1), slice(100, 107), slice(2400, 2500)):
            ws, i = moe.moe_route(x[rows], router, k, bias, score)
            assert torch.equal(i, index[rows]) and ((ws - w[rows]).abs() <= 2.0 ** -23 * w[rows]).all()


def test_leading_dimensions_strides_and_types():
    x, router, bias = operands(24, 20, 128, torch.bfloat16, torch.bfloat16)
    w, index = moe.moe_route(x.cuda(), router.cuda(), 3, bias.cuda())
    w3, i3 = moe.moe_route(x.cuda().view(2, 3, 4, 128), router.cuda(), 3, bias.cuda())
    assert w3.shape == (2, 3, 4, 3) and torch.equal(w3.view(24, 3), w) and torch.equal(i3.view(24, 3), index)
    w1, i1 = moe.moe_route(x.cuda()[5], router.cuda(), 3, bias.cuda())
    assert torch.equal(w1, w[5]) and torch.equal(i1, index[5])
    wide = torch.zeros((24, 257), dtype=torch.bfloat16, device="cuda")
    wide[:, 1:257:2] = x.cuda()
    strided = torch.zeros((40, 128), dtype=torch.bfloat16, device="cuda")
    strided[::2] = router.cuda()
    w2, i2 = moe.moe_route(wide[:, 1:257:2], strided[::2], 3, bias.cuda().double())
    assert torch.equal(w2, w) and torch.equal(i2, index)
    w0, i0 = moe.moe_route(x.cuda()[:0], router.cuda(), 3)
    assert w0.shape == i0.shape == (0, 3) and i0.dtype == torch.int64
    # a token's choice and weights do not depend on the batch that it is in
    for m in (1, 7, 17):
        wm, im = moe.moe_route(x.cuda()[:m], router.cuda(), 3, bias.cuda())
        assert torch.equal(im, index[:m]) and torch.equal(wm, w[:m])


def test_second_derivative_and_transforms():
    x, router, _ = operands(4, 6, 16, torch.float32, torch.float32)
    xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()

    def total(a, b):
        return (moe.moe_route(a, b, 2)[0] ** 2).sum()
    gx, = torch.autograd.grad(total(xd, rd), xd, create_graph=True)
    gg, = torch.autograd.grad(gx.pow(2).sum(), rd)
    xo, ro = x.double().requires_grad_(), router.double().requires_grad_()
    go, = torch.autograd.grad((plain(xo, ro, 2)[0] ** 2).sum(), xo, create_graph=True)
    want, = torch.autograd.grad(go.pow(2).sum(), ro)
    assert (gg.cpu().double() - want).norm() <= 1e-5 * want.norm()
    fx = torch.func.grad(total)(x.cuda(), router.cuda())
    assert (fx - gx.detach()).norm() <= 1e-5 * fx.norm()
    _, tangent = torch.func.jvp(lambda a: moe.moe_route(a, router.cuda(), 2)[0], (x.cuda(),), (torch.ones_like(x).cuda(),))
    assert tangent.shape == (4, 2) and tangent.isfinite().all()
    w, index = moe.moe_route(xd, rd, 2)
    w.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        w.sum().backward()
    with torch.no_grad():
        w, _ = moe.moe_route(xd, rd, 2)
    assert not w.requires_grad


def test_a_changed_operand_is_noticed():
    x, router, _ = operands(4, 6, 16, torch.float32, torch.float32)
    xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
    w, _ = moe.moe_route(xd * 1.0, rd, 2)
    with torch.no_grad():
        rd += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()


@pytest.mark.parametrize("what", ["rows of the router", "length of its rows", "type"])
def test_replaced_data_is_noticed(what):
    x, router, _ = operands(4, 6, 32, torch.float32, torch.float32)
    xd, rd = x.cuda().requires_grad_(), router.cuda()
    w, _ = moe.moe_route(xd, rd, 2)
    rd.data = {"rows of the router": rd[:4].clone(), "length of its rows": rd[:, :16].contiguous(), "type": rd.double()}[what]
    with pytest.raises(RuntimeError, match="not what the forward found"):
        w.sum().backward()


def test_refusals():
    x, router, bias = (v.cuda() for v in operands(4, 6, 16, torch.float32, torch.float32))
    for call, why in ((lambda: moe.moe_route(x, router, 7), "top_k"), (lambda: moe.moe_route(x, router, 0), "top_k"),
                      (lambda: moe.moe_route(x, router[:, :8], 2), "hidden"), (lambda: moe.moe_route(x[:, :12], router[:, :12], 2), "multiple of 8"),
                      (lambda: moe.moe_route(x, router, 2, bias[:3]), "bias"), (lambda: moe.moe_route(x, router, 2, score="tanh"), "score"),
                      (lambda: moe.moe_route(x.double(), router, 2), "float16"), (lambda: moe.moe_route(x, torch.zeros((1025, 16), device="cuda"), 2), "1024"),
                      (lambda: moe.moe_route(x.cpu(), router, 2), "no CPU implementation"), (lambda: moe.moe_route(x, router.cpu(), 2), "one GPU")):
        with pytest.raises(RuntimeError, match=why):
            call()


@pytest.mark.parametrize("how", ["in place", "under no_grad", "through a view", "fewer of them", "another type"])
def test_changed_indices_are_noticed(how):
    """The weights' gradient goes by the choice: where a caller has changed the returned indices since (tokens dropped, an offset added) it is refused, as a
    changed operand is; a changed copy is the caller's own."""
    x, router, _ = operands(8, 6, 16, torch.float32, torch.float32)
    xd, rd, g = x.cuda().requires_grad_(), router.cuda().requires_grad_(), torch.randn((8, 2), generator=gen(3)).cuda()
    w, index = moe.moe_route(xd, rd, 2)
    want = torch.autograd.grad(w, (xd, rd), g)
    w, index = moe.moe_route(xd.view(2, 4, 16) if how == "through a view" else xd, rd, 2)
    copied = index.clone()
    copied[1] = -1
    got = torch.autograd.grad(w, (xd, rd), g.view(w.shape), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if how == "fewer of them":
        index.data = index[:, :1].contiguous()
    elif how == "another type":
        index.data = index.int()
    else:
        with torch.set_grad_enabled(how != "under no_grad"):
            index[..., 0] = (index[..., 0] + 1) % 6
    with pytest.raises(RuntimeError, match="indices.*not what the forward found" if how in ("fewer of them", "another type") else "modified by an inplace operation"):
        torch.autograd.grad(w, (xd, rd), g.view(w.shape))


@pytest.mark.parametrize("score,renormalize,biased", RULES)
@pytest.mark.parametrize("hooked", [False, True])
def test_second_derivative_of_operands_that_depend_on_each_other(hooked, score, renormalize, biased):
    """x made from the router, as below a layer that shares it: with a graph of the gradients the router's has both ways, each once, and a hook on x runs once.

    float32 roundings, each 2^-24 of what it rounds: the weights, the gradients of both operands and their sum, twice over for the second derivative,
    some ten; sums of terms of either sign that leave a sixteenth or more of them: 10 * 16 * 2^-24 = 1e-5."""
    x, router, bias = operands(5, 6, 16, torch.float32, torch.float32)
    mix, v = torch.randn((5, 6), generator=gen(4)) * 0.5, torch.randn((5, 2), generator=gen(5))
    bias = bias if biased else None
    answers, calls = [], []
    for on_gpu in (False, True):
        move = (lambda t: t.cuda()) if on_gpu else (lambda t: t.double())
        leaf, r = move(x).requires_grad_(), move(router).requires_grad_()
        inner = leaf + move(mix) @ r
        if hooked:
            inner.register_hook(lambda g: calls.append(on_gpu) or 2 * g)
        b = None if bias is None else move(bias)
        w = moe.moe_route(inner, r, 2, b, score, renormalize, 1.5)[0] if on_gpu else plain(inner, r, 2, b, score, renormalize, 1.5)[0]
        first = torch.autograd.grad((w * move(v)).square().sum(), (leaf, r), create_graph=True)
        if hooked:
            assert calls.count(on_gpu) == 1
        second = torch.autograd.grad(sum(g.square().sum() for g in first), (leaf, r))
        answers.append([t.detach().cpu().double() for t in (*first, *second)])
    for want, got in zip(*answers):
        assert (got - want).norm() <= 1e-5 * want.norm(), (got - want).norm() / want.norm()


def test_gradients_of_several_vectors_at_once():
    x, router, _ = operands(5, 6, 16, torch.float32, torch.float32)
    xd, rd = x.cuda().requires_grad_(), router.cuda().requires_grad_()
    w, _ = moe.moe_route(xd, rd, 2)
    vectors = torch.randn((3, 5, 2), generator=gen(6)).cuda()
    got = torch.autograd.grad(w, (xd, rd), vectors, retain_graph=True, is_grads_batched=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(w, (xd, rd), vectors[i], retain_graph=True)):
            assert (a[i] - b).norm() <= 1e-5 * b.norm()      # (as above: some ten float32 roundings)


def test_saved_tensors_that_hooks_move_or_a_checkpoint_makes_again():
    from torch.utils.checkpoint import checkpoint
    x, router, _ = operands(8, 6, 16, torch.bfloat16, torch.float32)
    xd, rd, g = x.cuda().requires_grad_(), router.cuda().requires_grad_(), torch.randn((8, 2), generator=gen(3)).cuda()
    want = torch.autograd.grad(moe.moe_route(xd, rd, 2)[0], (xd, rd), g)
    with torch.autograd.graph.save_on_cpu():
        w, index = moe.moe_route(xd, rd, 2)
    index.fill_(-1)                                          # (the hook's copy is the one that counts)
    for got in (torch.autograd.grad(w, (xd, rd), g), torch.autograd.grad(checkpoint(lambda a: moe.moe_route(a, rd, 2)[0], xd, use_reentrant=False), (xd, rd), g)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
