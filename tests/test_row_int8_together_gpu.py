"""Row-scaled int8 as it is used: strides and biases, what may not be written, large offsets, streams, threads, graphs, whole models, a run of all of it."""
import copy
import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch import nn

import row_int8_util as u
from gpu_util import DT, ggml, stream
from ipex_llm.transformers import moe, row_int8 as ri

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]
ALL = HALF + [torch.float32]
IDS = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}


def ids(v):
    return IDS.get(v) if isinstance(v, torch.dtype) else None


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    """Equal values, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def whole(g, n, k, lead=()):
    """A weight whose scales are powers of two: with whole numbers for a gradient every product and sum is exact."""
    return torch.randint(-127, 128, (*lead, n, k), generator=g).to(torch.int8), torch.exp2(torch.randint(-10, -6, (*lead, n), generator=g).float())


def back(grad, w, ws):
    return (grad.double() * ws.double()) @ w.double()


def expert_case(seed, tokens, top_k, n_exp, hidden, inter, dtype):
    g = gen(seed)
    x = torch.randn((tokens, hidden), generator=g).to(dtype)
    index = torch.randint(0, n_exp, (tokens, top_k), generator=g)
    p = torch.rand((tokens, top_k), generator=g).to(dtype)
    return [t.cuda() for t in (x, index, p, *u.weight(g, 2 * inter, hidden, (n_exp,), 2 / hidden ** 0.5), *u.weight(g, hidden, inter, (n_exp,)))]


# ---------------------------------------------------------------- arguments

@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_strided_unaligned_and_batched_activations(dtype):
    g = gen(2)
    w, ws = u.weight(g, 48, 256)
    x = torch.randn((24, 256), generator=g).to(dtype)
    want, codes, scale = u.product(x, w, ws), *u.quantize(x)
    wd, sd = w.cuda(), ws.cuda()
    flat = torch.zeros(24 * 256 + 3, dtype=dtype, device="cuda")
    flat[3:] = x.cuda().reshape(-1)
    wide = torch.zeros((24, 300), dtype=dtype, device="cuda")
    wide[:, 17:273] = x.cuda()
    for v in (flat[3:].view(24, 256), wide[:, 17:273], x.cuda().t().contiguous().t()):
        assert torch.equal(ri.row_int8_linear(v, wd, sd).cpu(), want)
        got = ri.row_int8_quantize(v)
        assert torch.equal(got[0].cpu().long(), codes) and torch.equal(got[1].cpu(), scale)
    y = ri.row_int8_linear(x.cuda().view(2, 3, 4, 256), wd, sd)
    assert y.shape == (2, 3, 4, 48) and torch.equal(y.cpu().view(24, 48), want)
    assert torch.equal(ri.row_int8_linear(x[0].cuda(), wd, sd).cpu(), want[0])
    c, s = ri.row_int8_quantize(x.cuda().view(2, 12, 256))
    assert c.shape == (2, 12, 256) and s.shape == (2, 12)
    assert torch.equal(ri.row_int8_product(c, s, wd, sd, dtype=dtype).view(24, 48).cpu(), want)
    # codes and scales that are strided views, and codes off their 16 bytes
    held = torch.zeros((24, 300), dtype=torch.int8, device="cuda")
    held[:, 5:261] = c.view(24, 256)
    far = torch.zeros((24, 2), device="cuda")
    far[:, 1] = s.view(24)
    assert torch.equal(ri.row_int8_product(held[:, 5:261], far[:, 1], wd, sd, dtype=dtype).cpu(), want)
    assert ri.row_int8_linear(x[:0].cuda(), wd, sd).shape == (0, 48) and ri.row_int8_quantize(x[:0].cuda())[1].shape == (0,)
    assert ri.row_int8_product(c[:0], s[:0], wd, sd).shape == (0, 12, 48)


@pytest.mark.parametrize("m", [1, 9, 70, 300])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_biases(dtype, m):
    """Of x's type, of another one, strided, and one that wants a gradient."""
    g = gen(m)
    (w, ws), x = u.weight(g, 100, 144), torch.randn((m, 144), generator=g).to(dtype)
    bias = torch.randn(100, generator=g).to(dtype)
    wd, sd, xd, bd = w.cuda(), ws.cuda(), x.cuda(), bias.cuda()
    want = u.product(x, w, ws, bias)
    assert torch.equal(ri.row_int8_linear(xd, wd, sd, bd).cpu(), want)
    spread = torch.zeros((100, 3), dtype=dtype, device="cuda")
    spread[:, 1] = bd
    assert torch.equal(ri.row_int8_linear(xd, wd, sd, spread[:, 1]).cpu(), want)
    assert torch.equal(ri.row_int8_product(*ri.row_int8_quantize(xd), wd, sd, spread[:, 1], dtype=dtype).cpu(), want)
    for other in ALL:
        v = bias.to(other)
        codes, xs = u.quantize(x)
        steps = (u.sums(codes, w).float() * xs.unsqueeze(-1) * ws + v.float()).to(dtype)
        assert torch.equal(ri.row_int8_linear(xd, wd, sd, v.cuda()).cpu(), steps)
        assert torch.equal(ri.row_int8_product(*ri.row_int8_quantize(xd), wd, sd, v.cuda(), dtype=dtype).cpu(), steps)
    trained, leaf = bd.clone().requires_grad_(), xd.clone().requires_grad_()
    y = ri.row_int8_linear(leaf, wd, sd, trained)
    assert torch.equal(y.detach().cpu(), want)
    grad = torch.randint(-4, 5, (m, 100), generator=g).to(dtype)
    gb, = torch.autograd.grad(y, trained, grad.cuda())
    assert torch.equal(gb.cpu(), grad.double().sum(0).to(dtype))


def test_scales_of_zero_and_negative_ones():
    g = gen(21)
    for m in (2, 20, 50, 300):
        x, (w, ws) = torch.randn((m, 512), generator=g).bfloat16(), u.weight(g, 300, 512)
        ws[0], ws[1], ws[2] = 0, -ws[1], 2.0 ** -130
        assert torch.equal(ri.row_int8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu(), u.product(x, w, ws))


@pytest.mark.parametrize("m,n,k", [(1, 33, 144), (3, 130, 272), (14, 130, 272), (40, 257, 400), (300, 129, 144), (1347, 1459, 144)])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_nan_stays_in_its_row_and_column(dtype, m, n, k):
    """NaN in a row of x and of the gradient (a padded batch's), and in a column's scale: the results that they belong to and no others."""
    g = gen(m + k)
    x, (w, ws) = torch.randn((m, k), generator=g).to(dtype), whole(g, n, k)
    grad = torch.randint(-8, 9, (m, n), generator=g).to(dtype)
    want, first = u.product(x, w, ws), back(grad, w, ws)
    x[m - 1, k - 1], grad[m - 1, n - 1] = math.nan, math.nan
    leaf = x.cuda().requires_grad_()
    y = ri.row_int8_linear(leaf, w.cuda(), ws.cuda())
    got, = torch.autograd.grad(y, leaf, grad.cuda())
    want[m - 1], first[m - 1] = math.nan, math.nan
    assert same(y.detach().cpu(), want) and same(got.cpu(), first.to(dtype))
    ws[n - 1] = math.nan
    y = ri.row_int8_linear(leaf.detach(), w.cuda(), ws.cuda()).cpu()
    want[:, n - 1] = math.nan
    assert same(y, want)


@pytest.mark.parametrize("m", [1, 3, 12, 30, 70, 300, 1200])
def test_codes_of_minus_128(m):
    """The quantizer makes none, a checkpoint may hold them."""
    g = gen(m)
    x, (w, ws) = torch.randn((m, 272), generator=g).bfloat16(), whole(g, 200, 272)
    w[torch.rand(w.shape, generator=g) < 0.3] = -128
    grad = torch.randint(-8, 9, (m, 200), generator=g).bfloat16()
    leaf = x.cuda().requires_grad_()
    y = ri.row_int8_linear(leaf, w.cuda(), ws.cuda())
    assert torch.equal(y.detach().cpu(), u.product(x, w, ws))
    assert torch.equal(torch.autograd.grad(y, leaf, grad.cuda())[0].cpu(), back(grad, w, ws).bfloat16())


def test_tokens_whose_indices_name_no_expert_get_zeros_whatever_they_hold():
    x, index, p, *weights = expert_case(2, 5, 2, 4, 64, 32, torch.float32)
    x[1], x[2, 3] = math.nan, math.inf
    index[:3] = 9
    for leaf in (x, x.clone().requires_grad_()):
        y = ri.row_int8_experts(leaf, index, p, *weights)
        assert not y[:3].any() and y[3:].isfinite().all() and y[3:].any()
    index[:] = -1
    leaf, q = x.clone().requires_grad_(), p.clone().requires_grad_()
    y = ri.row_int8_experts(leaf, index, q, *weights)
    assert not y.any() and not ri.row_int8_experts(x, index, p, *weights).any()
    gx, gp = torch.autograd.grad(y.sum(), (leaf, q))
    assert not gx.any() and not gp.any()


# ---------------------------------------------------------------- nothing is written past a result

@pytest.mark.parametrize("m,n,k", [(1, 33, 256), (5, 40, 272), (20, 77, 400), (90, 130, 272), (300, 261, 144), (2, 16, 16384)])
def test_linear_product_and_gradient_write_where_they_say(m, n, k):
    g = gen(5)
    dtype = torch.float16
    x, (w, ws) = torch.randn((m, k), generator=g).to(dtype).cuda(), u.weight(g, n, k)
    w, ws, dt = w.cuda(), ws.cuda(), DT[dtype]
    codes, scale = ri.row_int8_quantize(x)
    grad = torch.randn((m, n), generator=g).to(dtype).cuda()
    need = {"linear": ggml._lib.lowbit_row_int8_linear_workspace_bytes(dt, m, n, k), "product": ggml._lib.lowbit_row_int8_product_workspace_bytes(dt, m, n, k),
            "backward": ggml._lib.lowbit_row_int8_backward_workspace_bytes(dt, m, n, k)}
    space = torch.full((max(need.values()) + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full((max(m * n, m * k) + 64,), float("nan"), dtype=dtype, device="cuda")
    want = ri.row_int8_linear(x, w, ws)
    leaf = x.clone().requires_grad_()
    first, = torch.autograd.grad(ri.row_int8_linear(leaf, w, ws), leaf, grad)
    at = (space.data_ptr(),)

    def clean(name, values, result):
        assert out[values:].isnan().all() and torch.equal(out[:values].view_as(result), result)
        assert (space[need[name]:] == 0x5a).all()
        space.fill_(0x5a)
        out.fill_(float("nan"))
    ggml.lowbit_row_int8_linear(x.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), dt, m, n, k, *at, need["linear"], stream())
    clean("linear", m * n, want)
    ggml.lowbit_row_int8_product(codes.data_ptr(), scale.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), dt, m, n, k, *at, need["product"], stream())
    clean("product", m * n, want)
    ggml.lowbit_row_int8_backward(grad.data_ptr(), w.data_ptr(), ws.data_ptr(), out.data_ptr(), dt, m, n, k, *at, need["backward"], stream())
    clean("backward", m * k, first)


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", [(1, 2, 8, 144, 48), (3, 2, 8, 272, 144), (40, 2, 5, 272, 80), (700, 3, 9, 144, 48)])
def test_experts_router_and_layer_write_where_they_say(tokens, top_k, n_exp, hidden, inter):
    dtype, lib = torch.bfloat16, ggml._lib
    x, index, p, gu, gs, dn, ds = expert_case(3, tokens, top_k, n_exp, hidden, inter, dtype)
    router = (torch.randn((n_exp, hidden), generator=gen(4)) / 8).to(dtype).cuda()
    p, dt = p.float(), DT[dtype]
    w, i = moe.moe_route(x, router, top_k)
    out = torch.full((tokens * hidden + 64,), float("nan"), dtype=dtype, device="cuda")
    need = lib.lowbit_row_int8_experts_workspace_bytes(tokens, top_k, n_exp, hidden, inter)
    whole_need = lib.lowbit_row_int8_moe_workspace_bytes(tokens, top_k, n_exp, hidden, inter)
    route_need = lib.lowbit_route_workspace_bytes(tokens, n_exp, hidden)
    space = torch.full((max(need, whole_need, route_need) + 4096,), 0x5a, dtype=torch.uint8, device="cuda")

    def clean(size, want):
        assert out[tokens * hidden:].isnan().all() and torch.equal(out[:tokens * hidden].view(tokens, hidden), want)
        assert (space[size:] == 0x5a).all()
        space.fill_(0x5a)
        out.fill_(float("nan"))
    weights = (gu.data_ptr(), gs.data_ptr(), dn.data_ptr(), ds.data_ptr(), space.data_ptr())
    assert lib.lowbit_row_int8_experts(x.data_ptr(), index.data_ptr(), p.data_ptr(), DT[torch.float32], tokens, top_k, n_exp, *weights, need, out.data_ptr(), dt,
                                       hidden, inter, 0, stream()) == 0
    clean(need, ri.row_int8_experts(x, index, p, gu, gs, dn, ds))
    assert lib.lowbit_row_int8_moe(x.data_ptr(), router.data_ptr(), dt, None, tokens, top_k, n_exp, 0, 1, 1.0, *weights, whole_need, out.data_ptr(), dt,
                                   hidden, inter, 0, stream()) == 0
    clean(whole_need, ri.row_int8_moe(x, router, top_k, gu, gs, dn, ds))
    rw, ri_ = torch.full((tokens * top_k + 64,), float("nan"), device="cuda"), torch.full((tokens * top_k + 64,), -7, device="cuda")
    assert lib.lowbit_route(x.data_ptr(), dt, router.data_ptr(), dt, None, tokens, n_exp, hidden, top_k, 0, 1, 1.0, rw.data_ptr(), ri_.data_ptr(), None,
                            space.data_ptr(), route_need, stream()) == 0
    assert rw[tokens * top_k:].isnan().all() and (ri_[tokens * top_k:] == -7).all() and (space[route_need:] == 0x5a).all()
    assert torch.equal(rw[:tokens * top_k].view(tokens, top_k), w) and torch.equal(ri_[:tokens * top_k].view(tokens, top_k), i)


# ---------------------------------------------------------------- gradients as autograd asks for them

def test_gradient_through_broadcast_strided_and_unused_results():
    g = gen(10)
    (w, ws), x = whole(g, 96, 256), torch.randn((12, 256), generator=g).bfloat16()
    d = w.double() * ws.double().unsqueeze(-1)
    w, ws = w.cuda(), ws.cuda()
    leaf = x.cuda().requires_grad_()
    ri.row_int8_linear(leaf.view(3, 4, 256), w, ws).sum().backward()              # a gradient of one expanded value
    assert torch.equal(leaf.grad.cpu(), d.sum(0).expand(12, 256).bfloat16())
    row = x[:1].cuda().requires_grad_()                                           # one row used many times: the sum of rounded gradients
    ri.row_int8_linear(row.expand(12, 256), w, ws).backward(torch.ones((96, 12), device="cuda", dtype=torch.bfloat16).t())
    off = (row.grad.cpu().double() - 12 * d.sum(0)).abs()
    assert (off <= 12 * 2.0 ** -8 * 2 * d.sum(0).abs() + 1e-30).all()
    leaf = x.cuda().requires_grad_()
    y = ri.row_int8_linear(leaf, w, ws)
    y[:, :0].sum().backward()
    assert (leaf.grad == 0).all()
    y = ri.row_int8_linear(leaf, w, ws)
    y.sum().backward(retain_graph=True)
    first = leaf.grad.clone()
    y.sum().backward()
    assert torch.equal(leaf.grad, (first.double() * 2).bfloat16())
    ri.row_int8_linear(x[:0].cuda().requires_grad_(), w, ws).sum().backward()


def test_second_derivative_tangent_and_transforms():
    g = gen(11)
    (w, ws), x = whole(g, 32, 128), torch.randn((3, 128), generator=g)
    d = w.double() * ws.double().unsqueeze(-1)
    wd, sd = w.cuda(), ws.cuda()
    leaf, v = x.cuda().requires_grad_(), torch.randint(-4, 5, (3, 32), generator=g).float().cuda().requires_grad_()
    gx, = torch.autograd.grad(ri.row_int8_linear(leaf, wd, sd), leaf, v, create_graph=True)
    t = torch.randint(-4, 5, (3, 128), generator=g).float()
    got, = torch.autograd.grad(gx, v, t.cuda())
    want = (t.double() @ d.t()).float()
    # (float32 sums of 128 terms, in torch's order)
    close = dict(rtol=1e-5, atol=128 * 2.0 ** -24 * float((t.double().abs() @ d.abs().t()).max()))
    assert torch.allclose(got.cpu(), want, **close)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.cuda(), t.cuda())
        y = torch.autograd.forward_ad.unpack_dual(ri.row_int8_linear(dual, wd, sd))
    assert torch.allclose(y.tangent.cpu(), want, **close)
    plain = ri.row_int8_linear(x.cuda(), wd, sd)
    grad = torch.func.grad(lambda a: (ri.row_int8_linear(a, wd, sd) * v.detach()).sum())(x.cuda())
    assert torch.allclose(grad.cpu(), back(v.detach().cpu(), w, ws).float(), rtol=1e-5, atol=32 * 2.0 ** -24 * float(back(v.detach().cpu().abs(), w.abs(), ws).max()))
    each = torch.func.vmap(lambda a: ri.row_int8_linear(a, wd, sd))(x.cuda())
    assert (each - plain).norm() <= 1e-5 * plain.norm()


def test_no_rows_carry_gradients_of_zero():
    g = gen(14)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    router = torch.randn((4, 64), generator=g).cuda().requires_grad_()
    bias = torch.randn(32, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    (w, ws), (gu, gus), (d, ds) = (tuple(t.cuda() for t in u.weight(g, n, k, lead)) for n, k, lead in ((32, 64, ()), (96, 64, (4,)), (64, 48, (4,))))
    p, index = moe.moe_route(x, router, 2)
    experts = ri.RowInt8Experts(4, 64, 48, torch.nn.functional.silu)
    for out, shape, leaves in ((ri.row_int8_linear(x, w, ws, bias), (0, 32), (x, bias)), (p, (0, 2), (x, router)),
                               (ri.row_int8_experts(x, index, p, gu, gus, d, ds), (0, 64), (x, router)), (experts(x, index, p), (0, 64), (x, router)),
                               (ri.row_int8_moe(x, router, 2, gu, gus, d, ds), (0, 64), (x, router))):
        assert out.shape == shape
        for leaf, grad in zip(leaves, torch.autograd.grad(out.sum(), leaves, retain_graph=True)):
            assert grad.shape == leaf.shape and not grad.any()


def test_a_changed_weight_is_noticed_and_trained_scales_are_refused():
    g = gen(12)
    (w, ws), x = u.weight(g, 32, 128), torch.randn((3, 128), generator=g)
    w, ws, leaf = w.cuda(), ws.cuda(), x.cuda().requires_grad_()
    y = ri.row_int8_linear(leaf, w, ws)
    with torch.no_grad():
        w += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="frozen"):
        ri.row_int8_linear(leaf, w, ws.requires_grad_())
    with torch.no_grad():
        ri.row_int8_linear(leaf, w, ws)


@pytest.mark.parametrize("what", ["fewer rows", "shorter rows", "other codes", "other scales"])
def test_replaced_data_is_noticed(what):
    g = gen(13)
    (w, ws), x = u.weight(g, 48, 128), torch.randn((3, 128), generator=g)
    w, ws, leaf = w.cuda(), ws.cuda(), x.cuda().requires_grad_()
    y = ri.row_int8_linear(leaf, w, ws)
    if what == "fewer rows":
        w.data, ws.data = w[:32].clone(), ws[:32].clone()
    elif what == "shorter rows":
        w.data = w[:, :64].contiguous()
    elif what == "other codes":
        w.data = w.float()
    else:
        ws.data = ws.half()
    with pytest.raises(RuntimeError, match="not what the forward found"):
        y.sum().backward()


def test_rows_of_several_launches():
    rows, few = (1 << 22) + 5, 7                                 # a launch takes 2^22
    x = torch.zeros((rows, 16), dtype=torch.float16, device="cuda")
    at = torch.cat([torch.arange(few), torch.arange((1 << 22) - few, rows)])
    given = torch.randn((len(at), 16), generator=gen(24)).half()
    x[at.cuda()] = given.cuda()
    codes, scale = ri.row_int8_quantize(x)
    want, by = u.quantize(given)
    assert torch.equal(codes[at.cuda()].cpu(), want.to(torch.int8)) and torch.equal(scale[at.cuda()].cpu(), by)
    assert int(codes.count_nonzero()) == int(want.count_nonzero())


# ---------------------------------------------------------------- offsets past 32 bits

def test_weights_of_more_than_2_to_32_codes():
    n, k, tail = (1 << 18) + 200, 16384, 200                     # the last 200 rows lie past 2^32
    g = gen(22)
    w, ws = torch.zeros((n, k), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    part, scale = whole(g, tail, k)
    w[n - tail:].copy_(part.cuda())
    ws[n - tail:].copy_(scale.cuda())
    for m in (1, 12, 40, 300):
        x = torch.randn((m, k), generator=g).bfloat16().cuda()
        y = ri.row_int8_linear(x, w, ws)
        assert torch.equal(y[:, n - tail:], ri.row_int8_linear(x, part.cuda(), scale.cuda())) and not y[:, :n - tail].any()
        del y
    x = torch.randn((33, k), generator=g).bfloat16().cuda().requires_grad_()
    grad = torch.zeros((33, n), dtype=torch.bfloat16, device="cuda")
    grad[:, n - tail:] = torch.randint(-8, 9, (33, tail), generator=g).cuda().bfloat16()
    got, = torch.autograd.grad(ri.row_int8_linear(x, w, ws), x, grad)
    assert torch.equal(got.cpu(), back(grad[:, n - tail:].cpu(), part, scale).bfloat16())
    dense = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    dense[n - 7:] = torch.randn((7, k), generator=g).cuda().bfloat16()
    codes, scales = ri.row_int8_quantize(dense)
    last, last_scale = ri.row_int8_quantize(dense[n - 7:])
    assert torch.equal(codes[n - 7:], last) and torch.equal(scales[n - 7:], last_scale) and not codes[:n - 7].any()


def test_results_of_more_than_2_to_32_bytes():
    g = gen(23)
    m, n, k = 150000, 16384, 128                                 # y: 4.9 GB
    w, ws = (t.cuda() for t in whole(g, n, k))
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn((300, k), generator=g).bfloat16().cuda()
    x[m - 300:] = tail
    y = ri.row_int8_linear(x, w, ws)
    assert torch.equal(y[m - 300:], ri.row_int8_linear(tail, w, ws)) and not y[:m - 300].any()
    del y
    # the gradient of as many values: x [m, n], a weight [k, n]
    w, ws = (t.cuda() for t in whole(g, k, n))
    x = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda").requires_grad_()
    grad = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    grad[m - 300:] = torch.randint(-8, 9, (300, k), generator=g).cuda().bfloat16()
    got, = torch.autograd.grad(ri.row_int8_linear(x, w, ws), x, grad)
    assert torch.equal(got[m - 300:].cpu(), back(grad[m - 300:].cpu(), w.cpu(), ws.cpu()).bfloat16()) and not got[:m - 300].any()


def test_experts_whose_weights_pass_2_to_32_codes():
    g = gen(24)
    n_exp, hidden, inter = 70, 4096, 8192                        # gate_up 4.7e9 codes, down 2.3e9
    small = expert_case(25, 4, 2, 2, hidden, inter, torch.bfloat16)[3:]
    big = []
    for t in small:
        all_of = torch.zeros((n_exp, *t.shape[1:]), dtype=t.dtype, device="cuda")
        all_of[n_exp - 2:].copy_(t)
        big.append(all_of)
    for tokens in (1, 50):
        x = torch.randn((tokens, hidden), generator=g).bfloat16().cuda()
        picks = torch.randint(0, 2, (tokens, 2), generator=g).cuda()
        p = torch.rand((tokens, 2), generator=g).bfloat16().cuda()
        got, want = ri.row_int8_experts(x, picks + n_exp - 2, p, *big), ri.row_int8_experts(x, picks, p, *small)
        # (another kernel may run the smaller case, whose float32 steps differ: each rounded once, and codes of h that lie on a border)
        assert (got.double() - want.double()).norm() <= 2.1 * 2.0 ** -8 * want.double().norm() and want.any()


# ---------------------------------------------------------------- streams, threads, graphs

def test_another_stream_and_many_at_once():
    g = gen(13)
    w, ws = (t.cuda() for t in u.weight(g, 512, 1024))
    xs = [torch.randn((m, 1024), generator=g).bfloat16().cuda() for m in (1, 8, 30, 300)]
    want = [ri.row_int8_linear(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 3]):
            got.append((i, ri.row_int8_linear(xs[i // 2 % 4], w, ws)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i // 2 % 4])


def test_threads_with_streams_of_their_own():
    g = gen(17)
    w, ws = (t.cuda() for t in u.weight(g, 512, 1024))
    router = (torch.randn((4, 256), generator=g) / 16).bfloat16().cuda()
    cases = []
    for m in (1, 2, 9, 24, 70, 300):
        cases.append((torch.randn((m, 1024), generator=g).bfloat16().cuda(), expert_case(m, m, 2, 4, 256, 128, torch.bfloat16),
                      torch.randn((m, 512), generator=g).bfloat16().cuda()))

    def all_of(x, ex, grad):
        leaf = x.clone().requires_grad_()
        y = ri.row_int8_linear(leaf, w, ws)
        gate = router.clone().requires_grad_()
        weights, index = moe.moe_route(ex[0], gate, 2)
        codes, scale = ri.row_int8_quantize(x)
        return (y.detach(), torch.autograd.grad(y, leaf, grad)[0], ri.row_int8_experts(*ex), ri.row_int8_moe(ex[0], router, 2, *ex[3:]), index, weights.detach(),
                torch.autograd.grad(weights.square().sum(), gate)[0], codes, scale, ri.row_int8_product(codes, scale, w, ws))
    want = [all_of(*c) for c in cases]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [all_of(*cases[i]) for _ in range(10)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(a, b) for one in got for a, b in zip(one, want[i]))
    with ThreadPoolExecutor(len(cases)) as pool:
        assert all(pool.map(run, range(len(cases))))


@pytest.mark.parametrize("m", [1, 8, 20, 200])
def test_two_captured_graphs_replayed_with_eager_work_between(m):
    g = gen(14)
    w, ws = (t.cuda() for t in u.weight(g, 384, 512))
    ex = expert_case(15, m, 2, 4, 256, 128, torch.bfloat16)
    router = (torch.randn((6, 512), generator=g) / 16).bfloat16().cuda()
    x = torch.randn((m, 512), generator=g).bfloat16().cuda()

    def both():
        codes, scale = ri.row_int8_quantize(x)
        return [ri.row_int8_linear(x, w, ws), ri.row_int8_product(codes, scale, w, ws), ri.row_int8_experts(*ex), codes, scale, *moe.moe_route(x, router, 2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    for i in range(4):
        x.copy_(torch.randn((m, 512), generator=gen(20 + i)).bfloat16())
        ex[0].copy_(torch.randn((m, 256), generator=gen(30 + i)).bfloat16())
        for t in [t for o in outs for t in o]:
            t.view(torch.uint8).fill_(0x7b)
        graphs[i % 2].replay()
        graphs[(i + 1) % 2].replay()
        torch.cuda.synchronize()
        want = both()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_training_step_captured(m):
    """A linear, a router and experts with their gradients in one graph, replayed with other values."""
    g = gen(16)
    w, ws = (t.cuda() for t in u.weight(g, 256, 384))
    router = (torch.randn((8, 384), generator=g) / 16).bfloat16().cuda().requires_grad_()
    x = torch.randn((m, 384), generator=g).bfloat16().cuda().requires_grad_()
    grad, top = torch.randn((m, 256), generator=g).bfloat16().cuda(), torch.randn((m, 2), generator=g).cuda()

    def step():
        y = ri.row_int8_linear(x, w, ws)
        weights, _ = moe.moe_route(x, router, 2)
        return torch.autograd.grad((y, weights), (x, router), (grad, top))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        grad.copy_(torch.randn((m, 256), generator=gen(40 + i)).bfloat16())
        with torch.no_grad():
            x.copy_(torch.randn((m, 384), generator=gen(50 + i)).bfloat16())
        for t in out:
            t.view(torch.uint8).fill_(0x7b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("tokens", [1, 6, 64])
def test_a_run_of_all_of_them(tokens):
    """One quantized activation through two projections, a router, experts and a linear, with the gradient of what it started from, against the same
    steps in 64 bits whose quantizers count as the identity for the gradient.

    float32: values that pass from one operator to the next are off by some 2^-22, so that of 64 * 256 codes less than one lies on the other
    side of a border; one code of a token moves its row by 1 / (127 * 0.3 * sqrt(256)) = 1.6e-3 of it, the whole by that over sqrt(tokens), and the
    products of the gradient by as much: 2e-3 bounds a run of one token, too."""
    g = gen(tokens)
    hidden, inter, n_exp = 256, 144, 6
    mats = {n: u.weight(g, *s) for n, s in dict(q=(hidden, hidden), k=(128, hidden), out=(hidden, hidden)).items()}
    mats["up"], mats["down"] = u.weight(g, 2 * inter, hidden, (n_exp,), 0.2), u.weight(g, hidden, inter, (n_exp,), 0.2)
    router, x = torch.randn((n_exp, hidden), generator=g) / 2, torch.randn((tokens, hidden), generator=g)
    dev = {n: tuple(t.cuda() for t in v) for n, v in mats.items()}
    rd, xd = router.cuda().requires_grad_(), x.cuda().requires_grad_()

    q = ri.row_int8_linear(xd, *dev["q"])
    codes, scale = ri.row_int8_quantize(xd.detach())
    assert torch.equal(ri.row_int8_product(codes, scale, *dev["q"], dtype=torch.float32), q.detach())
    k = ri.row_int8_product(codes, scale, *dev["k"], dtype=torch.float32)
    assert torch.equal(k, ri.row_int8_linear(xd, *dev["k"]).detach())
    weights, index = moe.moe_route(q, rd, 2)
    y = ri.row_int8_experts(q, index, weights, *dev["up"], *dev["down"])
    with torch.no_grad():
        assert torch.equal(ri.row_int8_moe(q, rd, 2, *dev["up"], *dev["down"]), ri.row_int8_experts(q, index, weights, *dev["up"], *dev["down"]))
    z = ri.row_int8_linear(y + q, *dev["out"])
    got = torch.autograd.grad(z.square().sum(), (xd, rd))

    def linear(a, w, ws):
        c, s = u.quantize(a.detach().float())
        values = c.double() * s.double().unsqueeze(-1)
        return (a + (values - a).detach()) @ (w.double() * ws.double().unsqueeze(-1)).t()
    xo, ro = x.double().requires_grad_(), router.double().requires_grad_()
    qo = linear(xo, *mats["q"])
    top = (qo @ ro.t()).topk(2, dim=-1)
    assert torch.equal(top.indices, index.cpu())
    p, yo = torch.softmax(top.values, -1), torch.zeros((tokens, hidden), dtype=torch.float64)
    for e in range(n_exp):
        t, j = torch.where(top.indices == e)
        a, b = linear(qo[t], mats["up"][0][e], mats["up"][1][e]).chunk(2, dim=-1)
        yo = yo.index_add(0, t, linear(nn.functional.silu(a) * b, mats["down"][0][e], mats["down"][1][e]) * p[t, j].unsqueeze(-1))
    zo = linear(yo + qo, *mats["out"])
    want = torch.autograd.grad(zo.square().sum(), (xo, ro))
    assert (z.detach().cpu().double() - zo.detach()).norm() <= 2e-3 * zo.norm()
    for a, b in zip(got, want):
        assert (a.cpu().double() - b).norm() <= 2e-3 * b.norm() and b.any()


class Experts(nn.Module):
    def __init__(self, n_exp, hidden, inter):
        super().__init__()
        self.gate_up_proj = nn.Parameter(torch.randn(n_exp, 2 * inter, hidden) * 0.05)
        self.down_proj = nn.Parameter(torch.randn(n_exp, hidden, inter) * 0.05)
        self.act_fn = nn.SiLU()

    def forward(self, x, index, p):
        out = torch.zeros_like(x)
        for e in range(self.gate_up_proj.shape[0]):
            t, j = torch.where(index == e)
            g, v = (x[t] @ self.gate_up_proj[e].t()).chunk(2, dim=-1)
            out.index_add_(0, t, (self.act_fn(g) * v) @ self.down_proj[e].t() * p[t, j, None])
        return out


class Block(nn.Module):
    """What stands around the operators in a model: a norm, a gated MLP, a mixture of experts."""

    def __init__(self, hidden, inter, n_exp):
        super().__init__()
        self.norm = nn.LayerNorm(hidden)
        self.gate_proj, self.up_proj = nn.Linear(hidden, inter, bias=False), nn.Linear(hidden, inter, bias=True)
        self.down_proj = nn.Linear(inter, hidden, bias=False)
        self.router = nn.Linear(hidden, n_exp)
        self.experts = Experts(n_exp, hidden, inter)

    def forward(self, x):
        h = self.norm(x)
        x = x + self.down_proj(nn.functional.silu(self.gate_proj(h)) * self.up_proj(h))
        flat = self.norm(x).reshape(-1, x.shape[-1])
        p, e = torch.softmax(self.router(flat).float(), dim=-1).topk(2, dim=-1)
        return x + self.experts(flat, e, p.to(x.dtype)).view_as(x)


@pytest.mark.parametrize("rows", [1, 5, 90])
def test_a_converted_model_runs_saves_loads_and_trains(rows, tmp_path):
    """Against the dense model: a code is off by up to half a step of a / 127, 1 / sqrt(12) at rms with a of some 3 to 4 standard deviations: 0.9 % of a
    value, both operands 1.3 % of a product, of which there are five one after the other or side by side, and bf16's 2^-9: under 5 % of a result,
    the gradient twice that."""
    from ipex_llm import optimize_model
    from ipex_llm.optimize import load_low_bit
    torch.manual_seed(3)
    dense = Block(256, 384, 4).eval()
    x = torch.randn((1, rows, 256), generator=gen(1))
    want = dense(x).detach()
    model = optimize_model(copy.deepcopy(dense), "sym_int8", row_int8=True)
    assert type(model.gate_proj) is ri.RowInt8Linear and type(model.experts) is ri.RowInt8Experts
    codes, scale = u.quantize(dense.down_proj.weight.data)
    assert torch.equal(model.down_proj.weight.long(), codes) and torch.equal(model.down_proj.weight_scale, scale)
    model = model.to(torch.bfloat16).cuda()
    assert model.gate_proj.weight.dtype == torch.int8 and model.gate_proj.weight_scale.dtype == torch.float32
    assert model.up_proj.bias.dtype == torch.bfloat16
    with torch.inference_mode():
        got = model(x.bfloat16().cuda())
    assert (got.float().cpu() - want).norm() <= 0.05 * want.norm()
    model.save_low_bit(str(tmp_path))
    again = load_low_bit(Block(256, 384, 4), str(tmp_path)).eval().to(torch.bfloat16).cuda()
    assert type(again.router) is ri.RowInt8Linear and type(again.experts) is ri.RowInt8Experts
    with torch.inference_mode():
        assert torch.equal(again(x.bfloat16().cuda()), got)
    model.train()
    leaf = x.bfloat16().cuda().requires_grad_()
    model(leaf).float().square().sum().backward()
    ref = x.clone().requires_grad_()
    dense(ref).square().sum().backward()
    assert leaf.grad.isfinite().all() and (leaf.grad.float().cpu() - ref.grad).norm() <= 0.1 * ref.grad.norm()


def test_a_layer_computes_what_its_function_does():
    g = gen(3)
    lin = nn.Linear(144, 100)
    lin.weight = nn.Parameter(u.weight(g, 100, 144)[0], requires_grad=False)
    lin.weight_scale = nn.Parameter(torch.rand((100, 1), generator=g) * 1e-3, requires_grad=False)
    layer = ri.RowInt8Linear.from_linear(lin).cuda()
    x = torch.randn((7, 144), generator=g).bfloat16()
    want = u.product(x, lin.weight.data, lin.weight_scale.data[:, 0], lin.bias.data.bfloat16())
    assert torch.equal(layer(x.cuda()).cpu(), want)
    layer.compute_dtype = torch.float16
    y = layer.train()(x.cuda())
    assert y.dtype == torch.bfloat16 and (y.float().cpu() - want.float()).norm() <= 2.0 ** -7 * want.float().norm()
    layer.mp_group = object()
    with pytest.raises(RuntimeError, match="mp_group"):
        layer(x.cuda())


def test_transforms_over_weights_biases_and_codes():
    """Stacked weights by vmap, as of experts: each as by itself.  Both factors of a product, its sum of 128 and the scales in float32 in another order: five roundings
    of 2^-24 of a product and sqrt(128) of its sum's, 1e-6 of the result's norm."""
    g = gen(31)
    (w, ws), x = u.weight(g, 32, 128, (3,)), torch.randn((5, 128), generator=g)
    w, ws, x, bias = w.cuda(), ws.cuda(), x.cuda(), torch.randn((3, 32), generator=g).cuda()
    want = torch.stack([ri.row_int8_linear(x, w[i], ws[i], bias[i]) for i in range(3)])
    got = torch.func.vmap(lambda a, s, b: ri.row_int8_linear(x, a, s, b))(w, ws, bias)
    assert (got - want).norm() <= 1e-6 * want.norm()
    turned = torch.func.vmap(lambda a, s, b: ri.row_int8_linear(x, a, s, b), in_dims=(2, 1, 1))(w.permute(1, 2, 0).contiguous(), ws.t().contiguous(), bias.t().contiguous())
    assert (turned - want).norm() <= 1e-6 * want.norm()
    only = torch.func.vmap(lambda b: ri.row_int8_linear(x, w[0], ws[0], b))(bias)
    assert (only - (want[0] - bias[0] + bias[:, None])).norm() <= 1e-6 * want.norm()
    codes, xs = ri.row_int8_quantize(x)
    got = torch.func.vmap(lambda a, s, b: ri.row_int8_product(codes, xs, a, s, b, torch.float32))(w, ws, bias)
    assert (got - want).norm() <= 1e-6 * want.norm()
    got = torch.func.vmap(lambda c, s: ri.row_int8_product(c, s, w[0], ws[0], dtype=torch.float32))(codes, xs)
    assert (got - (want[0] - bias[0])).norm() <= 1e-6 * want.norm()


def test_backwards_under_a_transform_or_a_mode():
    """Several vectors at once, and a dispatch mode around the backward only: by the dense product, sums of 48 in float32 (as above)."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watching(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    g = gen(32)
    (w, ws), leaf, v = u.weight(g, 48, 128), torch.randn((3, 128), generator=g), torch.randn((4, 3, 48), generator=g)
    leaf, w, ws, v = leaf.cuda().requires_grad_(), w.cuda(), ws.cuda(), v.cuda()
    y = ri.row_int8_linear(leaf, w, ws)
    want = torch.stack([torch.autograd.grad(y, leaf, v[i], retain_graph=True)[0] for i in range(4)])
    got, = torch.autograd.grad(y, leaf, v, retain_graph=True, is_grads_batched=True)
    assert (got - want).norm() <= 1e-6 * want.norm()
    with Watching():
        got, = torch.autograd.grad(y, leaf, v[0])
    assert (got - want[0]).norm() <= 1e-6 * want[0].norm()


def test_codes_of_more_than_one_launch():
    """Rows of 2^17 - 16 codes, which are copied to whole blocks, 2^32 pieces of 16 of them and more: rows of several launches, at both sides of a launch's end."""
    k, rows = (1 << 17) - 16, (1 << 19) + 3
    free = torch.cuda.mem_get_info()[0] / 2 ** 30
    if free < 150:
        pytest.skip(f"needs 150 GiB, {free:.0f} are free")
    g = gen(33)
    at = torch.tensor([0, 1, (1 << 18) - 1, 1 << 18, (1 << 19) - 1, 1 << 19, rows - 1])
    given, (w, ws) = torch.randint(-127, 128, (len(at), k), generator=g, dtype=torch.int8), u.weight(g, 17, k)
    codes, xs = torch.zeros((rows, k), dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda")
    for i, row in enumerate(at.tolist()):
        codes[row] = given[i].cuda()
    y = ri.row_int8_product(codes, xs, w.cuda(), ws.cuda(), dtype=torch.float32)
    assert torch.equal(y[at.cuda()].cpu(), u.sums(given, w).float() * ws)
    assert int((y != 0).any(dim=1).sum()) == len(at)
    del codes, y
    torch.cuda.empty_cache()


def test_a_layer_keeps_its_bias():
    """A float32 bias meets rows of any type, in that type, and stays what it was."""
    g = gen(41)
    lin = nn.Linear(144, 100)
    (codes, scale), x = u.weight(g, 100, 144), torch.randn((7, 144), generator=g)
    lin.weight, lin.weight_scale = nn.Parameter(codes, requires_grad=False), nn.Parameter(scale, requires_grad=False)
    bias = lin.bias.data.clone()
    layer = ri.RowInt8Linear.from_linear(lin).cuda().eval()
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        assert torch.equal(layer(x.to(dtype).cuda()).cpu(), u.product(x.to(dtype), codes, scale, bias.to(dtype)))
        assert layer.bias.dtype == torch.float32 and torch.equal(layer.bias.cpu(), bias)


def test_parts_added_in_more_than_one_launch():
    """The longest row goes in parts (any codes), whose sums are added four results a thread, 2^31 threads a launch: rows 65536 on of 2^17 results each are the second's."""
    k, n, m = 1 << 17, 1 << 17, 65600
    free = torch.cuda.mem_get_info()[0] / 2 ** 30
    if free < 150:
        pytest.skip(f"needs 150 GiB, {free:.0f} are free")
    g = gen(34)
    rows, cols = torch.tensor([0, 1, 65535, 65536, m - 1]), torch.tensor([0, 5, n - 1])
    a, b = torch.randint(-128, 128, (len(rows), k), generator=g, dtype=torch.int8), torch.randint(-128, 128, (len(cols), k), generator=g, dtype=torch.int8)
    a[3], b[2] = -128, -128
    codes, w = (torch.zeros((r, k), dtype=torch.int8, device="cuda") for r in (m, n))
    for i, row in enumerate(rows.tolist()):
        codes[row] = a[i].cuda()
    for i, col in enumerate(cols.tolist()):
        w[col] = b[i].cuda()
    y = ri.row_int8_product(codes, torch.ones(m, device="cuda"), w, torch.full((n,), 0.5, device="cuda"), dtype=torch.bfloat16)
    got = y[rows.cuda()][:, cols.cuda()].cpu()
    assert torch.equal(got, (u.sums(a, b).float() * 0.5).bfloat16()) and got[3, 2] == 2.0 ** 30
    assert int(y[rows.cuda()].count_nonzero()) == int(got.count_nonzero()) and not y[2:65535:1013].any() and not y[65537:m - 1].any()
    del codes, w, y
    torch.cuda.empty_cache()
