"""Block-scaled fp8: quantizers, products, gradients and experts against 64 bits on the host."""
import copy
import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch import nn

import block_fp8_util as u
from gpu_util import DT, ggml, stream
from ipex_llm.transformers import block_fp8 as bf

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


# ---------------------------------------------------------------- quantizers

def awkward(x):
    """Rows of every kind: zeros, one value, ties of the rounding, the least and largest numbers of the type."""
    info = torch.finfo(x.dtype)
    if x.shape[0] > 6:
        x[0] = 0
        x[1] = 0
        x[1, -1] = 3.0
        x[2] = (torch.arange(x.shape[1]) % 256).to(x.dtype) * 7     # 448 / a exact for many: quotients on borders
        x[3] *= info.smallest_normal
        x[4] = info.max
        x[4, ::2] = info.tiny
        x[5, 0] = info.smallest_normal / 4
        x[5, 1:] = 0
        x[6] = torch.linspace(0, 1, x.shape[1]).to(x.dtype) * 14
    return x


@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (7, 144), (33, 1024), (130, 2112), (300, 4096)])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_quantize_rows(dtype, m, k):
    x = awkward((torch.randn((m, k), generator=gen(m)) * 3).to(dtype))
    codes, scale = bf.block_fp8_quantize(x.cuda())
    want, ws = u.quantize(x, 1)
    assert codes.dtype == u.E4M3 and codes.shape == x.shape and scale.shape == (m, u.blocks(k))
    assert torch.equal(scale.cpu(), ws)
    off = codes.cpu().double() != want
    # float32: the quotient is rounded to float32 first, which moves one of 2^20 onto a border
    assert off.float().mean() <= (0 if dtype != torch.float32 else 2.0 ** -12), off.nonzero()[:5]
    assert torch.equal(bf.block_fp8_dequantize(codes, scale).cpu().double(), (codes.cpu().float() * u.spread(scale.cpu(), m, k, 1).float()).double())


@pytest.mark.parametrize("n,k,lead", [(1, 16, ()), (128, 128, ()), (129, 144, ()), (300, 1040, ()), (1000, 512, ()), (130, 272, (3,))])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_quantize_weight(dtype, n, k, lead):
    w = (torch.randn((*lead, n, k), generator=gen(n)) * 0.02).to(dtype)
    if n > 200:
        w[..., :128, :128] = 0
    codes, scale = bf.block_fp8_quantize_weight(w.cuda())
    want, ws = u.quantize(w, 128)
    assert torch.equal(scale.cpu(), ws)
    assert (codes.cpu().double() != want).float().mean() <= (0 if dtype != torch.float32 else 2.0 ** -12)


@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_quantize_blocks_with_nan_and_infinity(dtype):
    x = torch.randn((4, 384), generator=gen(3)).to(dtype)
    x[0, 5], x[1, 200], x[1, 201], x[2, 383] = math.nan, math.inf, math.nan, -math.inf
    codes, scale = bf.block_fp8_quantize(x.cuda())
    got = bf.block_fp8_dequantize(codes, scale).cpu()
    bad = torch.zeros((4, 3), dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(got.isnan(), bad.repeat_interleave(128, dim=1))
    w, ws = u.random_weight(gen(4), 32, 384)
    y = bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu()
    assert torch.equal(y.isnan().all(dim=1), torch.tensor([True, True, True, False])) and y[3].isfinite().all()


def test_every_finite_bfloat16_rounds_to_the_nearest_code():
    """All magnitudes beside each of the mantissas that a block's largest value can have."""
    v = torch.arange(0, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for mantissa in range(0, 128, 9):
        top = torch.tensor(0x4300 + mantissa, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
        small = v[v <= top]
        x = torch.zeros(((small.numel() + 126) // 127, 128), dtype=torch.bfloat16)
        x[:, 0] = top
        x[:, 1:].reshape(-1)
        flat = torch.zeros(x.shape[0] * 127, dtype=torch.bfloat16)
        flat[:small.numel()] = small
        x[:, 1:] = flat.view(-1, 127)
        codes, _ = bf.block_fp8_quantize(x.cuda())
        assert torch.equal(codes.cpu().double(), u.quantize(x, 1)[0])


# ---------------------------------------------------------------- products

SHAPES = u.SHAPES


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_product_is_exact_where_no_order_of_summation_rounds(dtype, m, n, k):
    g = gen(m * 7 + n)
    x, (w, ws) = u.activations(g, m, k, dtype), u.weight(g, n, k, base=-8)
    bias = (torch.randint(-64, 65, (n,), generator=g) * 2.0 ** -6).to(dtype)
    want = x.double() @ u.dense(w, ws).t()
    xd, wd, sd = x.cuda(), w.cuda(), ws.cuda()
    y = bf.block_fp8_linear(xd, wd, sd)
    assert y.dtype == dtype and torch.equal(y.cpu(), want.to(dtype))
    y = bf.block_fp8_linear(xd, wd, sd, bias.cuda())
    assert torch.equal(y.cpu(), (want + bias.double()).to(dtype))


@pytest.mark.parametrize("m,n,k", u.TILES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_product_in_tiles_of_every_form(dtype, m, n, k):
    test_product_is_exact_where_no_order_of_summation_rounds(dtype, m, n, k)


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (8, 300, 1040), (40, 1000, 4096), (130, 640, 2112), (600, 1100, 2048)])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_product_of_ordinary_numbers(dtype, m, n, k):
    """2-norm of the difference.  Rounding the result: at most half a unit, u.  The fp8 instruction drops what lies 13 bits below the
    largest of a few neighbouring products: of each of up to three, evenly within 2^-13 of the largest, so that a result's error is
    sqrt(3) 2^-13 of the root of its products' squares, which is the result's own size.  Sums in float32: a rounding per block."""
    g = gen(n)
    x = torch.randn((m, k), generator=g)
    x[:, :: 97] *= 20
    x, (w, ws) = x.to(dtype), u.random_weight(g, n, k)
    want = u.dense(*u.quantize(x, 1), 1) @ u.dense(w, ws).t()
    got = bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu().double()
    unit = torch.finfo(dtype).eps / 2
    limit = unit + (3 ** 0.5 * 2.0 ** -13 if dtype != torch.float32 else 128 * 2.0 ** -24) + u.blocks(k) * 2.0 ** -24
    assert (got - want).norm() <= limit * want.norm()
    if dtype == torch.float32:                           # its codes come out of a quotient in float32: at most one of 2^20 moves
        assert (got - want).norm() <= 2e-5 * want.norm()


def test_rows_of_zeros_and_far_scales():
    g = gen(1)
    w, ws = u.weight(g, 160, 512, base=-8)
    x = u.activations(g, 70, 512, torch.float32)
    x[3] = 0
    x[4] *= 2.0 ** 60
    x[5] *= 2.0 ** -60
    x[6, 128:256] = 0
    for dtype in (torch.float32, torch.bfloat16):
        y = bf.block_fp8_linear(x.to(dtype).cuda(), w.cuda(), ws.cuda()).cpu()
        assert torch.equal(y, (x.double() @ u.dense(w, ws).t()).to(dtype))


def test_strided_unaligned_and_batched_activations():
    g = gen(2)
    w, ws = u.weight(g, 48, 256, base=-8)
    x = u.activations(g, 24, 256, torch.bfloat16)
    want = (x.double() @ u.dense(w, ws).t()).bfloat16()
    wd, sd = w.cuda(), ws.cuda()
    flat = torch.zeros(24 * 256 + 3, dtype=torch.bfloat16, device="cuda")
    flat[3:] = x.cuda().reshape(-1)
    wide = torch.zeros((24, 300), dtype=torch.bfloat16, device="cuda")
    wide[:, 17:273] = x.cuda()
    turned = x.cuda().t().contiguous().t()
    for v in (flat[3:].view(24, 256), wide[:, 17:273], turned):
        assert torch.equal(bf.block_fp8_linear(v, wd, sd).cpu(), want)
    y = bf.block_fp8_linear(x.cuda().view(2, 3, 4, 256), wd, sd)
    assert y.shape == (2, 3, 4, 48) and torch.equal(y.cpu().view(24, 48), want)
    assert torch.equal(bf.block_fp8_linear(x[0].cuda(), wd, sd).cpu(), want[0])
    assert bf.block_fp8_linear(x[:0].cuda(), wd, sd).shape == (0, 48)


@pytest.mark.parametrize("m,n,k", [(1, 33, 256), (20, 77, 400), (90, 130, 272), (300, 261, 144)])
def test_nothing_is_written_past_the_result(m, n, k):
    """y and the workspace end where the call says they do."""
    g = gen(5)
    x, (w, ws) = u.activations(g, m, k, torch.float16).cuda(), u.weight(g, n, k, base=-8)
    w, ws = w.cuda(), ws.cuda()
    need = ggml.lowbit_block_fp8_linear_workspace_bytes(DT[torch.float16], m, n, k)
    space = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    y = torch.full((m * n + 64,), float("nan"), dtype=torch.float16, device="cuda")
    ggml.lowbit_block_fp8_linear(x.data_ptr(), w.data_ptr(), ws.data_ptr(), None, y.data_ptr(), DT[torch.float16], m, n, k, space.data_ptr(), need, stream())
    assert y[m * n:].isnan().all() and (space[need:] == 0x5a).all()
    assert torch.equal(y[:m * n].view(m, n), bf.block_fp8_linear(x, w, ws))


# ---------------------------------------------------------------- gradient

BACK = u.BACK_SHAPES


@pytest.mark.parametrize("m,n,k", BACK)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_gradient_is_grad_times_the_weight(dtype, m, n, k):
    """Whole numbers times powers of two: exact in any order."""
    g = gen(m + n)
    (w, ws), x = u.weight(g, n, k, base=-8), u.activations(g, m, k, dtype).cuda().requires_grad_()
    grad = torch.randint(-16, 17, (m, n), generator=g).to(dtype)
    y = bf.block_fp8_linear(x, w.cuda(), ws.cuda())
    got, = torch.autograd.grad(y, x, grad.cuda())
    assert got.dtype == dtype and torch.equal(got.cpu(), (grad.double() @ u.dense(w, ws)).to(dtype))


@pytest.mark.parametrize("m,n,k", u.BACK_TILES)
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_gradient_in_tiles_of_every_form(dtype, m, n, k):
    test_gradient_is_grad_times_the_weight(dtype, m, n, k)


@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_gradient_of_ordinary_numbers(dtype):
    g = gen(8)
    m, n, k = 210, 900, 656
    (w, ws), x = u.random_weight(g, n, k), torch.randn((m, k), generator=g).to(dtype).cuda().requires_grad_()
    grad = (torch.randn((m, n), generator=g) * 0.05).to(dtype)
    want, size = grad.double() @ u.dense(w, ws), grad.double().abs() @ u.dense(w, ws).abs()
    got, = torch.autograd.grad(bf.block_fp8_linear(x, w.cuda(), ws.cuda()), x, grad.cuda())
    limit = want.abs() * torch.finfo(dtype).eps / 2 + size * (n + 2) * 2.0 ** -24 + torch.finfo(dtype).smallest_normal
    assert ((got.cpu().double() - want).abs() <= limit).all()


def test_gradient_against_differences():
    """Where x quantizes to itself on both sides, the product's difference over a step is the gradient's."""
    g = gen(9)
    m, n, k = 6, 80, 384
    (w, ws), x = u.weight(g, n, k, base=-8), u.activations(g, m, k, torch.float32, spread_bits=0)
    w, ws = w.cuda(), ws.cuda()
    weights = torch.randint(-4, 5, (m, n), generator=g).float().cuda()
    at = x.bfloat16().cuda().requires_grad_()
    got, = torch.autograd.grad(bf.block_fp8_linear(at, w, ws), at, weights.bfloat16())
    for row, col in [(0, 0), (1, 130), (2, 383), (5, 200), (3, 77)]:
        if x[row, col].abs() >= 8:
            continue
        up, down = x.clone(), x.clone()
        up[row, col] += 1
        down[row, col] -= 1
        slope = ((bf.block_fp8_linear(up.cuda(), w, ws) - bf.block_fp8_linear(down.cuda(), w, ws)).double() * weights.double()).sum() / 2
        assert slope.item() == got[row, col].double().item()


def test_gradient_through_broadcast_strided_and_unused_results():
    g = gen(10)
    (w, ws), x = u.weight(g, 96, 256, base=-8), u.activations(g, 12, 256, torch.bfloat16)
    w, ws, d = w.cuda(), ws.cuda(), u.dense(w, ws)
    leaf = x.cuda().requires_grad_()
    bf.block_fp8_linear(leaf.view(3, 4, 256), w, ws).sum().backward()             # a gradient of one expanded value
    assert torch.equal(leaf.grad.cpu(), d.sum(0).expand(12, 256).bfloat16())
    row = x[:1].cuda().requires_grad_()                                           # one row used many times
    bf.block_fp8_linear(row.expand(12, 256), w, ws).backward(torch.ones((96, 12), device="cuda", dtype=torch.bfloat16).t())
    assert torch.equal(row.grad.cpu(), (12 * d.sum(0)).bfloat16()[None])
    leaf = x.cuda().requires_grad_()
    y = bf.block_fp8_linear(leaf, w, ws)
    y[:, :0].sum().backward()
    assert (leaf.grad == 0).all()
    y = bf.block_fp8_linear(leaf, w, ws)
    y.sum().backward(retain_graph=True)
    first = leaf.grad.clone()
    y.sum().backward()
    assert torch.equal(leaf.grad, (first.double() * 2).bfloat16())
    out = bf.block_fp8_linear(x[:0].cuda().requires_grad_(), w, ws)
    out.sum().backward()


def test_second_derivative_and_tangent():
    g = gen(11)
    (w, ws), x = u.weight(g, 32, 128, base=0), u.activations(g, 3, 128, torch.float32, spread_bits=0)
    leaf, v = x.cuda().requires_grad_(), torch.randint(-4, 5, (3, 32), generator=g).float().cuda().requires_grad_()
    gx, = torch.autograd.grad(bf.block_fp8_linear(leaf, w.cuda(), ws.cuda()), leaf, v, create_graph=True)
    t = torch.randint(-4, 5, (3, 128), generator=g).float()
    got, = torch.autograd.grad(gx, v, t.cuda())
    want = (t.double() @ u.dense(w, ws).t()).float()
    assert torch.allclose(got.cpu(), want, rtol=1e-6, atol=1e-3)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.cuda(), t.cuda())
        y = torch.autograd.forward_ad.unpack_dual(bf.block_fp8_linear(dual, w.cuda(), ws.cuda()))
    assert torch.allclose(y.tangent.cpu(), want, rtol=1e-6, atol=1e-3)


def test_backward_writes_nothing_past_the_result():
    g = gen(12)
    m, n, k = 70, 137, 272
    w, ws = u.weight(g, n, k, base=-8)
    grad = torch.randint(-16, 17, (m, n), generator=g).bfloat16()
    wd, sd, gd = w.cuda(), ws.cuda(), grad.cuda()
    need = ggml.lowbit_block_fp8_backward_workspace_bytes(DT[torch.bfloat16], m, n, k)
    space = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    gx = torch.full((m * k + 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    ggml.lowbit_block_fp8_backward(gd.data_ptr(), wd.data_ptr(), sd.data_ptr(), gx.data_ptr(), DT[torch.bfloat16], m, n, k, space.data_ptr(), need, stream())
    assert gx[m * k:].isnan().all() and (space[need:] == 0x5a).all()
    assert torch.equal(gx[:m * k].view(m, k).cpu(), (grad.double() @ u.dense(w, ws)).bfloat16())


# ---------------------------------------------------------------- experts

def act64(g, act):
    return g * torch.sigmoid(g) if act == 0 else 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))


def experts64(x, ids_, p, gu, gus, dn, dns, act):
    """(result, the most it may move where a code of h lies within 2^-18 of a border, its pairs' sizes for the rounding of each)."""
    out = torch.zeros((x.shape[0], x.shape[1]), dtype=torch.float64)
    slack, size = torch.zeros_like(out), torch.zeros_like(out)
    inter = gu.shape[1] // 2
    for e in range(gu.shape[0]):
        t, j = torch.where(ids_ == e)
        if not t.numel():
            continue
        s = x[t].double() @ u.dense(gu[e], gus[e]).t()
        h = act64(s[:, :inter], act) * s[:, inter:]
        codes, hs = u.quantize(h, 1)
        d = u.dense(dn[e], dns[e])
        q = h * 448 / (u.spread(hs, h.shape[0], inter, 1) * 448)
        lo, hi = u.e4m3(q * (1 - 2.0 ** -18)), u.e4m3(q * (1 + 2.0 ** -18))
        y = u.dense(codes, hs, 1) @ d.t()
        w = p[t, j].double()[:, None]
        out.index_add_(0, t, y * w)
        slack.index_add_(0, t, (((hi - lo).abs() * u.spread(hs, h.shape[0], inter, 1)) @ d.abs().t()) * w.abs())
        size.index_add_(0, t, (y * w).abs())
    return out, slack, size


def expert_case(seed, tokens, top_k, n_exp, hidden, inter, dtype):
    """x and gate_up whose products are exact, so that h is the host's but for the activation's last bits."""
    g = gen(seed)
    x = u.activations(g, tokens, hidden, dtype, spread_bits=0)
    gu, gus = u.weight(g, 2 * inter, hidden, base=-10, lead=(n_exp,))
    dn, dns = u.random_weight(g, hidden, inter, lead=(n_exp,))
    picks = torch.rand((tokens, n_exp), generator=g).argsort(dim=1)[:, :top_k] if top_k <= n_exp else \
        torch.randint(0, n_exp, (tokens, top_k), generator=g)
    p = torch.rand((tokens, top_k), generator=g).to(dtype)
    return x, picks, p, gu, gus, dn, dns


def check_experts(case, dtype, act=0):
    x, picks, p, gu, gus, dn, dns = case
    got = bf.block_fp8_experts(x.cuda(), picks.cuda(), p.cuda(), gu.cuda(), gus.cuda(), dn.cuda(), dns.cuda(), act).cpu().double()
    want, slack, size = experts64(x, picks, p, gu, gus, dn, dns, act)
    unit = torch.finfo(dtype).eps / 2
    # the sum over a token's pairs is rounded to the type; the second product's instruction as in test_product_of_ordinary_numbers
    limit = unit * want.norm() + 3 ** 0.5 * 2.0 ** -13 * size.norm() + slack.norm() + 2.0 ** -18 * size.norm()
    assert (got - want).norm() <= limit
    # nobody's row is another's: the same per token, with the statistics of a row
    per = (got - want).norm(dim=1) - slack.norm(dim=1)
    assert (per <= (unit + 4 * 3 ** 0.5 * 2.0 ** -13) * size.norm(dim=1) + 1e-30).all()
    return got


EXPERTS = u.EXPERTS


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", EXPERTS)
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_experts(dtype, tokens, top_k, n_exp, hidden, inter):
    check_experts(expert_case(tokens + hidden, tokens, top_k, n_exp, hidden, inter, dtype), dtype, act=tokens % 2)


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", u.EXPERT_TILES)
def test_experts_in_tiles_of_every_form(tokens, top_k, n_exp, hidden, inter):
    check_experts(expert_case(tokens, tokens, top_k, n_exp, hidden, inter, torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize("tokens", [1, 3, 50, 1500])
def test_experts_skip_indices_that_name_none_and_experts_without_rows(tokens):
    case = list(expert_case(4, tokens, 3, 6, 256, 256, torch.bfloat16))
    case[1] = torch.where(case[1] == 2, torch.tensor(4), case[1])
    case[1][0, 0], case[1][-1, -1] = -1, 6
    if tokens > 2:
        case[1][1] = torch.tensor([7, -5, 2 ** 40])          # a token that goes nowhere
    got = check_experts(case, torch.bfloat16)
    if tokens > 2:
        assert (got[1] == 0).all()


def test_experts_all_rows_to_one_expert_and_the_same_expert_twice():
    case = list(expert_case(5, 140, 2, 9, 256, 128, torch.float16))
    case[1] = torch.full((140, 2), 7)
    check_experts(case, torch.float16)


def test_experts_index_and_weight_types():
    case = list(expert_case(6, 20, 2, 4, 128, 128, torch.bfloat16))
    base = bf.block_fp8_experts(*[t.cuda() for t in case])
    for pt in (torch.float32, torch.float16):
        other = list(case)
        other[2] = case[2].to(pt)
        if torch.equal(other[2].double(), case[2].double()):
            assert torch.equal(bf.block_fp8_experts(*[t.cuda() for t in other]), base)
    other = list(case)
    other[1] = case[1].int()
    assert torch.equal(bf.block_fp8_experts(*[t.cuda() for t in other]), base)
    none = bf.block_fp8_experts(case[0][:0].cuda(), case[1][:0].cuda(), case[2][:0].cuda(), *[t.cuda() for t in case[3:]])
    assert none.shape == (0, 128)


def test_experts_gradients_run_expert_by_expert():
    case = expert_case(7, 24, 2, 4, 256, 128, torch.float32)
    x, picks, p, gu, gus, dn, dns = case
    x, p = x.cuda().requires_grad_(), p.cuda().requires_grad_()
    w = [t.cuda() for t in (gu, gus, dn, dns)]
    v = torch.randn((24, 256), generator=gen(1))
    gx, gp = torch.autograd.grad(bf.block_fp8_experts(x, picks.cuda(), p, *w), (x, p), v.cuda())
    # the formula's, on the host: the quantization of x and of h counts as the identity
    x64, p64 = case[0].double().requires_grad_(), case[2].double().requires_grad_()
    out = torch.zeros((24, 256), dtype=torch.float64)
    for e in range(4):
        t, j = torch.where(picks == e)
        s = x64[t] @ u.dense(gu[e], gus[e]).t()
        h = act64(s[:, :128], 0) * s[:, 128:]
        hq = h + (u.dense(*u.quantize(h.detach(), 1), 1) - h).detach()
        out = out.index_add(0, t, (hq @ u.dense(dn[e], dns[e]).t()) * p64[t, j, None])
    wx, wp = torch.autograd.grad(out, (x64, p64), v.double())
    # float32 throughout but for codes of h next to a border, one of some 2^18: a step of 2^-3 of one of 128 terms
    assert (gx.cpu().double() - wx).norm() <= 1e-3 * wx.norm() and (gp.cpu().double() - wp).norm() <= 1e-3 * wp.norm()


# ---------------------------------------------------------------- what a product must keep apart

@pytest.mark.parametrize("m,n,k", [(1, 33, 144), (3, 130, 272), (14, 130, 272), (40, 257, 400), (300, 129, 144), (1347, 1459, 144)])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_nan_stays_in_its_row_and_column(dtype, m, n, k):
    """NaN in a row of x (a padded batch's), in the weight's last row and in a block's scale: the results that they belong to and no others,
    also where a tile or a block ends inside."""
    g = gen(m + k)
    x, (w, ws) = u.activations(g, m, k, dtype), u.weight(g, n, k, base=-8)
    grad = torch.randint(-8, 9, (m, n), generator=g).to(dtype)
    want, back = x.double() @ u.dense(w, ws).t(), grad.double() @ u.dense(w, ws)
    bad_x, bad_w, bad_g = x.clone(), w.clone(), grad.clone()
    bad_w.view(torch.uint8)[n - 1, k - 1] = 0x7f
    if m > 1:
        bad_x[m - 1, k - 1], bad_g[m - 1, n - 1] = math.nan, math.nan
    leaf = bad_x.cuda().requires_grad_()
    y = bf.block_fp8_linear(leaf, bad_w.cuda(), ws.cuda())
    got, = torch.autograd.grad(y, leaf, bad_g.cuda())
    want[:, n - 1], back[:, k - 1] = math.nan, math.nan
    if m > 1:
        want[m - 1], back[m - 1] = math.nan, math.nan
    assert same(y.detach().cpu(), want.to(dtype)) and same(got.cpu(), back.to(dtype))
    scale = ws.clone()
    scale[-1, -1] = math.nan
    y = bf.block_fp8_linear(x.cuda(), w.cuda(), scale.cuda()).cpu()
    first = (n - 1) // 128 * 128
    assert y[:, first:].isnan().all() and torch.equal(y[:, :first], (x.double() @ u.dense(w, ws).t()).to(dtype)[:, :first])


def test_scales_of_zero_and_negative_ones():
    g = gen(21)
    x, (w, ws) = u.activations(g, 50, 512, torch.bfloat16), u.weight(g, 300, 512, base=-8)
    ws[0, 1], ws[1], ws[2, 3] = 0, 0, -ws[2, 3]
    assert torch.equal(bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu(), (x.double() @ u.dense(w, ws).t()).bfloat16())


# ---------------------------------------------------------------- offsets past 32 bits

def test_weights_of_more_than_2_to_32_codes():
    n, k, tail = (1 << 18) + 200, 16384, 200                     # the last 200 rows lie past 2^32
    g = gen(22)
    w, ws = torch.zeros((n, k), dtype=torch.uint8, device="cuda").view(u.E4M3), torch.zeros((u.blocks(n), k // 128), device="cuda")
    part, scale = u.weight(g, tail, k, base=-10)
    w[n - tail:].copy_(part.cuda())
    ws[-2:].copy_(scale.cuda())
    assert (n - tail) % 128 == 0
    for m in (1, 40, 300):
        x = u.activations(g, m, k, torch.bfloat16, spread_bits=0).cuda()
        y = bf.block_fp8_linear(x, w, ws)
        assert torch.equal(y[:, n - tail:], bf.block_fp8_linear(x, part.cuda(), scale.cuda())) and not y[:, :n - tail].any()
        del y
    x = u.activations(g, 33, k, torch.bfloat16, spread_bits=0).cuda().requires_grad_()
    grad = torch.zeros((33, n), dtype=torch.bfloat16, device="cuda")
    grad[:, n - tail:] = torch.randint(-8, 9, (33, tail), generator=g).cuda().bfloat16()
    got, = torch.autograd.grad(bf.block_fp8_linear(x, w, ws), x, grad)
    assert torch.equal(got.cpu(), (grad[:, n - tail:].cpu().double() @ u.dense(part, scale)).bfloat16())
    dense = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    dense[n - 7:] = torch.randn((7, k), generator=g).cuda().bfloat16()
    codes, scales = bf.block_fp8_quantize_weight(dense)
    last, last_scale = bf.block_fp8_quantize_weight(dense[n - 72:])
    assert torch.equal(codes[n - 72:].view(torch.uint8), last.view(torch.uint8)) and torch.equal(scales[-1:], last_scale)
    codes, scales = bf.block_fp8_quantize(dense)
    last, last_scale = bf.block_fp8_quantize(dense[n - 7:])
    assert torch.equal(codes[n - 7:].view(torch.uint8), last.view(torch.uint8)) and torch.equal(scales[n - 7:], last_scale)


def test_results_of_more_than_2_to_32_bytes():
    g = gen(23)
    m, n, k = 150000, 16384, 128                                 # y: 4.9 GB
    w, ws = (t.cuda() for t in u.weight(g, n, k, base=-8))
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    tail = u.activations(g, 300, k, torch.bfloat16).cuda()
    x[m - 300:] = tail
    y = bf.block_fp8_linear(x, w, ws)
    assert torch.equal(y[m - 300:], bf.block_fp8_linear(tail, w, ws)) and not y[:m - 300].any()
    del y
    # the gradient of as many values: x [m, n], a weight [k, n]
    w, ws = (t.cuda() for t in u.weight(g, k, n, base=-8))
    x = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda").requires_grad_()
    grad = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    grad[m - 300:] = torch.randint(-8, 9, (300, k), generator=g).cuda().bfloat16()
    got, = torch.autograd.grad(bf.block_fp8_linear(x, w, ws), x, grad)
    assert torch.equal(got[m - 300:].cpu(), (grad[m - 300:].cpu().double() @ u.dense(w.cpu(), ws.cpu())).bfloat16()) and not got[:m - 300].any()


def test_experts_whose_weights_pass_2_to_32_codes():
    g = gen(24)
    n_exp, hidden, inter = 70, 4096, 8192                        # gate_up 4.7e9 codes, down 2.3e9
    small = expert_case(25, 4, 2, 2, hidden, inter, torch.bfloat16)
    big = []
    for t in small[3:]:
        whole = torch.zeros((n_exp, *t.shape[1:]), dtype=torch.uint8 if t.dtype == u.E4M3 else t.dtype, device="cuda")
        whole = whole.view(u.E4M3) if t.dtype == u.E4M3 else whole
        whole[n_exp - 2:].copy_(t.cuda())
        big.append(whole)
    for tokens in (1, 50):
        x = u.activations(g, tokens, hidden, torch.bfloat16, spread_bits=0).cuda()
        picks = torch.randint(0, 2, (tokens, 2), generator=g).cuda()
        p = torch.rand((tokens, 2), generator=g).bfloat16().cuda()
        got = bf.block_fp8_experts(x, picks + n_exp - 2, p, *big)
        want = bf.block_fp8_experts(x, picks, p, *(t.cuda() for t in small[3:]))
        # (another kernel may run the smaller case: each rounded once, sums in another order)
        assert (got.double() - want.double()).norm() <= 2.1 * 2.0 ** -8 * want.double().norm() and want.any()


# ---------------------------------------------------------------- streams, graphs, together

def test_another_stream_and_many_at_once():
    g = gen(13)
    w, ws = (t.cuda() for t in u.weight(g, 512, 1024, base=-8))
    xs = [u.activations(g, m, 1024, torch.bfloat16).cuda() for m in (1, 30, 300)]
    want = [bf.block_fp8_linear(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append((i, bf.block_fp8_linear(xs[(i + i // 3) % 3], w, ws)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[(i + i // 3) % 3])


def test_threads_with_streams_of_their_own():
    g = gen(17)
    w, ws = (t.cuda() for t in u.weight(g, 512, 1024, base=-8))
    cases = []
    for m in (2, 24, 70, 300):
        x = u.activations(g, m, 1024, torch.bfloat16).cuda()
        ex = [t.cuda() for t in expert_case(m, m, 2, 4, 256, 128, torch.bfloat16)]
        grad = torch.randint(-8, 9, (m, 512), generator=g).bfloat16().cuda()
        cases.append((x, ex, grad))

    def all_of(x, ex, grad):
        leaf = x.clone().requires_grad_()
        y = bf.block_fp8_linear(leaf, w, ws)
        return y.detach(), torch.autograd.grad(y, leaf, grad)[0], bf.block_fp8_experts(*ex), bf.block_fp8_quantize(x)[1]
    want = [all_of(*c) for c in cases]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [all_of(*cases[i]) for _ in range(10)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(a, b) for one in got for a, b in zip(one, want[i]))
    with ThreadPoolExecutor(len(cases)) as pool:
        assert all(pool.map(run, range(len(cases))))


@pytest.mark.parametrize("m", [1, 20, 200])
def test_two_captured_graphs_replayed_with_eager_work_between(m):
    g = gen(14)
    w, ws = (t.cuda() for t in u.weight(g, 384, 512, base=-8))
    case = expert_case(15, m, 2, 4, 256, 128, torch.bfloat16)
    ex = [t.cuda() for t in case]
    x = u.activations(g, m, 512, torch.bfloat16).cuda()

    def both():
        return bf.block_fp8_linear(x, w, ws), bf.block_fp8_experts(*ex), *bf.block_fp8_quantize(x)
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
        x.copy_(u.activations(gen(20 + i), m, 512, torch.bfloat16))
        ex[0].copy_(u.activations(gen(30 + i), m, 256, torch.bfloat16, spread_bits=0))
        for t in [t for o in outs for t in o]:
            t.view(torch.uint8).fill_(0x7b)
        graphs[i % 2].replay()
        graphs[(i + 1) % 2].replay()
        torch.cuda.synchronize()
        want = both()
        for o in outs:
            assert all(same(a.float(), b.float()) for a, b in zip(o, want))


def test_training_step_captured():
    g = gen(16)
    w, ws = (t.cuda() for t in u.weight(g, 256, 384, base=-8))
    x = u.activations(g, 40, 384, torch.bfloat16).cuda().requires_grad_()
    grad = torch.randint(-8, 9, (40, 256), generator=g).bfloat16().cuda()

    def step():
        return torch.autograd.grad(bf.block_fp8_linear(x, w, ws), x, grad)[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        grad.copy_(torch.randint(-8, 9, (40, 256), generator=gen(40 + i)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


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


class Experts(nn.Module):
    def __init__(self, n_exp, hidden, inter):
        super().__init__()
        self.gate_up_proj = nn.Parameter(torch.randn(n_exp, 2 * inter, hidden) * 0.05)
        self.down_proj = nn.Parameter(torch.randn(n_exp, hidden, inter) * 0.05)
        self.act_fn = nn.SiLU()

    def forward(self, x, ids_, p):
        out = torch.zeros_like(x)
        for e in range(self.gate_up_proj.shape[0]):
            t, j = torch.where(ids_ == e)
            g, v = (x[t] @ self.gate_up_proj[e].t()).chunk(2, dim=-1)
            out.index_add_(0, t, (self.act_fn(g) * v) @ self.down_proj[e].t() * p[t, j, None])
        return out


@pytest.mark.parametrize("rows", [1, 5, 90])
def test_a_converted_model_runs_saves_loads_and_trains(rows, tmp_path):
    from ipex_llm import optimize_model
    from ipex_llm.optimize import load_low_bit
    torch.manual_seed(3)
    dense = Block(256, 384, 4).eval()
    x = torch.randn((1, rows, 256), generator=gen(1))
    # against the dense model: e4m3 keeps 4 bits, half a step is 2^-4 of a value, a quarter of that in the mean; six products one after
    # the other, errors of their many terms independent
    want = dense(x).detach()

    model = optimize_model(copy.deepcopy(dense), "fp8_e4m3", block_fp8=True)
    assert type(model.gate_proj) is bf.BlockFP8Linear and type(model.experts) is bf.BlockFP8Experts
    model = model.to(torch.bfloat16).cuda()
    assert model.gate_proj.weight.dtype == u.E4M3 and model.gate_proj.weight_scale_inv.dtype == torch.float32
    assert model.up_proj.bias.dtype == torch.bfloat16
    with torch.inference_mode():
        got = model(x.bfloat16().cuda())
    assert (got.float().cpu() - want).norm() <= 0.1 * want.norm()
    model.save_low_bit(str(tmp_path))
    again = load_low_bit(Block(256, 384, 4), str(tmp_path)).eval().to(torch.bfloat16).cuda()
    assert type(again.router) is bf.BlockFP8Linear
    with torch.inference_mode():
        assert torch.equal(again(x.bfloat16().cuda()), got)
    # training: the gradient of the input against the dequantized model's, both quantizing nothing on the way back
    model.train()
    leaf = x.bfloat16().cuda().requires_grad_()
    model(leaf).float().square().sum().backward()
    ref = x.clone().requires_grad_()
    dense(ref).square().sum().backward()
    assert leaf.grad.isfinite().all() and (leaf.grad.float().cpu() - ref.grad).norm() <= 0.2 * ref.grad.norm()


def test_a_block_scaled_checkpoint_layer_keeps_its_codes():
    from ipex_llm.transformers.convert import ggml_convert_low_bit
    g = gen(17)
    w, ws = u.random_weight(g, 200, 272)
    lin = nn.Linear(272, 200, bias=False)
    lin.weight = nn.Parameter(w, requires_grad=False)
    lin.weight_scale_inv = nn.Parameter(ws, requires_grad=False)
    model = ggml_convert_low_bit(nn.Sequential(lin), 15).cuda()
    assert type(model[0]) is bf.BlockFP8Linear and torch.equal(model[0].weight.cpu().float(), w.float())
    x = torch.randn((9, 272), generator=g)
    assert torch.equal(model(x.cuda()), bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda()))


@pytest.mark.parametrize("tokens,top_k,n_exp,apart", [(200, 8, 160, 0), (401, 4, 2, 0), (3200, 1, 400, 0), (3201, 1, 400, 0), (1600, 2, 321, 0), (1600, 2, 319, 0),
                                                      (1600, 1, 1, 0), (300, 8, 2100, 0), (800, 4, 4096, 0), (801, 4, 2100, 1), (1025, 4, 9, 1)])
def test_experts_sorted_in_every_way(tokens, top_k, n_exp, apart):
    """Pairs counted each by a wave, sorted by one workgroup, or counted and placed by two launches, at the borders between them, some ids naming none."""
    assert ggml.lowbit_block_fp8_experts_plan(tokens, top_k, n_exp, 16, 128)[3] == apart
    case = list(expert_case(tokens + n_exp, tokens, top_k, n_exp, 16, 128, torch.bfloat16))
    case[1][::7, 0], case[1][5::11, -1] = -1, n_exp
    case[1][3] = 2 ** 33
    got = check_experts(case, torch.bfloat16)
    assert (got[3] == 0).all()
