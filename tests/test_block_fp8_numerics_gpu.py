"""Block-scaled fp8: values, types and sizes at which a step's rounding shows, against 64 bits on the host."""
import pytest
import torch

import block_fp8_util as u
from ipex_llm.transformers import block_fp8 as bf

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]
ALL = HALF + [torch.float32]
IDS = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}


def ids(v):
    return IDS.get(v) if isinstance(v, torch.dtype) else None


def gen(seed):
    return torch.Generator().manual_seed(seed)


def act64(g, act):
    return g * torch.sigmoid(g) if act == 0 else g * torch.sigmoid(2 * 0.7978845608028654 * (g + 0.044715 * g ** 3))


def h_error(g, act):
    """How far, relative, h = act(g) v may be off in float32, in hardware's exp2 and reciprocal (a unit of 2^-23 each).  The exponent is off by
    its own size times the roundings that made it, half a unit each: 1.4427 g (a constant, a product), or 2.885 u of u = 0.798 (g + 0.0447 g g g)
    (three constants, five products, a sum).  Beside it: exp2 2, 1 + e 1, the reciprocal 2, two products 2, h / scale 2, units of 2^-24."""
    u_ = 0.7978845608028654 * (g + 0.044715 * g ** 3)
    return 2.0 ** -24 * (9 + (2 * g.abs() if act == 0 else 9 * 2 * u_.abs()))


def experts64(x, picks, p, gu, gus, dn, dns, act, border=0.0):
    """(result, the most it may move where h * 448 / a lies within h_error (of h and of the block's largest) and `border`, relative, of a border
    of two codes, the size of its pairs)."""
    out = torch.zeros((x.shape[0], x.shape[1]), dtype=torch.float64)
    slack, size, inter = torch.zeros_like(out), torch.zeros_like(out), gu.shape[1] // 2
    rows = u.dense(*u.quantize(x, 1), 1)
    for e in range(gu.shape[0]):
        t, j = torch.where(picks == e)
        if not t.numel():
            continue
        s = rows[t] @ u.dense(gu[e], gus[e]).t()
        h = act64(s[:, :inter], act) * s[:, inter:]
        codes, hs = u.quantize(h, 1)
        step, d, w = u.spread(hs, h.shape[0], inter, 1), u.dense(dn[e], dns[e]), p[t, j].double()[:, None]
        y = (codes * step) @ d.t()
        own = h_error(s[:, :inter], act)
        largest = torch.where(h.abs() >= 447.99 * step, own, 0.0)     # of each block: its scale's error
        block = torch.nn.functional.pad(largest, (0, -inter % 128)).unflatten(-1, (-1, 128)).amax(-1).repeat_interleave(128, -1)[:, :inter]
        wide = own + block + border
        # (a scale that is off moves every product of its block, by as much)
        off = (u.e4m3(h / step * (1 + wide)) - u.e4m3(h / step * (1 - wide))).abs() * step + (codes * step).abs() * block
        out.index_add_(0, t, y * w)
        slack.index_add_(0, t, off @ d.abs().t() * w.abs())
        size.index_add_(0, t, (y * w).abs())
    return out, slack, size


@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_gelu_of_gates_far_below_zero(dtype, tokens):
    """Gates of -5.5 to -6.5: act(g) is 1e-9 to 1e-13 of them, and the codes are made of nothing else."""
    g = gen(tokens)
    picks, p = torch.rand((tokens, 4), generator=g).argsort(dim=1)[:, :2], (torch.rand((tokens, 2), generator=g) + 0.5).to(dtype)
    x = torch.zeros((tokens, 128))
    x[:, 0], x[:, 1] = 8, 448                                # codes of themselves, scale 1
    x = x.to(dtype)
    gu, gus = u.weight(g, 512, 128, base=-6, lead=(4,))
    gate = torch.zeros((4, 256, 128))
    gate[..., 0] = -torch.randint(11, 14, (4, 256), generator=g).float()
    gu[:, :256] = gate.to(u.E4M3)                            # (g = 8 * code * 2^-4)
    gus[:, :2] = 2.0 ** -4
    dn, dns = u.random_weight(g, 128, 256, lead=(4,))
    dns *= 2.0 ** 30                                         # results within the types' range
    case = (x, picks, p, gu, gus, dn, dns)
    got = bf.block_fp8_experts(*(t.cuda() for t in case), 1).cpu().double()
    want, slack, size = experts64(*case, 1)                  # (g and u are exact: one product each)
    assert (want.abs().amax(dim=1) > 0.01).all() and slack.norm() < 0.1 * want.norm()
    unit = torch.finfo(dtype).eps / 2
    # (a result is rounded once; the second product drops bits as in any product)
    assert (got - want).norm() <= unit * want.norm() + slack.norm() + (3 ** 0.5 * 2.0 ** -13 + 2.0 ** -18) * size.norm()


def expert_case(seed, tokens, top_k, n_exp, hidden, inter, dtype):
    """Ordinary numbers, experts of which some get no token, and an index that names none."""
    g = gen(seed)
    x, p = torch.randn((tokens, hidden), generator=g).to(dtype), torch.rand((tokens, top_k), generator=g).to(dtype)
    picks = torch.rand((tokens, n_exp - 1), generator=g).argsort(dim=1)[:, :top_k]
    picks[-1, -1] = n_exp
    return x, picks, p, *u.random_weight(g, 2 * inter, hidden, lead=(n_exp,)), *u.random_weight(g, hidden, inter, lead=(n_exp,))


def near(got, case, act, dtype, drops=0.0):
    """Rounded once, sums in float32: half a unit of the type; codes of h that may lie on either side of a border, g and u being float32
    sums of a few blocks; and `drops` for what the fp8 instruction leaves out."""
    want, slack, size = experts64(*case, act, 2.0 ** -19)
    unit = torch.finfo(dtype).eps / 2
    assert (got.double().cpu() - want).norm() <= unit * want.norm() + slack.norm() + (drops + 2.0 ** -18) * size.norm()


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", [(1, 2, 4, 128, 128), (24, 3, 6, 400, 256), (64, 4, 9, 1024, 512)])
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_experts_below_a_gradient_round_once_as_the_native_call_does(dtype, tokens, top_k, n_exp, hidden, inter):
    case = expert_case(tokens, tokens, top_k, n_exp, hidden, inter, dtype)
    on_gpu = [t.cuda() for t in case]
    near(bf.block_fp8_experts(*on_gpu), case, 0, dtype, 3 ** 0.5 * 2.0 ** -13)
    for which in (0, 2):                                     # x, the routing weights
        leaves = list(on_gpu)
        leaves[which] = on_gpu[which].clone().requires_grad_()
        out = bf.block_fp8_experts(*leaves, tokens % 2)
        assert out.dtype == dtype and out.requires_grad
        near(out.detach(), case, tokens % 2, dtype)


@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_gradients_of_experts_in_16_bits(dtype):
    tokens, n_exp, hidden, inter = 60, 5, 512, 384
    case = expert_case(3, tokens, 2, n_exp, hidden, inter, dtype)
    x, picks, p, gu, gus, dn, dns = case
    leaf, weights = x.cuda().requires_grad_(), p.cuda().requires_grad_()
    v = torch.randn((tokens, hidden), generator=gen(4)).to(dtype)
    out = bf.block_fp8_experts(leaf, picks.cuda(), weights, *(t.cuda() for t in case[3:]))
    gx, gp = torch.autograd.grad(out, (leaf, weights), v.cuda())
    assert gx.dtype == dtype and gp.dtype == dtype
    x64, p64, total = x.double().requires_grad_(), p.double().requires_grad_(), torch.zeros((tokens, hidden), dtype=torch.float64)
    rows = x64 + (u.dense(*u.quantize(x, 1), 1) - x.double())        # the quantization counts as the identity
    for e in range(n_exp):
        t, j = torch.where(picks == e)
        s = rows[t] @ u.dense(gu[e], gus[e]).t()
        h = act64(s[:, :inter], 0) * s[:, inter:]
        h = h + (u.dense(*u.quantize(h.detach(), 1), 1) - h.detach())
        total = total.index_add(0, t, h @ u.dense(dn[e], dns[e]).t() * p64[t, j, None])
    wx, wp = torch.autograd.grad(total, (x64, p64), v.double())
    unit = torch.finfo(dtype).eps / 2
    # on the way to x: p grad, the gradients of h and of (g | u), a pair's rows, and their sum are rounded; to p: once, of sums in float32 (and
    # one code of h in 2^14 may be on the other side of a border: a step of 2^-3 of one of its terms, 2^-3 / sqrt(2^14) and less)
    assert (gx.double().cpu() - wx).norm() <= 5 * unit * wx.norm()
    assert (gp.double().cpu() - wp).norm() <= (unit + 2.0 ** -10) * wp.norm()
    assert (gp[-1, -1] == 0).all()                           # of a pair that goes nowhere


class _Relu(torch.nn.Module):
    def forward(self, t):
        return t.clamp(min=0)


@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_experts_that_no_kernel_takes_round_once_too(dtype):
    """An activation of another kind, and more experts for a token than the library takes."""
    case = expert_case(6, 20, 2, 5, 256, 128, dtype)
    with torch.device("meta"):
        module = bf.BlockFP8Experts(5, 256, 128, _Relu())
    for name, t in zip(("gate_up_proj", "gate_up_proj_scale_inv", "down_proj", "down_proj_scale_inv"), case[3:]):
        setattr(module, name, torch.nn.Parameter(t.cuda(), requires_grad=False))
    got = module(*(t.cuda() for t in case[:3]))
    relu = torch.zeros((20, 256), dtype=torch.float64)
    x, picks, p, gu, gus, dn, dns = case
    rows, exactly = u.dense(*u.quantize(x, 1), 1), torch.zeros((20, 256), dtype=torch.float64)
    for e in range(5):
        t, j = torch.where(picks == e)
        s = rows[t] @ u.dense(gu[e], gus[e]).t()
        y = u.dense(*u.quantize(s[:, :128].clamp(min=0) * s[:, 128:], 1), 1) @ u.dense(dn[e], dns[e]).t() * p[t, j].double()[:, None]
        exactly.index_add_(0, t, y)
        relu.index_add_(0, t, y.abs())
    unit = torch.finfo(dtype).eps / 2
    # (one code of h in 2^14 may be on the other side of a border, a step of 2^-3 of one of 128 terms)
    assert (got.double().cpu() - exactly).norm() <= unit * exactly.norm() + 2.0 ** -12 * relu.norm()
    many = expert_case(7, 3, 66, 70, 128, 128, dtype)
    near(bf.block_fp8_experts(*(t.cuda() for t in many)), many, 0, dtype)


@pytest.mark.parametrize("m", [1, 6, 40])
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_a_bias_is_added_before_the_result_is_rounded(dtype, m):
    """Of another type, strided, or one that is trained itself: sums that are exact in float32 but for the bias' own last bits."""
    g = gen(m)
    x, (w, ws) = u.activations(g, m, 512, dtype), u.weight(g, 200, 512, base=-8)
    product = x.double() @ u.dense(w, ws).t()
    xd, wd, sd = x.cuda(), w.cuda(), ws.cuda()
    long = (torch.randint(-1 << 10, 1 << 10, (200,), generator=g) * 2.0 ** -8).float()    # exact beside multiples of 2^-10
    for bias in (long, long.double()):
        assert torch.equal(bf.block_fp8_linear(xd, wd, sd, bias.cuda()).cpu(), (product + bias.double()).to(dtype))
    short = (torch.randint(-64, 65, (200,), generator=g) * 2.0 ** -6).to(dtype)
    short[3] = -float("inf")
    want = (product + short.double()).to(dtype)
    strided = torch.stack([short, short], dim=1).cuda()[:, 0]
    assert torch.equal(bf.block_fp8_linear(xd, wd, sd, strided).cpu(), want)
    v = torch.randint(-8, 9, (m, 200), generator=g).to(dtype).cuda()
    for bias in (short, long):
        leaf, row = bias.cuda().requires_grad_(), xd.clone().requires_grad_()
        for at in (xd, row):
            y = bf.block_fp8_linear(at, wd, sd, leaf)
            assert torch.equal(y.detach().cpu(), (product + bias.double()).to(dtype))
            grads = torch.autograd.grad(y, (leaf, at) if at.requires_grad else (leaf,), v)
            finite = bias.isfinite()
            assert grads[0].dtype == bias.dtype and torch.equal(grads[0].cpu()[finite], v.cpu().double().sum(0).to(bias.dtype)[finite])
            if at.requires_grad:
                assert torch.equal(grads[1].cpu(), (v.cpu().double() @ u.dense(w, ws)).to(dtype))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(short.cuda(), torch.full((200,), 2.0, dtype=dtype, device="cuda"))
        y = torch.autograd.forward_ad.unpack_dual(bf.block_fp8_linear(xd, wd, sd, dual))
    assert torch.equal(y.primal.cpu(), want) and (y.tangent[:, torch.arange(200) != 3] == 2).all()


class _Seen(torch.utils._python_dispatch.TorchDispatchMode):
    """Counts the operators that a call shows."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("weight", [False, True], ids=["rows", "weight"])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_quantizers_under_a_trace_a_dispatch_mode_and_vmap(dtype, weight):
    call = bf.block_fp8_quantize_weight if weight else bf.block_fp8_quantize
    g = gen(31)
    x, other = ((torch.randn((6, 130, 272), generator=g) * 3).to(dtype).cuda() for _ in range(2))
    want = [t.float() for t in call(x)]
    traced = torch.jit.trace(lambda t: tuple(v.float() for v in call(t)), other, check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(traced(x), want))
    with _Seen() as mode:
        got = call(x)
    assert len(mode.names) > 4 and all(torch.equal(a.float(), b) for a, b in zip(got, want))
    got = torch.func.vmap(lambda t: tuple(v.float() for v in call(t)))(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = x.float().requires_grad_()
    assert not any(t.requires_grad for t in call(leaf))


@pytest.mark.parametrize("m,n,k", u.FEW_ROWS)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_few_rows_of_every_number_of_waves(dtype, m, n, k):
    g = gen(m + n)
    x, (w, ws) = u.activations(g, m, k, dtype, spread_bits=0), u.weight(g, n, k, base=-8)
    # every partial sum is a whole multiple of the least product, 2^-9, below 2^24 of them: exact in any order
    assert (x.double().abs() @ u.dense(w, ws).abs().t()).max() < 2.0 ** 15
    want = x.double() @ u.dense(w, ws).t()
    assert torch.equal(bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu(), want.to(dtype))


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", u.FEW_PAIRS)
@pytest.mark.parametrize("dtype", HALF, ids=ids)
def test_few_pairs_of_every_number_of_waves(dtype, tokens, top_k, n_exp, hidden, inter):
    case = expert_case(hidden, tokens, top_k, n_exp, hidden, inter, dtype)       # (the last pair's index names no expert)
    near(bf.block_fp8_experts(*(t.cuda() for t in case), tokens % 2), case, tokens % 2, dtype, 3 ** 0.5 * 2.0 ** -13)


# What the fp8 instruction drops, of the result's norm: measured over three seeds and 512 x 1024 to 2048 x 4096, the largest of nine, and half
# as much again for another seed's
DROPS = {"normal": (1.6e-5, lambda x, g: x), "loud channels": (3.4e-5, lambda x, g: torch.where(torch.arange(x.shape[1]) % 97 == 0, 20 * x, x)),
         "lognormal": (5.6e-5, lambda x, g: x * torch.exp(1.5 * torch.randn(x.shape, generator=g)))}


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("kind", DROPS)
def test_what_the_fp8_instruction_drops(kind, m):
    """Seen past the result's own rounding: a bias that takes all but the result's last bits away, ahead of the one rounding."""
    g = gen(11)
    n, k = 1000, 4096
    w, ws = u.random_weight(g, n, k)
    x = DROPS[kind][1](torch.randn((1, k), generator=g), g).half()
    want = (u.dense(*u.quantize(x, 1), 1) @ u.dense(w, ws).t())[0]
    bias = -want.half()
    got = bf.block_fp8_linear(x.cuda().expand(m, -1).contiguous(), w.cuda(), ws.cuda(), bias.cuda()).cpu().double()
    # what is left, 2^-12 of a value, is rounded to 11 bits or to a subnormal: 2^-24 of the value, 2^-25
    limit = 1.5 * DROPS[kind][0] * want.norm() + 2.0 ** -23 * want.norm() + 2.0 ** -24 * n ** 0.5
    assert ((got - (want + bias.double())).norm(dim=1) <= limit).all()


def test_what_is_dropped_goes_by_the_terms_where_they_cancel():
    """Pairs of neighbours whose large products cancel: the loss is of the terms' size, and the result is far smaller than they are."""
    g = gen(12)
    n, k = 512, 4096
    w, ws = u.random_weight(g, n, k)
    w = w.float()
    w[:, 1::2] = -w[:, ::2]
    w[:, ::8] *= 0.5                                         # (one pair of four does not cancel)
    w, x = w.to(u.E4M3), torch.randn((1, k), generator=g)
    x[:, 1::2] = x[:, ::2]
    x = x.half()
    xv, wv = u.dense(*u.quantize(x, 1), 1), u.dense(w, ws)
    want, terms = (xv @ wv.t())[0], ((xv ** 2) @ (wv ** 2).t()).sqrt()
    got = bf.block_fp8_linear(x.cuda(), w.cuda(), ws.cuda(), -want.half().cuda()).cpu().double()
    off = (got - (want - want.half().double())).norm()
    assert want.norm() < 0.3 * terms.norm() and off <= 1.5 * 1.6e-5 * terms.norm() + 2.0 ** -23 * want.norm() + 2.0 ** -24 * n ** 0.5


@pytest.mark.parametrize("weight", [False, True], ids=["rows", "weight"])
def test_float32_codes_are_those_of_the_quotient_rounded_to_float32(weight):
    """Every code: the quotient is correctly rounded but for what 64 bits cannot tell, and a product with a float32 reciprocal, 1e-7 off, would
    move one of some 10^6 by a step."""
    g = gen(13)
    x = torch.randn((2048, 4096), generator=g) * torch.exp(torch.randn((2048, 1), generator=g) * 4)
    high = 128 if weight else 1
    codes, scale = bf.block_fp8_quantize_weight(x.cuda()) if weight else bf.block_fp8_quantize(x.cuda())
    _, want_scale = u.quantize(x, high)
    a = x.abs().unflatten(-1, (-1, 128)).amax(-1)
    a = (a.unflatten(0, (-1, 128)).amax(1) if weight else a).clamp(min=2.0 ** -100)
    q = (x.double() * 448 / u.spread(a, *x.shape, high)).float()
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(codes.cpu().double(), u.e4m3(q.double()))
    # what a quotient in float32 throughout would make of these numbers (here, on the host: another answer)
    cheap = x * (1.0 / want_scale.repeat_interleave(high, 0).repeat_interleave(128, 1)[:x.shape[0], :x.shape[1]])
    assert not torch.equal(u.e4m3(cheap.double().clamp(-448, 448)), u.e4m3(q.double()))


def test_operators_repeat_themselves_bit_for_bit():
    g = gen(14)
    for m, n, k in ((1, 512, 4096), (40, 1000, 4096), (300, 1030, 2048), (700, 640, 8192)):
        (w, ws), x = u.random_weight(g, n, k), torch.randn((m, k), generator=g)
        w, ws, grad = w.cuda(), ws.cuda(), torch.randn((m, n), generator=g).cuda()
        for dtype in ALL:
            leaf = x.to(dtype).cuda().requires_grad_()
            first = None
            for _ in range(3):
                y = bf.block_fp8_linear(leaf, w, ws)
                both = y.detach(), torch.autograd.grad(y, leaf, grad.to(dtype))[0]
                first = first or both
                assert torch.equal(both[0], first[0]) and (dtype == torch.float32 or torch.equal(both[1], first[1]))
    for tokens, top_k, n_exp in ((1, 2, 8), (300, 2, 8), (2000, 4, 20)):
        case = [t.cuda() for t in expert_case(tokens, tokens, top_k, n_exp, 512, 256, torch.bfloat16)]
        case[1][:, 1] = case[1][:, 0]                        # the same expert twice
        first = bf.block_fp8_experts(*case)
        leaf = case[0].clone().requires_grad_()
        below = bf.block_fp8_experts(leaf, *case[1:]).detach()
        for _ in range(3):
            assert torch.equal(bf.block_fp8_experts(*case), first)
            assert torch.equal(bf.block_fp8_experts(leaf, *case[1:]).detach(), below)


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter", u.EXPERT_TILES)
def test_experts_in_tiles_of_every_form_in_float16(tokens, top_k, n_exp, hidden, inter):
    from test_block_fp8_gpu import expert_case as exact_case
    case = exact_case(tokens + 1, tokens, top_k, n_exp, hidden, inter, torch.float16)          # g and u are exact in any order
    got = bf.block_fp8_experts(*(t.cuda() for t in case), 1).cpu().double()
    want, slack, size = experts64(*case, 1)
    unit = torch.finfo(torch.float16).eps / 2
    assert (got - want).norm() <= unit * want.norm() + slack.norm() + (3 ** 0.5 * 2.0 ** -13 + 2.0 ** -18) * size.norm()
    # nobody's row is another's (of one row the instruction's loss, 3^0.5 2^-13 in the mean, may be four times that).  Results below 2^-14, of
    # tokens with a routing weight of some 1e-5, are subnormal: half a step, 2^-25, for each of the row's
    per = (got - want).norm(dim=1) - slack.norm(dim=1)
    assert (per <= (unit + 4 * 3 ** 0.5 * 2.0 ** -13) * size.norm(dim=1) + 2.0 ** -25 * hidden ** 0.5).all()


def test_more_blocks_than_a_launch_has_workgroups_for():
    """9 million weights of one block each, and 537 million rows of one block: several launches, whose parts meet without a seam."""
    n = 9_000_000
    w = (torch.arange(n * 16, device="cuda", dtype=torch.int32) % 4093 - 2046).view(n, 1, 16).bfloat16()
    codes, scale = bf.block_fp8_quantize_weight(w)
    seam = (1 << 32) // 512 - 8
    for part in (slice(0, 1000), slice(seam - 500, seam + 500), slice(n - 1000, n)):
        want, ws = u.quantize(w[part].cpu(), 128)
        assert torch.equal(codes[part].cpu().double(), want) and torch.equal(scale[part].cpu(), ws)
    del w, codes, scale
    seam = ((1 << 32) // 256 - 8) * 32
    n = seam + 3000
    x = torch.empty((n, 16), dtype=torch.bfloat16, device="cuda")
    for at in range(0, n, 1 << 26):
        part = x[at:at + (1 << 26)]
        part.copy_((torch.arange(part.numel(), device="cuda", dtype=torch.int32) % 4093 - 2046).view_as(part))
    codes, scale = bf.block_fp8_quantize(x)
    for part in (slice(0, 1000), slice(seam - 500, seam + 500), slice(n - 1000, n)):
        want, ws = u.quantize(x[part].cpu(), 1)
        assert torch.equal(codes[part].cpu().double(), want) and torch.equal(scale[part].cpu(), ws)


@pytest.mark.parametrize("tokens,top_k,n_exp,hidden,inter,parts", [(70000, 4, 5, 1040, 128, 2), (300000, 1, 3, 1552, 128, 3), (300000, 2, 3, 1296, 128, 6)])
def test_pairs_results_of_more_than_a_gib_are_summed_in_parts(tokens, top_k, n_exp, hidden, inter, parts):
    """Columns in several launches; as the same tokens in calls of their own, and as 64 bits for some."""
    assert -(-hidden // max(256, (1 << 30) // (4 * tokens * top_k) // 256 * 256)) == parts
    g = gen(hidden)
    case = list(expert_case(hidden, 600, top_k, n_exp, hidden, inter, torch.bfloat16))
    rows = torch.randint(0, 600, (tokens,), generator=g)
    rows[:600], rows[-600:] = torch.arange(600), torch.arange(600)
    on_gpu = [t.cuda() for t in case]
    got = bf.block_fp8_experts(*(t[rows.cuda()] for t in on_gpu[:3]), *on_gpu[3:])
    near(got[:600], case, 0, torch.bfloat16, 3 ** 0.5 * 2.0 ** -13)
    assert torch.equal(got, got[:600][rows.cuda()])          # (a row's sums are the same wherever it stands)


def test_tangents_through_experts():
    """Of x and of the routing weights, in float32: the formula's, the quantization counting as the identity."""
    case = expert_case(21, 12, 2, 4, 256, 128, torch.float32)
    x, picks, p, gu, gus, dn, dns = case
    g = gen(22)
    tx, tp = torch.randn(x.shape, generator=g), torch.randn(p.shape, generator=g)
    with torch.autograd.forward_ad.dual_level():
        make = torch.autograd.forward_ad.make_dual
        out = bf.block_fp8_experts(make(x.cuda(), tx.cuda()), picks.cuda(), make(p.cuda(), tp.cuda()), *(t.cuda() for t in case[3:]))
        got = torch.autograd.forward_ad.unpack_dual(out).tangent.cpu().double()
    want = torch.zeros((12, 256), dtype=torch.float64)
    rows = u.dense(*u.quantize(x, 1), 1)
    for e in range(4):
        t, j = torch.where(picks == e)
        w, d = u.dense(gu[e], gus[e]), u.dense(dn[e], dns[e])
        s, ds = rows[t] @ w.t(), tx[t].double() @ w.t()
        a, v = s[:, :128], s[:, 128:]
        slope = torch.sigmoid(a) * (1 + a * (1 - torch.sigmoid(a)))
        h, dh = act64(a, 0) * v, slope * ds[:, :128] * v + act64(a, 0) * ds[:, 128:]
        hq = u.dense(*u.quantize(h, 1), 1)
        want.index_add_(0, t, dh @ d.t() * p[t, j].double()[:, None] + hq @ d.t() * tp[t, j].double()[:, None])
    # (one code of h in 2^14 may be on the other side of a border, a step of 2^-3 of one of its terms)
    assert (got - want).norm() <= 2.0 ** -10 * want.norm()


@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_experts_with_a_gate_of_their_own_on_the_gpu(dtype):
    from test_block_fp8_cpu import FusedExperts
    from ipex_llm.transformers.convert import ggml_convert_low_bit
    fused = FusedExperts(4, 256, 128, limit=0.5, alpha=1.7).eval()
    new = ggml_convert_low_bit(torch.nn.Sequential(fused), 15, torch_dtype=dtype)[0].cuda()
    g = gen(23)
    x, p = torch.randn((20, 256), generator=g).to(dtype), torch.rand((20, 2), generator=g).to(dtype)
    picks = torch.rand((20, 4), generator=g).argsort(dim=1)[:, :2]
    got = new(x.cuda(), picks.cuda(), p.cuda()).cpu().double()
    want, size, clamped = torch.zeros((20, 256), dtype=torch.float64), torch.zeros((20, 256), dtype=torch.float64), 0
    rows = u.dense(*u.quantize(x, 1), 1)
    for e in range(4):
        t, j = torch.where(picks == e)
        s = rows[t] @ u.dense(fused.gate_up_proj[e], fused.gate_up_proj_scale_inv[e]).t()
        clamped += (s > 0.5).sum()
        y = u.dense(*u.quantize(fused._apply_gate(s), 1), 1) @ u.dense(fused.down_proj[e], fused.down_proj_scale_inv[e]).t() * p[t, j].double()[:, None]
        want.index_add_(0, t, y)
        size.index_add_(0, t, y.abs())
    assert clamped > 100
    # (codes of h: as in test_experts_that_no_kernel_takes_round_once_too)
    assert (got - want).norm() <= torch.finfo(dtype).eps / 2 * want.norm() + 2.0 ** -12 * size.norm()


@pytest.mark.parametrize("kind", ["dense", "experts"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_a_block_scaled_checkpoint_runs(dtype, kind, tmp_path):
    """Through from_pretrained, beside the dense model that holds the same numbers.  It differs by the quantization of each product's
    activations: e4m3 keeps 4 bits, 0.026 of a value in the mean, independent over seven products of one or three layers' branches."""
    from test_block_fp8_cpu import tiny_llama, write_checkpoint
    from ipex_llm.transformers import AutoModelForCausalLM
    if kind == "dense":
        model, apart = tiny_llama(), ("lm_head",)
    else:
        from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM
        torch.manual_seed(5)
        model, apart = Qwen3MoeForCausalLM(Qwen3MoeConfig(hidden_size=256, intermediate_size=384, moe_intermediate_size=128, num_experts=4,
                                                          num_experts_per_tok=4, num_hidden_layers=1, num_attention_heads=4,
                                                          num_key_value_heads=2, vocab_size=64)).eval(), ("lm_head", "mlp.gate")
    write_checkpoint(tmp_path, model, apart)
    with torch.no_grad():
        for name, v in model.named_parameters():             # what the codes stand for
            if v.dim() == 3 or (name.endswith("proj.weight") and not any(a in name for a in apart)):
                high = [v] if v.dim() == 2 else [part for w in v for part in (w.chunk(2) if name.endswith("gate_up_proj") else [w])]
                for w in high:
                    w.copy_(u.dense(*u.quantize(w, 128)))
            else:
                v.copy_(v.bfloat16())
    loaded = AutoModelForCausalLM.from_pretrained(str(tmp_path), load_in_low_bit="fp8_e4m3", torch_dtype=dtype, modules_to_not_convert=list(apart))
    loaded = loaded.cuda()
    tokens = torch.randint(0, 64, (2, 9), generator=gen(24))
    with torch.inference_mode():
        want = model(tokens).logits
        got = loaded(tokens.cuda()).logits.float().cpu()
        again = loaded.to(torch.float16)(tokens.cuda()).logits.float().cpu() if dtype == torch.float32 else loaded.half()(tokens.cuda()).logits.float().cpu()
    assert (got - want).norm() <= 0.1 * want.norm() and (again - want).norm() <= 0.1 * want.norm()
