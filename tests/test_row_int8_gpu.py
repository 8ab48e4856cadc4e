"""Row-scaled int8: quantizer, products and gradients against whole numbers and 64 bits on the host."""
import math

import pytest
import torch

import row_int8_util as u
from gpu_util import DT, ggml, stream
from ipex_llm.transformers import row_int8 as ri

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


# ---------------------------------------------------------------- quantizer

def awkward(x):
    """Rows of every kind: zeros, one value, ties of the rounding, the least and largest numbers of the type."""
    info = torch.finfo(x.dtype)
    if x.shape[0] > 7:
        x[0] = 0
        x[1] = 0
        x[1, -1] = 3.0
        x[2] = (torch.arange(x.shape[1]) % 255 - 127).to(x.dtype)           # codes themselves
        x[3] *= info.smallest_normal
        x[4] = info.max
        x[4, ::2] = info.tiny
        x[5, 0] = info.smallest_normal / 4
        x[5, 1:] = 0
        x[6] = (torch.arange(x.shape[1]) % 255 - 127).to(x.dtype) / 2       # every other one half way between two codes
        x[6, 0] = 127
        x[7] = torch.linspace(-1, 1, x.shape[1]).to(x.dtype) * 14
    return x


@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (9, 144), (33, 1024), (10, 1040), (130, 2112), (300, 4096), (9, 4112), (8, 8208), (8, 28672), (8, 40016)])
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_quantize(dtype, m, k):
    x = awkward((torch.randn((m, k), generator=gen(m)) * 3).to(dtype))
    codes, scale = ri.row_int8_quantize(x.cuda())
    want, ws = u.quantize(x)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scale.shape == (m,)
    assert torch.equal(scale.cpu(), ws)
    assert torch.equal(codes.cpu().long(), want)
    assert torch.equal(ri.row_int8_dequantize(codes, scale).cpu(), codes.cpu().float() * ws.unsqueeze(-1))


def test_quantize_decides_next_to_every_border_as_the_true_quotient_does():
    """float32 values next to each border between two codes, on both sides and on it where it is a number."""
    rows = []
    for a in (1.0, 127.0, 254.0, 1.2345678, 3.1e38, 2.0 ** -90, 1.0 - 2.0 ** -24, 16777213.0):
        top = torch.tensor(a, dtype=torch.float32)
        border = ((torch.arange(-127, 127).double() + 0.5) * top.double() / 127).float()
        near = torch.cat([border, torch.nextafter(border, torch.tensor(math.inf)), torch.nextafter(border, torch.tensor(-math.inf)), top.view(1), -top.view(1)])
        rows.append(torch.nn.functional.pad(near, (0, -near.numel() % 16)))
    x = torch.stack(rows)
    codes, scale = ri.row_int8_quantize(x.cuda())
    want, ws = u.quantize(x)
    assert torch.equal(codes.cpu().long(), want) and torch.equal(scale.cpu(), ws)


def test_quantize_every_finite_bfloat16():
    """All magnitudes beside each of the mantissas that a row's largest value can have."""
    v = torch.arange(0, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for mantissa in range(0, 128, 3):
        top = torch.tensor(0x4300 + mantissa, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
        x = v[v <= top]
        x = torch.nn.functional.pad(x, (0, -x.numel() % 16)).view(1, -1)
        codes, _ = ri.row_int8_quantize(x.cuda())
        assert torch.equal(codes.cpu().long(), u.quantize(x)[0])


@pytest.mark.parametrize("dtype", ALL, ids=ids)
@pytest.mark.parametrize("m,n", [(5, 32), (40, 100)], ids=["few_rows", "tiles"])
def test_rows_with_nan_and_infinity(dtype, m, n):
    x = torch.randn((m, 400), generator=gen(3)).to(dtype)
    x[0, 5], x[1, 200], x[1, 201], x[2, 399] = math.nan, math.inf, math.nan, -math.inf
    codes, scale = ri.row_int8_quantize(x.cuda())
    assert scale.cpu().isnan().tolist() == [True] * 3 + [False] * (m - 3) and not codes[:3].any()
    w, ws = u.weight(gen(4), n, 400)
    ws[7] = math.nan
    y = ri.row_int8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu()
    assert same(y, u.product(x, w, ws))
    assert y[:3].isnan().all() and y[:, 7].isnan().all() and y[3:, 8:].isfinite().all()


# ---------------------------------------------------------------- products

def check_product(dtype, m, n, k, seed=0):
    g = gen(m * 7 + n + seed)
    x = (torch.randn((m, k), generator=g) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=g).float())).to(dtype)
    w, ws = u.weight(g, n, k)
    bias = torch.randn(n, generator=g).to(dtype)
    xd, wd, sd, bd = x.cuda(), w.cuda(), ws.cuda(), bias.cuda()
    y = ri.row_int8_linear(xd, wd, sd)
    assert y.dtype == dtype and y.shape == (m, n)
    assert torch.equal(y.cpu(), u.product(x, w, ws))
    assert torch.equal(ri.row_int8_linear(xd, wd, sd, bd).cpu(), u.product(x, w, ws, bias))
    assert torch.equal(ri.row_int8_product(*ri.row_int8_quantize(xd), wd, sd, bd, dtype).cpu(), u.product(x, w, ws, bias))


@pytest.mark.parametrize("m,n,k", u.SHAPES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_product_equals_its_float32_steps(dtype, m, n, k):
    check_product(dtype, m, n, k)


@pytest.mark.parametrize("m,n,k", u.TILES + u.STREAMED)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_product_in_every_form(dtype, m, n, k):
    check_product(dtype, m, n, k)


def test_every_form_is_run():
    """The sizes above reach each form of tiles, alone and in parts, the streaming kernel with four and eight waves, one and two tiles of rows, alone
    and in parts, and the kernel of few rows with each number of waves."""
    seen = {ggml.lowbit_row_int8_plan(1, 0, *s) + (ggml.lowbit_row_int8_waves(*s),) for s in u.SHAPES + u.TILES + u.STREAMED}
    forms = {(p[0], p[1], p[3]) for p in seen if p[1] > 16}
    assert forms == {(256, 256, 1), (192, 256, 1), (128, 256, 1), (128, 128, 1), (64, 128, 1), (32, 128, 1), (64, 64, 2), (64, 32, 4)}, forms
    assert {p[2] > 1 for p in seen if p[1] > 16} == {False, True}
    assert {(p[0], p[4], p[2] > 1) for p in seen if p[1] == 16} == {(r, w, s) for r in (16, 32) for w in (4, 8) for s in (False, True)}
    assert {p[4] for p in seen if p[1] == 0} == {4, 8}
    back = {ggml.lowbit_row_int8_plan(1, 1, *s)[:2] for s in u.BACK_SHAPES + u.BACK_TILES}
    assert back == {(128, 256), (64, 128), (32, 128), (128, 128), (256, 256), (192, 256)}, back


def test_longest_row():
    """The largest sum that K = 2^17 can make, 127 * 127 * 2^17, still fits 32 bits."""
    k = 1 << 17
    for m in (1, 40):
        x = torch.full((m, k), 2.0)
        w = torch.full((33, k), 127, dtype=torch.int8)
        w[1] = -127
        ws = torch.ones(33)
        y = ri.row_int8_linear(x.cuda(), w.cuda(), ws.cuda()).cpu()
        assert torch.equal(y, u.product(x, w, ws))


# ---------------------------------------------------------------- gradients

def back_tolerance(dtype):
    """Of a row's 2-norm.  Each g * ws is rounded to 11 bits (float32: 22): off by up to half a unit, 2^-11 of itself, evenly spread, which is
    2^-10 / sqrt(12) at rms, over mantissas from 1 to 2 divided by sqrt(2): 2^-12.3 (2^-23.3).  A row's error is a sum of those with random signs,
    2^-12.3 of the row's size in the mean; rows of few terms share them among all their values, so that of 66000 rows some lie at four and a half times
    that: 6 times is beyond all (a normal variable passes it once in 5 * 10^8).  Sums in float32, a rounding of 2^-24 for each of up to 300
    instructions, their squares summed: sqrt(300) * 2^-24 = 1e-6.  The result: half a unit of its type."""
    if dtype == torch.float32:
        return 6 * 2.0 ** -23.3 + 1e-6 + 2.0 ** -24
    return 6 * 2.0 ** -12.3 + 1e-6 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("m,n,k", u.BACK_SHAPES + u.BACK_TILES)
@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_gradient(dtype, m, n, k):
    g = gen(m + n)
    x = torch.randn((m, k), generator=g).to(dtype).cuda().requires_grad_()
    w, ws = u.weight(g, n, k)
    ws = ws * torch.exp2(torch.randint(-6, 7, (n,), generator=g).float())
    grad = (torch.randn((m, n), generator=g) * torch.exp2(torch.randint(-9, 3, (m, 1), generator=g).float())).to(dtype)
    y = ri.row_int8_linear(x, w.cuda(), ws.cuda())
    gx, = torch.autograd.grad(y, x, grad.cuda())
    want = (grad.double() * ws.double()) @ w.double()
    assert gx.dtype == dtype and gx.shape == x.shape
    off = (gx.cpu().double() - want).norm(dim=1)
    assert (off <= back_tolerance(dtype) * want.norm(dim=1)).all(), (off / want.norm(dim=1)).max()


@pytest.mark.parametrize("dtype", ALL, ids=ids)
def test_gradient_rows_of_awkward_numbers(dtype):
    info = torch.finfo(dtype)
    g = gen(5)
    w, ws = u.weight(g, 70, 144)
    grad = torch.randn((8, 70), generator=g).to(dtype)
    grad[0] = 0
    grad[1] = 0
    grad[1, 69] = info.max
    grad[2] *= info.tiny
    grad[3, 5], grad[4, 69], grad[5, 0] = math.nan, math.inf, -math.inf
    x = torch.randn((8, 144), generator=g).to(dtype).cuda().requires_grad_()
    gx, = torch.autograd.grad(ri.row_int8_linear(x, w.cuda(), ws.cuda()), x, grad.cuda())
    gx = gx.cpu()
    assert gx[3:6].isnan().all() and not gx[0].any()
    want = (grad.double() * ws.double()) @ w.double()
    for row in (1, 6, 7):
        assert (gx[row].double() - want[row]).norm() <= back_tolerance(dtype) * want[row].norm()
    # (the second row's products lie among the type's subnormals: a unit of those)
    assert (gx[2].double() - want[2]).abs().max() <= info.tiny * info.eps + back_tolerance(dtype) * want[2].norm()


def test_gradient_against_differences():
    """The product is linear in x once x's codes are exact: differences of one code step against the gradient."""
    g = gen(6)
    w, ws = u.weight(g, 48, 64)
    x = torch.randint(-100, 101, (3, 64), generator=g).float()
    x[:, 0] = 127
    grad = torch.randn((3, 48), generator=g)
    wd, sd = w.cuda(), ws.cuda()
    xd = x.cuda().requires_grad_()
    gx, = torch.autograd.grad(ri.row_int8_linear(xd, wd, sd), xd, grad.cuda())
    for row, col in [(0, 1), (1, 30), (2, 63)]:
        step = torch.zeros_like(x)
        step[row, col] = 1
        up, down = (ri.row_int8_linear((x + s).cuda(), wd, sd).cpu().double() for s in (step, -step))
        d = ((up - down) / 2 * grad.double()).sum()
        # 48 results, each rounded to 2^-24 of itself
        assert abs(gx[row, col].cpu().double() - d) <= 2.0 ** -22 * (up[row].abs() * grad[row].abs()).sum() + 1e-6 * gx[row].norm().cpu()


@pytest.mark.parametrize("m", [1, 16, 40, 300])
def test_every_code_in_the_longest_row(m):
    """128 * 128 * 2^17 = 2^31, which a product of codes of -128 on both sides reaches and 32 bits do not hold; sums beside it, and one row shorter."""
    for k in (1 << 17, (1 << 17) - 16):
        codes, w = torch.full((m, k), -128, dtype=torch.int8), torch.full((33, k), -128, dtype=torch.int8)
        w[1], w[2], w[3, 0], codes[m // 2, 5] = 127, 0, 0, -127
        xs, ws, bias = torch.full((m,), 0.5), torch.arange(1.0, 34.0), torch.ones(33)
        want = torch.full((m, 1), 0.5).double() * ws.double() * u.sums(codes, w)         # (whole numbers below 2^53)
        for dtype in ALL[1:]:
            for b in (None, bias):
                y = ri.row_int8_product(codes.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None if b is None else b.to(dtype).cuda(), dtype).cpu()
                steps = u.sums(codes, w).float() * xs.unsqueeze(-1) * ws
                assert torch.equal(y, (steps if b is None else steps + b).to(dtype))
                assert ((y.double() - want).abs() <= want.abs() * torch.finfo(dtype).eps + 1).all()


# Sizes of each form of tiles in parts (128 x 128: of four waves, then of eight), rows and columns that end inside a tile and K inside a block
PARTS = [(33, 17, 3264, (32, 128, 1)), (2699, 71, 6800, (32, 128, 1)), (66, 1009, 16016, (64, 64, 2)), (34, 4299, 5232, (64, 64, 2)), (65, 2018, 6224, (64, 128, 1)),
         (68, 4126, 3424, (64, 128, 1)), (34, 115, 3888, (64, 32, 4)), (4047, 442, 10192, (128, 128, 1)), (135, 5618, 5088, (128, 128, 1)), (67, 2711, 8416, (128, 128, 1)),
         (195, 8228, 8624, (128, 256, 1)), (135, 5843, 12880, (192, 256, 1)), (267, 5396, 13200, (192, 256, 1)), (391, 4413, 17600, (256, 256, 1)), (417, 8380, 9008, (256, 256, 1))]


@pytest.mark.parametrize("m,n,k,form", PARTS)
def test_every_form_in_parts(form, m, n, k):
    """Whole numbers of sixteenths up to 127 with a largest of 127 in each row: codes that every type holds, so that one sum serves all."""
    rows, cols, parts, groups = ggml.lowbit_row_int8_plan(1, 0, m, n, k)
    assert (rows, cols, groups) == form and parts > 1
    g = gen(m + n)
    codes = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    codes[:, k // 2] = 127
    w, ws = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g) * 0.01
    sums, xs = u.sums(codes, w).float(), torch.full((m, 1), 127 / 16) / torch.tensor(127.0)
    wd, sd, bias = w.cuda(), ws.cuda(), torch.randn(n, generator=g)
    for dtype in ALL:
        b = bias.to(dtype)
        y = ri.row_int8_linear((codes.to(dtype) / 16).cuda(), wd, sd).cpu()
        assert torch.equal(y, (sums * xs * ws).to(dtype))
        y = ri.row_int8_product(codes.cuda(), xs.view(-1).cuda(), wd, sd, b.cuda(), dtype).cpu()
        assert torch.equal(y, (sums * xs * ws + b.float()).to(dtype))


BACK_PARTS = [(66, 4359, 6064, (128, 256)), (5757, 7598, 144, (192, 256)), (161, 4057, 11376, (192, 256)), (390, 5333, 10448, (256, 256)), (5950, 4975, 736, (256, 256))]


@pytest.mark.parametrize("m,n,k,form", BACK_PARTS)
def test_large_forms_of_the_gradient_in_parts(form, m, n, k):
    assert ggml.lowbit_row_int8_plan(1, 1, m, n, k)[:2] == form and ggml.lowbit_row_int8_plan(1, 1, m, n, k)[2] > 1
    g = gen(m + n)
    x = torch.randn((m, k), generator=g).bfloat16().cuda().requires_grad_()
    w, ws = u.weight(g, n, k)
    grad = (torch.randn((m, n), generator=g) * torch.exp2(torch.randint(-9, 3, (m, 1), generator=g).float())).bfloat16()
    gx, = torch.autograd.grad(ri.row_int8_linear(x, w.cuda(), ws.cuda()), x, grad.cuda())
    want = (grad.double() * ws.double()) @ w.double()
    off = (gx.cpu().double() - want).norm(dim=1)
    assert (off <= back_tolerance(torch.bfloat16) * want.norm(dim=1)).all(), (off / want.norm(dim=1)).max()
