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


def experts64(x, picks, p, gu, gus, dn, dns, act, border):
    """(result, the most it may move where h * 448 / a lies within `border`, relative, of a border of two codes, the size of its pairs)."""
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
        off = (u.e4m3(h / step * (1 + border)) - u.e4m3(h / step * (1 - border))).abs() * step
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
    # h: u of -15 at most, whose four roundings and the exponent's count 2 |u| each, half a unit of 2^-23 each, and some units more
    want, slack, size = experts64(*case, 1, 2.0 ** -24 * (5 * 2 * 15 + 8))
    assert (want.abs().amax(dim=1) > 0.01).all() and slack.norm() < 0.1 * want.norm()
    unit = torch.finfo(dtype).eps / 2
    # (a result is rounded once; the second product drops bits as in any product)
    assert (got - want).norm() <= unit * want.norm() + slack.norm() + (3 ** 0.5 * 2.0 ** -13 + 2.0 ** -18) * size.norm()
