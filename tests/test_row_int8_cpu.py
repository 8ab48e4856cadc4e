"""Row-scaled int8 without a GPU: refusals, conversion rules, what moves with a model and what does not."""
import pytest
import torch

import row_int8_util as u
import ipex_llm.ggml.model.llama.llama_cpp as ggml
from ipex_llm.transformers import row_int8 as ri

lib = ggml._lib
P = 4096                                                     # an aligned address that nothing reads
EARG, ESIZE, EDTYPE, ESHAPE = -1, -3, -4, -5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def test_dequantize():
    codes, scale = u.weight(gen(2), 30, 272)
    assert torch.equal(ri.row_int8_dequantize(codes, scale), codes.float() * scale.unsqueeze(-1))
    assert ri.row_int8_dequantize(codes[0], scale[0], torch.bfloat16).dtype == torch.bfloat16
    for bad in ((codes, scale[:2]), (codes.float(), scale), (codes, scale.unsqueeze(-1))):
        with pytest.raises(RuntimeError, match="fit together"):
            ri.row_int8_dequantize(*bad)


def test_the_steps_of_the_quantizer_round_as_the_oracle_does():
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        x = (torch.randn((9, 272), generator=gen(1)) * 5).to(dtype)
        x[0] = 0
        x[1] = (torch.arange(272) % 255 - 127).to(dtype) / 2
        x[2, 3], x[3, 4] = float("nan"), float("-inf")
        codes, scale = ri._quantize_steps(x)
        want, ws = u.quantize(x)
        assert torch.equal(codes.long(), want) and torch.equal(scale.nan_to_num(nan=-1), ws.nan_to_num(nan=-1))


def test_host_tensors_are_refused():
    w, ws = u.weight(gen(3), 16, 32)
    x = torch.zeros((2, 32), dtype=torch.bfloat16)
    for call in (lambda: ri.row_int8_linear(x, w, ws), lambda: ri.row_int8_quantize(x),
                 lambda: ri.row_int8_product(w[:2], ws[:2], w, ws)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ri.row_int8_product(w[:2], ws[:2], w, ws, dtype=torch.float64)


def test_abi_refuses_before_it_touches_the_gpu():
    lin, product, back, q = lib.lowbit_row_int8_linear, lib.lowbit_row_int8_product, lib.lowbit_row_int8_backward, lib.lowbit_row_int8_quantize
    assert lin(P, P, P, None, P, 3, 1, 16, 128, None, 0, None) == EDTYPE
    assert lin(P, P, P, None, P, 0, -1, 16, 128, None, 0, None) == EARG
    assert lin(P, P, P, None, P, 0, 1, 16, 120, None, 0, None) == ESHAPE
    assert lin(P, P, P, None, P, 0, 1 << 22, 16, 128, None, 0, None) == ESIZE
    assert lin(P, P, P, None, P, 0, 1, 1 << 23, 128, None, 0, None) == ESIZE
    assert lin(P, P, P, None, P, 0, 1, 16, (1 << 17) + 16, None, 0, None) == ESIZE
    assert lin(P, P, P, None, P, 0, 1, 16, 0, None, 0, None) == ESHAPE
    assert lin(P + 8, P, P, None, P, 0, 1, 16, 128, None, 0, None) == EARG
    assert lin(P, P, None, None, P, 0, 1, 16, 128, None, 0, None) == EARG
    assert lin(P, P, P + 2, None, P, 0, 1, 16, 128, None, 0, None) == EARG
    need = lib.lowbit_row_int8_linear_workspace_bytes(1, 512, 256, 512)
    assert need >= 512 * 512 + 512 * 4
    assert lin(P, P, P, None, P, 1, 512, 256, 512, None, 0, None) == ESIZE
    assert lin(P, P, P, None, P, 1, 512, 256, 512, P, need - 1, None) == ESIZE
    assert lin(P, P, P, None, P, 1, 512, 256, 512, P + 8, need, None) == ESIZE
    assert lin(None, None, None, None, None, 1, 0, 256, 512, None, 0, None) == 0
    assert lin(None, None, None, None, None, 1, 7, 0, 512, None, 0, None) == 0
    assert product(P, None, P, P, None, P, 1, 4, 16, 128, None, 0, None) == EARG
    assert product(P, P, P, P, None, P, 5, 4, 16, 128, None, 0, None) == EDTYPE
    assert product(P, P, P, P, None, P, 1, 4, 16, 144, None, 0, None) == ESIZE       # (rows that do not fill whole blocks are copied)
    assert back(P, P, P, P, 1, 4, 16, 128, None, 0, None) == ESIZE
    assert back(P, P, P, P, 1, 4, 0, 128, None, 0, None) == ESHAPE
    assert back(P, P, P, P, 7, 4, 16, 128, None, 0, None) == EDTYPE
    assert back(None, None, None, None, 1, 0, 16, 128, None, 0, None) == 0
    assert q(P, 0, -1, 128, P, P, None) == EARG and q(P, 0, 1, 120, P, P, None) == ESHAPE and q(P, 9, 1, 128, P, P, None) == EDTYPE
    assert q(P, 0, 1, 1 << 23, P, P, None) == ESIZE and q(P, 0, 1, -16, P, P, None) == EARG and q(P, 0, 1, 128, None, P, None) == EARG
    assert q(None, 0, 0, 128, None, None, None) == 0 and q(None, 0, 5, 0, None, None, None) == 0
    with pytest.raises(Exception, match="plan"):
        ggml.lowbit_row_int8_plan(0, 0, 0, 16, 16)
    with pytest.raises(Exception, match="waves"):
        ggml.lowbit_row_int8_waves(1, 16, 24)


def test_plans_cover_every_size():
    """Whatever is asked for has a plan whose parts have blocks, and a workspace that holds them."""
    for m in (1, 4, 5, 16, 17, 64, 300, 4000):
        for n in (1, 64, 1000, 28672):
            for k in (16, 128, 144, 4096, 1 << 17):
                rows, cols, splits, groups = ggml.lowbit_row_int8_plan(1, 0, m, n, k)
                assert (rows == 0 or cols == 16) == (ggml.lowbit_row_int8_waves(m, n, k) > 0)      # (few rows, or streamed)
                assert 1 <= splits <= (k + 127) // 128 and groups in (1, 2, 4)
                if rows:
                    need = m * ((k + 127) // 128 * 128) + m * 4 + (splits * m * n * 4 if splits > 1 else 0)
                    assert ggml.lowbit_row_int8_linear_workspace_bytes(1, m, n, k) >= need
                for dtype, terms in ((0, 1), (2, 2)):
                    splits = ggml.lowbit_row_int8_plan(dtype, 1, m, n, k)[2]
                    assert 1 <= splits <= (n + 63) // 64 * terms
                    assert ggml.lowbit_row_int8_backward_workspace_bytes(dtype, m, n, k) >= m * n * 2 * terms + (splits * m * k * 4 if splits > 1 else 0)


@pytest.mark.parametrize("m", [2, 300, 2048, 20000])
def test_gradient_tiles_of_very_long_rows_stay_within_32_bit_offsets(m):
    for n in (5000, (1 << 21) - 64, (1 << 21) + 64, (1 << 22) + 1, (1 << 23) - 1):
        for dtype, size in ((0, 2), (1, 2), (2, 4)):
            for k in (16, 1024, 4096):
                rows = ggml.lowbit_row_int8_plan(dtype, 1, m, n, k)[0]
                assert rows * ((n + 63) // 64 * 64) * size <= 1 << 31


def test_experts_router_and_layer_refuse_before_they_touch_the_gpu():
    ex, route, back, layer = lib.lowbit_row_int8_experts, lib.lowbit_route, lib.lowbit_route_backward, lib.lowbit_row_int8_moe

    def experts(x=P, ids=P, weight=P, wdt=2, tokens=2, top_k=2, n_exp=4, gu=P, gus=P, d=P, ds=P, ws=P, bytes_=1 << 40, y=P, dt=1, hidden=128, inter=64, act=0):
        return ex(x, ids, weight, wdt, tokens, top_k, n_exp, gu, gus, d, ds, ws, bytes_, y, dt, hidden, inter, act, None)
    assert experts(dt=3) == EDTYPE and experts(wdt=9) == EDTYPE and experts(act=2) == EARG
    assert experts(top_k=0) == ESIZE and experts(top_k=65) == ESIZE and experts(n_exp=4097) == ESIZE and experts(tokens=1 << 20, top_k=4) == ESIZE
    assert experts(hidden=(1 << 17) + 16) == ESIZE and experts(inter=(1 << 17) + 16) == ESIZE and experts(tokens=-1) == ESIZE
    assert experts(hidden=120) == ESHAPE and experts(inter=72) == ESHAPE
    assert experts(x=P + 8) == EARG and experts(gus=P + 4) == EARG and experts(ids=P + 4) == EARG and experts(y=None) == EARG
    assert experts(ws=None) == ESIZE and experts(bytes_=16) == ESIZE
    assert experts(tokens=0, x=None, ids=None, y=None, ws=None) == 0
    need = lib.lowbit_row_int8_experts_workspace_bytes
    assert need(300, 2, 8, 512, 256) >= 600 * (5 * 256 + 4 * 512) + 300 * 512 and need(300, 2, 8, 512, 250) == 0 and need(0, 2, 8, 512, 256) == 0
    assert need(1 << 20, 2, 8, 8192, 8192) <= (1 << 31) + (1 << 30)             # (tokens go in parts)

    def router(x=P, xdt=1, r=P, rdt=1, bias=None, tokens=2, n_exp=8, hidden=64, top_k=2, score=0, w=P, ids=P, z=None, ws=P, bytes_=1 << 40):
        return route(x, xdt, r, rdt, bias, tokens, n_exp, hidden, top_k, score, 1, 1.0, w, ids, z, ws, bytes_, None)
    assert router(xdt=3) == EDTYPE and router(rdt=-1) == EDTYPE and router(score=2) == EARG and router(tokens=-1) == EARG and router(hidden=0) == EARG
    assert router(hidden=60) == ESHAPE and router(n_exp=1025) == ESIZE and router(top_k=9) == ESIZE and router(top_k=0) == ESIZE
    assert router(n_exp=100, top_k=65) == ESIZE and router(tokens=(1 << 21) + 1) == ESIZE
    assert router(x=P + 4) == EARG and router(bias=P + 2) == EARG and router(z=P + 4) == EARG and router(w=None) == EARG
    assert router(n_exp=64, hidden=8192, bytes_=8) == ESIZE and router(n_exp=64, hidden=8192, ws=None) == ESIZE
    assert lib.lowbit_route_workspace_bytes(2, 8, 64) == 0 < lib.lowbit_route_workspace_bytes(2, 64, 8192)       # (small routers need none)
    assert router(tokens=0, x=None, r=None) == 0
    assert back(P, P, P, P, 1, P, 1, 0, 8, 64, 2, 0, 1, 1.0, P, P, P, 1 << 40, None) == EARG
    assert back(P, None, P, P, 1, P, 1, 2, 8, 64, 2, 0, 1, 1.0, P, P, P, 1 << 40, None) == EARG
    assert back(P, P, P, P, 1, P, 1, 2, 8, 64, 2, 0, 1, 1.0, P, P, P, 8, None) == ESIZE

    def whole(x=P, r=P, rdt=1, bias=None, tokens=2, top_k=2, n_exp=8, score=0, gu=P, gus=P, d=P, ds=P, ws=P, bytes_=1 << 40, y=P, dt=1, hidden=128, inter=64, act=0):
        return layer(x, r, rdt, bias, tokens, top_k, n_exp, score, 1, 1.0, gu, gus, d, ds, ws, bytes_, y, dt, hidden, inter, act, None)
    assert whole(dt=7) == EDTYPE and whole(score=5) == EARG and whole(act=3) == EARG and whole(hidden=72) == ESHAPE and whole(top_k=9) == ESIZE
    assert whole(r=None) == EARG and whole(gu=None) == EARG and whole(bytes_=100) == ESIZE and whole(n_exp=1030) == ESIZE
    assert whole(tokens=0, x=None, y=None) == 0
    assert lib.lowbit_row_int8_moe_workspace_bytes(2, 2, 8, 128, 64) >= need(2, 2, 8, 128, 64)


def test_router_and_layers_refuse_host_tensors():
    from ipex_llm.transformers import moe
    x, router = torch.zeros((2, 32)), torch.zeros((4, 32))
    w, ws = u.weight(gen(3), 32, 32, (4,))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        moe.moe_route(x, router, 2)
    with pytest.raises(RuntimeError, match="score is"):
        moe.moe_route(x, router, 2, score="relu")
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ri.row_int8_experts(x, torch.zeros((2, 1), dtype=torch.int64), torch.ones((2, 1)), w, ws, w[:, :, :16].contiguous(), ws)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ri.row_int8_moe(x, router, 2, w, ws, w[:, :, :16].contiguous(), ws)


def test_route_steps_are_the_formula():
    from ipex_llm.transformers import moe
    x, router, bias = torch.randn((5, 16), generator=gen(1)), torch.randn((6, 16), generator=gen(2)), torch.randn(6, generator=gen(3))
    z = x.double() @ router.double().t()
    w, index = moe._route_steps(x, router, 2, None, "softmax", True, 2.0)
    top = z.topk(2, dim=-1)
    assert torch.equal(index, top.indices) and torch.allclose(w.double(), 2 * torch.softmax(top.values, -1), atol=1e-7)
    w, index = moe._route_steps(x, router, 3, bias, "sigmoid", False, 1.0)
    assert torch.equal(index, (torch.sigmoid(z) + bias.double()).topk(3, dim=-1).indices)
    assert torch.allclose(w.double(), torch.sigmoid(z).gather(1, index), atol=1e-7)


def test_the_longest_row_of_given_codes_goes_in_parts():
    """Of given codes 128 * 128 * 2^17 does not fit 32 bits, so that their product has two parts at least, for which the workspace has room."""
    for m, n in ((1, 17), (16, 300), (40, 33), (300, 3000), (2000, 2100)):
        k = 1 << 17
        assert ggml.lowbit_row_int8_product_workspace_bytes(0, m, n, k) >= 2 * m * ((n + 3) // 4 * 4) * 4
