"""Block-scaled fp8 without a GPU: refusals, conversion rules, what moves with a model and what does not."""
import pytest
import torch
from torch import nn

import block_fp8_util as u
import ipex_llm.ggml.model.llama.llama_cpp as ggml
from ipex_llm.transformers import block_fp8 as bf
from ipex_llm.transformers.convert import ggml_convert_low_bit, is_block_fp8

FP8 = 15
lib = ggml._lib


def scaled_linear(n, k, bias=False, seed=1):
    w, ws = u.random_weight(torch.Generator().manual_seed(seed), n, k)
    lin = nn.Linear(k, n, bias=bias)
    lin.weight = nn.Parameter(w, requires_grad=False)
    lin.weight_scale_inv = nn.Parameter(ws, requires_grad=False)
    return lin


def test_the_oracle_rounds_as_torch_does():
    q = torch.linspace(-448, 448, 100003, dtype=torch.float64).float()
    q = torch.cat([q, q * 2.0 ** -8, q * 2.0 ** -14, torch.tensor([17.0, 18.0, 19.0, 21.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    assert torch.equal(u.e4m3(q.double()), q.to(u.E4M3).double())


def test_dequantize():
    codes, scale = u.weight(torch.Generator().manual_seed(2), 300, 272)
    assert torch.equal(bf.block_fp8_dequantize(codes, scale).double(), u.dense(codes, scale))
    rows = torch.exp2(torch.arange(300 * 3) % 5).view(300, 3).float()
    assert torch.equal(bf.block_fp8_dequantize(codes, rows, torch.bfloat16), (codes.double() * u.spread(rows, 300, 272, 1)).bfloat16())
    with pytest.raises(RuntimeError, match="fit together"):
        bf.block_fp8_dequantize(codes, scale[:2])
    with pytest.raises(RuntimeError, match="fit together"):
        bf.block_fp8_dequantize(codes.float(), scale)


def test_host_tensors_are_refused():
    w, ws = u.weight(torch.Generator().manual_seed(3), 16, 32)
    x = torch.zeros((2, 32), dtype=torch.bfloat16)
    for call in (lambda: bf.block_fp8_linear(x, w, ws), lambda: bf.block_fp8_quantize(x), lambda: bf.block_fp8_quantize_weight(x),
                 lambda: bf.block_fp8_experts(x, torch.zeros((2, 1), dtype=torch.int64), torch.ones((2, 1)), w[None], ws[None], w[None], ws[None])):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(RuntimeError, match="act is 0"):
        bf.block_fp8_experts(x, x, x, w, ws, w, ws, act=2)


P = 4096                                                     # an aligned address that nothing reads


def test_abi_refuses_before_it_touches_the_gpu():
    lin, back, q, qw, ex = (lib.lowbit_block_fp8_linear, lib.lowbit_block_fp8_backward, lib.lowbit_block_fp8_quantize,
                            lib.lowbit_block_fp8_quantize_weight, lib.lowbit_block_fp8_experts)
    assert lin(P, P, P, None, P, 3, 1, 16, 128, None, 0, None) == -4
    assert lin(P, P, P, None, P, 0, -1, 16, 128, None, 0, None) == -1
    assert lin(P, P, P, None, P, 0, 1, 16, 120, None, 0, None) == -5
    assert lin(P, P, P, None, P, 0, 1 << 22, 16, 128, None, 0, None) == -3
    assert lin(P, P, P, None, P, 0, 1, 16, 1 << 23, None, 0, None) == -3
    assert lin(P, P, P, None, P, 0, 1, 16, 0, None, 0, None) == -5
    assert lin(None, P, P, None, P, 0, 1, 16, 128, None, 0, None) == -1
    assert lin(P + 8, P, P, None, P, 0, 1, 16, 128, None, 0, None) == -1
    assert lin(P, P, P, None, P, 0, 100, 16, 128, None, 0, None) == -3          # without the workspace it asks for
    assert b"workspace" in lib.lowbit_last_error()
    assert lin(P, P, P, None, P, 0, 0, 16, 128, None, 0, None) == 0 == lin(P, P, P, None, P, 0, 5, 0, 128, None, 0, None)
    assert back(P, P, P, P, 2, 1, 16, 128, None, 0, None) == -4                 # float32
    assert back(P, P, P, P, 0, 1, 16, 100, None, 0, None) == -5
    assert back(P, P, P, P, 0, 1, 0, 128, None, 0, None) == -5
    assert back(P, P + 4, P, P, 0, 1, 16, 128, None, 0, None) == -1
    assert back(P, P, P, P, 0, 0, 16, 128, None, 0, None) == 0
    assert q(P, 3, 1, 128, P, P, None) == -4 and q(P, 0, 1, 8, P, P, None) == -5 and q(P, 0, -1, 16, P, P, None) == -1
    assert q(P + 2, 0, 1, 16, P, P, None) == -1 and q(P, 0, 0, 16, P, P, None) == 0
    assert qw(P, 3, 1, 16, 128, P, P, None) == -4 and qw(P, 0, 1, 16, 24, P, P, None) == -5 and qw(P, 0, -1, 16, 16, P, P, None) == -1
    assert qw(P, 0, 1, 1 << 23, 16, P, P, None) == -3 and qw(P, 0, 0, 16, 16, P, P, None) == 0

    def experts(x=P, wdt=0, tokens=4, top_k=2, n=4, dt=0, hidden=128, inter=128, act=0, ws=None, size=0):
        return ex(x, P, P, wdt, tokens, top_k, n, P, P, P, P, ws, size, P, dt, hidden, inter, act, None)
    assert experts(dt=2) == -4 and experts(wdt=3) == -4 and experts(act=2) == -1 and experts(tokens=0) == 0
    assert experts(top_k=65) == -3 and experts(n=4097) == -3 and experts(tokens=1 << 21) == -3 and experts(tokens=-1) == -3
    assert experts(hidden=24) == -5 and experts(inter=64) == -5 and experts(x=None) == -1
    assert experts() == -3 and b"workspace" in lib.lowbit_last_error()
    assert lib.lowbit_block_fp8_experts_workspace_bytes(4, 2, 4, 128, 64) == 0
    assert lib.lowbit_block_fp8_linear_workspace_bytes(0, 100, 16, 100) == 0 < lib.lowbit_block_fp8_linear_workspace_bytes(0, 100, 16, 112)


def test_conversion_replaces_block_scaled_layers_and_keeps_their_codes():
    lin = scaled_linear(200, 272, bias=True)
    assert is_block_fp8(lin) and not is_block_fp8(nn.Linear(16, 16))
    codes, scales = lin.weight.data.clone(), lin.weight_scale_inv.data.clone()
    model = ggml_convert_low_bit(nn.Sequential(lin, nn.ReLU()).eval(), FP8, torch_dtype=torch.bfloat16)
    new = model[0]
    assert type(new) is bf.BlockFP8Linear and not new.training and not any(p.requires_grad for p in new.parameters())
    assert torch.equal(new.weight.float(), codes.float()) and torch.equal(new.weight_scale_inv, scales)
    assert set(new.state_dict()) == {"weight", "weight_scale_inv", "bias"}
    with pytest.raises(RuntimeError, match="fp8_e4m3"):
        ggml_convert_low_bit(nn.Sequential(scaled_linear(32, 128)), 2)
    bad = scaled_linear(200, 272)
    bad.weight_scale_inv = nn.Parameter(torch.ones(1, 3), requires_grad=False)
    with pytest.raises(RuntimeError, match="one scale for each block"):
        ggml_convert_low_bit(nn.Sequential(bad), FP8)
    again = ggml_convert_low_bit(model, FP8)
    assert again[0] is new                                   # converted layers stay as they are


def test_block_fp8_asks_for_fp8():
    from ipex_llm import optimize_model
    with pytest.raises(RuntimeError, match="use it with fp8_e4m3"):
        optimize_model(nn.Sequential(nn.Linear(64, 64)), "sym_int4", block_fp8=True)


def test_shape_only_conversion_of_dense_layers():
    with torch.device("meta"):
        model = nn.Sequential(nn.Linear(272, 200), nn.Linear(200, 100), nn.Linear(192, 64))
    model = ggml_convert_low_bit(model, FP8, convert_shape_only=True, block_fp8=True)
    assert type(model[0]) is bf.BlockFP8Linear and model[0].weight.shape == (200, 272) and model[0].weight_scale_inv.shape == (2, 3)
    assert type(model[1]) is nn.Linear                       # 200 is no multiple of 16
    with torch.device("meta"):
        model = nn.Sequential(nn.Linear(256, 64), nn.Linear(256, 64))
    model = ggml_convert_low_bit(model, FP8, convert_shape_only=True, block_fp8={"1"})
    assert type(model[1]) is bf.BlockFP8Linear and type(model[0]).__name__ == "LowBitLinear"


def test_codes_and_scales_keep_their_format_when_a_model_moves():
    new = bf.BlockFP8Linear.from_linear(scaled_linear(130, 144, bias=True))
    codes, scales = new.weight.data.clone(), new.weight_scale_inv.data.clone()
    for move in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu"), lambda m: m.float()):
        m = move(new)
        assert m.weight.dtype == u.E4M3 and m.weight_scale_inv.dtype == torch.float32
        assert torch.equal(m.weight.float(), codes.float()) and torch.equal(m.weight_scale_inv, scales)
    assert new.half().bias.dtype == torch.float16
    assert new.to("meta").weight.device.type == "meta" and new.weight.dtype == u.E4M3


def test_experts_module_from_dense_shapes_and_from_scaled_weights():
    class Fused(nn.Module):
        def __init__(self, e, h, i, dtype=torch.float32):
            super().__init__()
            self.gate_up_proj = nn.Parameter(torch.zeros((e, 2 * i, h)).to(dtype), requires_grad=False)
            self.down_proj = nn.Parameter(torch.zeros((e, h, i)).to(dtype), requires_grad=False)
            self.act_fn = nn.SiLU()

    with torch.device("meta"):
        model = nn.Sequential(Fused(3, 256, 128), Fused(3, 256, 64))
    model = ggml_convert_low_bit(model, FP8, convert_shape_only=True, block_fp8=True)
    assert type(model[0]) is bf.BlockFP8Experts and model[0].down_proj_scale_inv.shape == (3, 2, 1)
    assert type(model[1]) is Fused                           # experts of 64 columns do not divide into blocks
    fused = Fused(3, 256, 128, u.E4M3)
    fused.gate_up_proj_scale_inv = nn.Parameter(torch.ones(3, 2, 2), requires_grad=False)
    fused.down_proj_scale_inv = nn.Parameter(torch.ones(3, 2, 1), requires_grad=False)
    model = ggml_convert_low_bit(nn.Sequential(fused).eval(), FP8)
    assert type(model[0]) is bf.BlockFP8Experts and not model[0].training
    with pytest.raises(RuntimeError, match="multiple of 16"):
        bf.BlockFP8Experts(2, 24, 128, nn.SiLU())


def test_block_scaled_projections_are_not_merged():
    from ipex_llm.transformers.models.common import merge_linear
    assert merge_linear([scaled_linear(128, 128), scaled_linear(128, 128)]) is None
    assert merge_linear([nn.Linear(32, 16), nn.Linear(32, 16)]) is not None


def test_saved_layers_are_found_again(tmp_path):
    from ipex_llm.optimize import block_fp8_layers, unconverted_linears
    model = nn.ModuleDict({"q_proj": bf.BlockFP8Linear.from_linear(scaled_linear(128, 128)), "head": nn.Linear(16, 16)})
    state = model.state_dict()
    assert block_fp8_layers(state) == ({"q_proj"}, True) and unconverted_linears(state) == ["head"]
    torch.save(state, tmp_path / "m.bin")
    again = torch.load(tmp_path / "m.bin", weights_only=True)
    assert again["q_proj.weight"].dtype == u.E4M3


def test_sizes_of_the_gpu_tests_reach_every_kernel():
    f32, bf16 = ggml.DT_F32, ggml.DT_BF16

    def kinds(plans):
        return {(rows, cols, groups, splits > 1) for rows, cols, splits, groups in plans}

    def both(*forms):
        return {(*form, split) for form in forms for split in (False, True)}

    every, few = both((32, 128, 1), (64, 128, 1), (128, 256, 1)), {(0, 0, 1, False)}
    shared = both((64, 64, 2), (64, 128, 2))
    assert kinds(ggml.lowbit_block_fp8_plan(f32, 0, *s) for s in u.SHAPES + u.TILES) == every | few | shared
    assert kinds(ggml.lowbit_block_fp8_plan(bf16, 0, *s) for s in u.SHAPES + u.TILES) == every | few | shared | both((128, 128, 1), (192, 256, 1), (256, 256, 1))
    assert kinds(ggml.lowbit_block_fp8_plan(bf16, 1, *s) for s in u.BACK_SHAPES + u.BACK_TILES) == every
    plans = {ggml.lowbit_block_fp8_experts_plan(*s) for s in u.EXPERTS + u.EXPERT_TILES}
    assert {p[0] for p in plans} == {0, 64, 96, 128} and {p[3] for p in plans} == {0, 1}
    assert {p[1:3] for p in plans} == {(0, 0), (32, 128), (64, 128), (128, 128), (128, 256), (192, 256), (256, 256)}


def test_plans_hold_for_any_size():
    """Whatever the size: a tile that is there, no empty part of the sum, and no more workspace than codes, scales and 256 MB of sums."""
    for m in (1, 4, 5, 31, 128, 1000, 8192, (1 << 22) - 1):
        for n in (1, 7, 128, 4097, 28672, (1 << 23) - 1):
            for k in (16, 128, 144, 4096, 16384, (1 << 23) - 16):
                for dtype in (ggml.DT_F16, ggml.DT_F32):
                    rows, cols, splits, _ = ggml.lowbit_block_fp8_plan(dtype, 0, m, n, k)
                    assert (rows == 0) == (cols == 0) and 1 <= splits <= 8 and splits <= u.blocks(k)
                    parts = -(-u.blocks(k) // splits)
                    assert parts * (splits - 1) < u.blocks(k)
                    bound = m * u.blocks(k) * (128 * (2 if dtype == ggml.DT_F32 else 1) + 4) + (256 << 20) + 1024
                    assert ggml.lowbit_block_fp8_linear_workspace_bytes(dtype, m, n, k) <= bound
                rows, cols, splits, _ = ggml.lowbit_block_fp8_plan(ggml.DT_BF16, 1, m, n, k)
                assert rows and cols and -(-u.blocks(n) // splits) * (splits - 1) < u.blocks(n)
                assert ggml.lowbit_block_fp8_backward_workspace_bytes(ggml.DT_BF16, m, n, k) <= m * (n + 64) * 2 + (256 << 20) + 1024
    for call in (lambda: ggml.lowbit_block_fp8_plan(ggml.DT_F32, 1, 1, 16, 16), lambda: ggml.lowbit_block_fp8_plan(ggml.DT_F16, 0, 0, 16, 16),
                 lambda: ggml.lowbit_block_fp8_plan(ggml.DT_F16, 0, 1, 16, 24), lambda: ggml.lowbit_block_fp8_experts_plan(0, 1, 1, 16, 128),
                 lambda: ggml.lowbit_block_fp8_experts_plan(1, 65, 1, 16, 128)):
        with pytest.raises(Exception):
            call()


class FusedExperts(nn.Module):
    """Experts in one module, block-scaled or dense; `limit` and `alpha` change the gate, as some models' do."""

    def __init__(self, e, h, i, limit=None, alpha=None, blocks=True):
        super().__init__()
        gen = torch.Generator().manual_seed(5)
        self.act_fn, self.limit, self.alpha = nn.SiLU(), limit, alpha
        for name, n, k in (("gate_up_proj", 2 * i, h), ("down_proj", h, i)):
            w, ws = u.random_weight(gen, n, k, lead=(e,))
            setattr(self, name, nn.Parameter(w if blocks else torch.randn((e, n, k), generator=gen) * 0.05, requires_grad=False))
            if blocks:
                setattr(self, name + "_scale_inv", nn.Parameter(ws, requires_grad=False))

    def _apply_gate(self, gu):
        g, v = gu.chunk(2, dim=-1)
        if self.limit is not None:
            g, v = g.clamp(max=self.limit), v.clamp(-self.limit, self.limit)
        return self.act_fn(g) * v if self.alpha is None else (v + 1) * g * torch.sigmoid(g * self.alpha)


GATES = [dict(limit=7.0), dict(limit=7.0, alpha=1.7), dict(limit=500.0), dict(alpha=1.7)]


@pytest.mark.parametrize("own", GATES, ids=str)
def test_experts_keep_a_gate_of_their_own(own, monkeypatch):
    module = FusedExperts(3, 256, 128, **own).eval()
    new = ggml_convert_low_bit(nn.Sequential(module).eval(), FP8)[0]
    assert type(new) is bf.BlockFP8Experts
    gu = torch.randn((9, 256), generator=torch.Generator().manual_seed(2)) * 30
    assert torch.equal(new.own_gate(gu), module._apply_gate(gu))
    held = [v for v in vars(new.own_gate.__self__).values() if isinstance(v, torch.Tensor)]
    assert not held and not list(new.own_gate.__self__.parameters())      # a gate without the module's weights
    # (the products by the formula: there is no GPU here)
    monkeypatch.setattr(bf, "_exact_product", lambda x, w, s, dtype: (x.double() @ u.dense(w, s).t()).float())
    x, picks = torch.randn((6, 256), generator=torch.Generator().manual_seed(3)) * 8, torch.tensor([[0, 2]] * 5 + [[1, 7]])
    p, want = torch.full((6, 2), 0.5), torch.zeros((6, 256))
    for e in range(3):
        t, j = torch.where(picks == e)
        gu = (x[t].double() @ u.dense(module.gate_up_proj[e], module.gate_up_proj_scale_inv[e]).t()).float()
        want.index_add_(0, t, (module._apply_gate(gu).double() @ u.dense(module.down_proj[e], module.down_proj_scale_inv[e]).t()).float() * 0.5)
    assert torch.allclose(new(x, picks, p), want, rtol=1e-4, atol=1e-4)


def test_experts_with_the_plain_gate_or_none_run_in_the_native_call():
    class NoGate(FusedExperts):
        _apply_gate = None
    for module in (FusedExperts(2, 256, 128), NoGate(2, 256, 128, limit=7.0)):
        assert ggml_convert_low_bit(nn.Sequential(module), FP8)[0].own_gate is None


class _GateOfTensors(FusedExperts):
    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.bound = nn.Parameter(torch.ones(1), requires_grad=False)

    def _apply_gate(self, gu):
        g, v = gu.chunk(2, dim=-1)
        return self.act_fn(g) * v.clamp(max=self.bound)


def test_a_gate_that_needs_the_modules_tensors():
    with pytest.raises(RuntimeError, match="gate depends on tensors"):
        bf.BlockFP8Experts.from_fused(_GateOfTensors(2, 256, 128))
    with pytest.raises(RuntimeError, match="holds .'bound'"):
        ggml_convert_low_bit(nn.Sequential(_GateOfTensors(2, 256, 128)), FP8)
    model = ggml_convert_low_bit(nn.Sequential(_GateOfTensors(2, 256, 128, blocks=False)), 2)
    assert type(model[0]) is _GateOfTensors                  # dense experts stay as they are


@pytest.mark.parametrize("own", GATES[:2], ids=str)
def test_low_bit_experts_keep_a_gate_of_their_own(own):
    from ipex_llm.transformers.moe import LowBitExperts
    module = FusedExperts(3, 256, 128, blocks=False, **own).eval()
    with torch.device("meta"):
        shapes = FusedExperts(3, 256, 128, blocks=False, **own).eval()
    new = LowBitExperts.from_fused(shapes.to("meta"), 2, convert_shape_only=True)
    for layers, w in ((new.gate, module.gate_up_proj[:, :128]), (new.up, module.gate_up_proj[:, 128:]), (new.down, module.down_proj)):
        for e in range(3):                                   # (dense layers in their place: there is no GPU here)
            layers[e] = nn.Linear(*reversed(w[e].shape), bias=False)
            layers[e].weight.data = w[e].clone()
    x, picks = torch.randn((6, 256), generator=torch.Generator().manual_seed(3)) * 30, torch.tensor([[0, 2]] * 5 + [[1, 2]])
    p, want = torch.full((6, 2), 0.5), torch.zeros((6, 256))
    for e in range(3):
        t, j = torch.where(picks == e)
        want.index_add_(0, t, module._apply_gate(x[t] @ module.gate_up_proj[e].t()) @ module.down_proj[e].t() * 0.5)
    with torch.no_grad():
        got = new(x, picks, p)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)
    assert LowBitExperts.from_fused(FusedExperts(3, 256, 128, blocks=False).to("meta"), 2, convert_shape_only=True).own_gate is None


def held(module, **more):
    for name, v in more.items():
        setattr(module, name, nn.Parameter(v, requires_grad=False) if isinstance(v, torch.Tensor) else v)
    return module


OTHER_FORMS = [
    ("dynamic", lambda: held(scaled_linear(256, 256), activation_scheme="static")),
    ("activation_scale", lambda: held(scaled_linear(256, 256), activation_scale=torch.ones(1))),
    ("2 groups", lambda: held(scaled_linear(256, 128), n_groups=2)),
    ("128 x 128, not", lambda: held(scaled_linear(64, 64), block_size=(64, 64))),
    ("rotation", lambda: held(scaled_linear(256, 256), rotation=torch.ones(256))),
    ("dynamic", lambda: held(FusedExperts(2, 256, 128), activation_scheme="static")),
    ("down_proj_activation_scale", lambda: held(FusedExperts(2, 256, 128), down_proj_activation_scale=torch.ones(2))),
    ("gate_up_proj_bias", lambda: held(FusedExperts(2, 256, 128), gate_up_proj_bias=torch.ones(2, 256))),
    ("weight_scale'", lambda: held(nn.Linear(256, 256), weight=torch.zeros(256, 256).to(u.E4M3), weight_scale=torch.ones(1))),
]


@pytest.mark.parametrize("message,make", OTHER_FORMS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(OTHER_FORMS)])
def test_other_forms_of_fp8_checkpoints_are_refused(message, make):
    with pytest.raises(RuntimeError, match=message):
        ggml_convert_low_bit(nn.ModuleDict({"layer": make()}), FP8)
    model = ggml_convert_low_bit(nn.ModuleDict({"layer": make(), "other": scaled_linear(128, 128)}), FP8, modules_to_not_convert=["layer"])
    assert type(model["layer"]) in (nn.Linear, FusedExperts) and type(model["other"]) is bf.BlockFP8Linear


def test_block_scaled_layers_with_a_named_form_convert():
    lin = held(scaled_linear(200, 272), activation_scheme="dynamic", block_size=[128, 128], n_groups=1)
    powers = torch.exp2(torch.randint(-9, -5, (2, 3)).float())
    lin.weight_scale_inv = nn.Parameter(powers.to(torch.float8_e8m0fnu), requires_grad=False)     # scales held as their exponents
    new = ggml_convert_low_bit(nn.Sequential(lin), FP8)[0]
    assert type(new) is bf.BlockFP8Linear and torch.equal(new.weight_scale_inv, powers)
    dense = nn.Linear(256, 256)
    dense.register_buffer("weight_scale_factor", torch.ones(1))           # not fp8: nothing of a checkpoint's
    from ipex_llm.transformers.convert import check_block_fp8
    check_block_fp8(dense, "dense", [])


def test_dense_layers_that_compute_more_than_a_product_stay_dense():
    with torch.device("meta"):
        grouped, biased = held(nn.Linear(256, 128), n_groups=2), held(FusedExperts(2, 256, 128, blocks=False), gate_up_proj_bias=torch.ones(2, 256))
        for qtype, block_fp8 in ((FP8, True), (FP8, False), (2, False)):
            model = nn.ModuleDict({"grouped": grouped, "experts": biased, "other": nn.Linear(256, 128)})
            model = ggml_convert_low_bit(model, qtype, convert_shape_only=True, block_fp8=block_fp8)
            assert model["grouped"] is grouped and model["experts"] is biased and type(model["other"]) is not nn.Linear


def tiny_llama():
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(4)
    return LlamaForCausalLM(LlamaConfig(hidden_size=256, intermediate_size=384, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                                        vocab_size=64)).eval()


@pytest.mark.parametrize("apart", [False, True], ids=["merged", "disable_optimize_pre"])
def test_a_model_with_some_block_scaled_layers_saves_and_loads(apart, tmp_path):
    """Layer 1's projections block-scaled, the others' q, k and v dense: merged where they may be, layer by layer."""
    from ipex_llm import optimize_model
    from ipex_llm.optimize import load_low_bit, unmerged_attentions
    model = tiny_llama()
    for part in (model.model.layers[1].self_attn, model.model.layers[1].mlp):
        for name, lin in list(part.named_children()):
            if isinstance(lin, nn.Linear):
                setattr(part, name, scaled_linear(*lin.weight.shape))
    model = optimize_model(model, "fp8_e4m3", modules_to_not_convert=["layers.0", "layers.2", "lm_head"], disable_optimize_pre=apart)
    assert hasattr(model.model.layers[0].self_attn, "qkv_proj") != apart and not hasattr(model.model.layers[1].self_attn, "qkv_proj")
    model.save_low_bit(str(tmp_path))
    again = load_low_bit(tiny_llama(), str(tmp_path))
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got) and all(torch.equal(got[k].float(), v.float()) and got[k].dtype == v.dtype for k, v in want.items())
    assert type(again.model.layers[1].self_attn.q_proj) is bf.BlockFP8Linear and type(again.model.layers[2].mlp.up_proj) is nn.Linear
    every = {f"model.layers.{i}.self_attn" for i in range(3)}
    assert unmerged_attentions(want) == (every if apart else {"model.layers.1.self_attn"})
    assert unmerged_attentions({"q_proj.weight": 0, "a.xq_proj.weight": 0, "b.q_proj.bias": 0}) == {"", "b"}


def test_layers_left_out_of_the_conversion_keep_their_codes():
    model = nn.ModuleDict({"left": scaled_linear(128, 256, bias=True), "other": scaled_linear(128, 256), "norm": nn.LayerNorm(256), "experts": FusedExperts(2, 256, 128)})
    codes, scales = model["left"].weight.data.clone(), model["left"].weight_scale_inv.data.clone()
    model = ggml_convert_low_bit(model, FP8, torch_dtype=torch.bfloat16, modules_to_not_convert=["left", "experts"])
    assert model["norm"].weight.dtype == torch.bfloat16 and type(model["other"]) is bf.BlockFP8Linear
    left = model["left"]
    assert left.weight.dtype == u.E4M3 and torch.equal(left.weight.float(), codes.float()) and torch.equal(left.weight_scale_inv, scales)
    assert model["experts"].down_proj.dtype == u.E4M3 and model["experts"].down_proj_scale_inv.dtype == torch.float32


def write_checkpoint(path, model, apart=("lm_head",)):
    """A Hugging Face directory whose projections are block-scaled, but for those that `apart` names."""
    from safetensors.torch import save_file
    state = {}
    for name, v in model.state_dict().items():
        if v.dim() == 3:                                     # experts, one by one
            for e, w in enumerate(v):
                for part, t in zip(("gate_proj", "up_proj"), w.chunk(2)) if name.endswith("gate_up_proj") else (("down_proj", w),):
                    at = f"{name.rpartition('.')[0]}.{e}.{part}.weight"
                    codes, state[at + "_scale_inv"] = u.quantize(t, 128)
                    state[at] = codes.float().to(u.E4M3)
        elif name.endswith("proj.weight") and not any(a in name for a in apart):
            codes, state[name + "_scale_inv"] = u.quantize(v, 128)
            state[name] = codes.float().to(u.E4M3)
        else:
            state[name] = v.bfloat16()
    model.config.architectures, model.config.dtype = [type(model).__name__], torch.bfloat16
    model.config.quantization_config = {"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "dynamic",
                                        "modules_to_not_convert": list(apart)}
    model.config.save_pretrained(path)
    save_file({k: v.contiguous() for k, v in state.items()}, str(path / "model.safetensors"), metadata={"format": "pt"})
    return state


@pytest.mark.parametrize("apart", [("lm_head",), ("lm_head", "model.layers.0.self_attn")], ids=["all", "mixed"])
def test_a_block_scaled_checkpoint_loads_moves_saves_and_loads(apart, tmp_path, monkeypatch):
    from ipex_llm.transformers import AutoModelForCausalLM
    held = write_checkpoint(tmp_path, tiny_llama(), apart)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)          # transformers reads such a checkpoint where a GPU is
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda *a: (9, 5))
    model = AutoModelForCausalLM.from_pretrained(str(tmp_path), load_in_low_bit="fp8_e4m3", torch_dtype=torch.bfloat16,
                                                 modules_to_not_convert=list(apart))
    monkeypatch.undo()
    layers = model.model.layers
    assert type(layers[0].mlp.up_proj) is bf.BlockFP8Linear and type(layers[1].self_attn.q_proj) is bf.BlockFP8Linear
    for move, dtype in ((model.half, torch.float16), (model.float, torch.float32), (model.bfloat16, torch.bfloat16)):
        move()
        assert model.model.embed_tokens.weight.dtype == dtype
        for name, v in model.state_dict().items():
            if name in held and held[name].dtype == u.E4M3:
                assert v.dtype == u.E4M3 and torch.equal(v.float(), held[name].float())
                assert torch.equal(model.state_dict()[name + "_scale_inv"], held[name + "_scale_inv"])
    model.save_low_bit(str(tmp_path / "low"))
    again = AutoModelForCausalLM.load_low_bit(str(tmp_path / "low"))
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got) and all(torch.equal(got[k].float(), v.float()) and got[k].dtype == v.dtype for k, v in want.items())
    assert again.half().model.embed_tokens.weight.dtype == torch.float16


def test_a_checkpoint_with_layers_left_to_its_quantizer_stays_its(tmp_path, monkeypatch):
    from ipex_llm.transformers import AutoModelForCausalLM
    write_checkpoint(tmp_path, tiny_llama())
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda *a: (9, 5))
    model = AutoModelForCausalLM.from_pretrained(str(tmp_path), load_in_low_bit="fp8_e4m3", torch_dtype=torch.bfloat16,
                                                 modules_to_not_convert=["lm_head", "layers.2"])
    with pytest.raises(ValueError, match="half"):
        model.half()                                         # would turn codes into numbers without their scales


def test_a_block_scaled_checkpoint_with_experts_loads_saves_and_loads(tmp_path, monkeypatch):
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM
    from ipex_llm.transformers import AutoModelForCausalLM
    torch.manual_seed(5)
    dense = Qwen3MoeForCausalLM(Qwen3MoeConfig(hidden_size=256, intermediate_size=384, moe_intermediate_size=128, num_experts=4, num_experts_per_tok=2,
                                               num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2, vocab_size=64)).eval()
    held = write_checkpoint(tmp_path, dense, ("lm_head", "mlp.gate"))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda *a: (9, 5))
    model = AutoModelForCausalLM.from_pretrained(str(tmp_path), load_in_low_bit="fp8_e4m3", torch_dtype=torch.bfloat16,
                                                 modules_to_not_convert=["lm_head", "mlp.gate"])
    monkeypatch.undo()
    experts = model.model.layers[0].mlp.experts
    assert type(experts) is bf.BlockFP8Experts and experts.own_gate is None
    for e in range(4):
        at = f"model.layers.0.mlp.experts.{e}."
        gate_up = torch.cat([held[at + "gate_proj.weight"].float(), held[at + "up_proj.weight"].float()])
        assert torch.equal(experts.gate_up_proj[e].float(), gate_up)
        assert torch.equal(experts.gate_up_proj_scale_inv[e], torch.cat([held[at + p + ".weight_scale_inv"] for p in ("gate_proj", "up_proj")]))
        assert torch.equal(experts.down_proj[e].float(), held[at + "down_proj.weight"].float())
        assert torch.equal(experts.down_proj_scale_inv[e], held[at + "down_proj.weight_scale_inv"])
    model.half().save_low_bit(str(tmp_path / "low"))
    again = AutoModelForCausalLM.load_low_bit(str(tmp_path / "low"))
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got) and all(torch.equal(got[k].float(), v.float()) and got[k].dtype == v.dtype for k, v in want.items())


def test_sizes_of_the_gpu_tests_reach_every_number_of_waves():
    for dtype in (ggml.DT_F16, ggml.DT_BF16, ggml.DT_F32):
        assert {ggml.lowbit_block_fp8_waves(dtype, *s) for s in u.FEW_ROWS} == {4, 8, 16}
    assert {ggml.lowbit_block_fp8_experts_waves(*s) for s in u.FEW_PAIRS} == {8, 16}
    assert ggml.lowbit_block_fp8_waves(ggml.DT_BF16, 100, 4096, 4096) == 0 == ggml.lowbit_block_fp8_experts_waves(100, 2, 8, 4096, 256)
    for call in (lambda: ggml.lowbit_block_fp8_waves(ggml.DT_F16, 0, 16, 16), lambda: ggml.lowbit_block_fp8_waves(3, 1, 16, 16),
                 lambda: ggml.lowbit_block_fp8_experts_waves(1, 65, 1, 16, 128)):
        with pytest.raises(Exception, match="waves"):
            call()


def test_sizes_past_a_launch_are_refused_by_the_library():
    """One weight of 2^24 blocks, and experts whose rows or tiles pass 2^32 threads: by arithmetic, with nothing launched (there is no GPU)."""
    assert lib.lowbit_block_fp8_quantize_weight(P, 0, 1, 1 << 20, 1 << 18, P, P, None) == -3 and b"too large" in lib.lowbit_last_error()
    size = lib.lowbit_block_fp8_experts_workspace_bytes(1 << 21, 1, 2, 1 << 17, 128)
    assert lib.lowbit_block_fp8_experts(P, P, P, 0, 1 << 21, 1, 2, P, P, P, P, P, size, P, 0, 1 << 17, 128, 0, None) == -3
    size = lib.lowbit_block_fp8_linear_workspace_bytes(0, (1 << 22) - 1, (1 << 23) - 1, 128)
    assert size < 1 << 31                                    # (2^27 tiles; their sums are never split)
    size = lib.lowbit_block_fp8_backward_workspace_bytes(0, (1 << 22) - 1, 128, (1 << 23) - 16)
    assert lib.lowbit_block_fp8_backward(P, P, P, P, 0, (1 << 22) - 1, 128, (1 << 23) - 16, P, size, None) == -3


def test_the_experts_workspace_is_bounded_beside_what_goes_in():
    """Codes of x (as 16-bit numbers) and of h, and a GiB, or a KiB for each pair, of pairs' results: not all of them at once."""
    for tokens, top_k, n_exp, hidden, inter in ((512, 8, 256, 7168, 2048), (4096, 8, 256, 7168, 2048), (32768, 8, 256, 7168, 2048),
                                                (262144, 8, 128, 2048, 768), (1 << 21, 1, 8, 4096, 256), (100000, 2, 8, 4096, 14336)):
        pairs = tokens * top_k
        own = tokens * u.blocks(hidden) * (256 + 4) + pairs * (inter + inter // 32 + 8) + 4 * 257 * n_exp
        bound = own + max(1 << 30, pairs * 1024) + (1 << 16)
        assert lib.lowbit_block_fp8_experts_workspace_bytes(tokens, top_k, n_exp, hidden, inter) <= bound
    assert lib.lowbit_block_fp8_experts_workspace_bytes(512, 8, 256, 7168, 2048) > 512 * 8 * 7168 * 4      # (all at once where they fit)


def test_fp8_weights_without_scales_that_were_left_out_stay_left_out(tmp_path):
    from ipex_llm import optimize_model
    from ipex_llm.optimize import load_low_bit

    def model():
        plain = nn.Linear(128, 64, bias=False)
        plain.weight = nn.Parameter(torch.arange(64 * 128).view(64, 128).remainder(9).float().to(u.E4M3), requires_grad=False)
        return nn.ModuleDict({"plain": plain, "scaled": scaled_linear(128, 256)}).eval()
    want = optimize_model(model(), "fp8_e4m3", modules_to_not_convert=["plain"])
    want.save_low_bit(str(tmp_path))
    again = load_low_bit(model(), str(tmp_path))
    assert type(again["plain"]) is nn.Linear and type(again["scaled"]) is bf.BlockFP8Linear
    assert again["plain"].weight.dtype == u.E4M3 and torch.equal(again["plain"].weight.float(), want["plain"].weight.float())


def test_experts_take_no_second_launch_for_few_pairs_of_many_experts():
    """Up to 3200 pairs are placed in the rows' launch however many experts there are; where a second launch places them the workspace has 256 counts of each
    expert beside what another expert takes elsewhere, its offset."""
    for tokens, top_k, n_exp, apart in ((300, 8, 2100, 0), (800, 4, 4095, 0), (3200, 1, 2048, 0), (3201, 1, 2047, 0), (3201, 1, 2049, 1), (4097, 1, 900, 1)):
        assert ggml.lowbit_block_fp8_experts_plan(tokens, top_k, n_exp, 16, 128)[3] == apart
        size, more = (ggml._lib.lowbit_block_fp8_experts_workspace_bytes(tokens, top_k, e, 16, 128) for e in (n_exp, n_exp + 1))
        assert more - size == 1024 * apart or more - size == 1024 * apart + 256
