"""Row-scaled int8 in models without a GPU: which layers are converted, what is refused, what moves, is saved and is found again."""
import pytest
import torch
from torch import nn

import row_int8_util as u
from ipex_llm import optimize_model
from ipex_llm.ggml.quantize import ggml_tensor_qtype
from ipex_llm.optimize import load_low_bit, row_int8_layers, unconverted_linears
from ipex_llm.transformers import row_int8 as ri
from ipex_llm.transformers.convert import ggml_convert_low_bit, is_row_int8

INT8 = ggml_tensor_qtype["sym_int8"]


def scaled_linear(n, k, bias=False, seed=1, column=False, dtype=torch.float32):
    """A checkpoint's layer: codes and scales, [n] or [n, 1]."""
    lin = nn.Linear(k, n, bias=bias)
    codes, scale = u.weight(torch.Generator().manual_seed(seed), n, k)
    lin.weight = nn.Parameter(codes, requires_grad=False)
    lin.weight_scale = nn.Parameter((scale.unsqueeze(-1) if column else scale).to(dtype), requires_grad=False)
    return lin


class FusedExperts(nn.Module):
    def __init__(self, e, h, i, limit=None, rows=True, column=False):
        super().__init__()
        gen = torch.Generator().manual_seed(5)
        self.act_fn, self.limit = nn.SiLU(), limit
        for name, n, k in (("gate_up_proj", 2 * i, h), ("down_proj", h, i)):
            codes, scale = u.weight(gen, n, k, (e,))
            setattr(self, name, nn.Parameter(codes if rows else torch.randn((e, n, k), generator=gen) * 0.05, requires_grad=False))
            if rows:
                setattr(self, name + "_scale", nn.Parameter(scale.unsqueeze(-1) if column else scale, requires_grad=False))

    def _apply_gate(self, gu):
        g, v = gu.chunk(2, dim=-1)
        return self.act_fn(g if self.limit is None else g.clamp(max=self.limit)) * v


def held(module, **more):
    for name, v in more.items():
        setattr(module, name, nn.Parameter(v, requires_grad=False) if isinstance(v, torch.Tensor) else v)
    return module


@pytest.mark.parametrize("column", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_conversion_keeps_a_checkpoints_codes(column, dtype):
    lin = scaled_linear(200, 272, True, column=column, dtype=dtype)
    assert is_row_int8(lin) and not is_row_int8(nn.Linear(16, 16))
    codes, scale = lin.weight.data.clone(), lin.weight_scale.data.clone().float().view(-1)
    model = ggml_convert_low_bit(nn.Sequential(lin, nn.ReLU()).eval(), INT8, torch_dtype=torch.bfloat16)
    new = model[0]
    assert type(new) is ri.RowInt8Linear and not new.training and not any(p.requires_grad for p in new.parameters())
    assert torch.equal(new.weight, codes) and torch.equal(new.weight_scale, scale) and new.weight_scale.dtype == torch.float32
    assert set(new.state_dict()) == {"weight", "weight_scale", "bias"}
    assert torch.equal(new.dequantize(), codes.float() * scale.unsqueeze(-1))
    assert ggml_convert_low_bit(model, INT8)[0] is new       # converted layers stay as they are
    assert ggml_convert_low_bit(model, 2)[0] is new


def test_codes_that_start_between_sixteens_are_copied():
    lin = scaled_linear(8, 32)
    flat = torch.zeros(8 * 32 + 8, dtype=torch.int8)
    start = next(i for i in range(1, 8) if (flat.data_ptr() + i) % 16)
    flat[start:start + 256] = lin.weight.data.view(-1)
    lin.weight.data = flat[start:start + 256].view(8, 32)
    new = ri.RowInt8Linear.from_linear(lin)
    assert new.weight.data_ptr() % 16 == 0 and torch.equal(new.weight.data, lin.weight.data)


OTHER_FORMS = [
    ("dynamic", lambda: held(scaled_linear(32, 64), activation_scheme="static")),
    ("input_scale", lambda: held(scaled_linear(32, 64), input_scale=torch.ones(1))),
    ("weight_zero_point", lambda: held(scaled_linear(32, 64), weight_zero_point=torch.zeros(32))),
    ("2 groups", lambda: held(scaled_linear(32, 64), n_groups=2)),
    ("a scale for each row", lambda: held(scaled_linear(32, 64), weight_scale=torch.ones(32, 2))),
    ("a scale for each row", lambda: held(scaled_linear(32, 64), weight_scale=torch.ones(1))),
    ("a scale for each row", lambda: held(scaled_linear(32, 64), weight_scale=torch.ones(()))),
    ("multiple of 16", lambda: scaled_linear(32, 72)),
    ("dynamic", lambda: held(FusedExperts(2, 64, 32), activation_scheme="static")),
    ("gate_up_proj_bias", lambda: held(FusedExperts(2, 64, 32), gate_up_proj_bias=torch.ones(2, 64))),
    ("down_proj_scale", lambda: held(FusedExperts(2, 64, 32), down_proj_scale=torch.ones(2))),
    ("multiples of 16", lambda: FusedExperts(2, 64, 24)),
]


@pytest.mark.parametrize("message,make", OTHER_FORMS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(OTHER_FORMS)])
def test_other_forms_of_int8_checkpoints_are_refused(message, make):
    with pytest.raises(RuntimeError, match=message):
        ggml_convert_low_bit(nn.ModuleDict({"layer": make()}), INT8)
    model = ggml_convert_low_bit(nn.ModuleDict({"layer": make(), "other": scaled_linear(32, 64)}), INT8, modules_to_not_convert=["layer"])
    assert type(model["layer"]) in (nn.Linear, FusedExperts) and type(model["other"]) is ri.RowInt8Linear


def test_row_int8_asks_for_sym_int8():
    with pytest.raises(RuntimeError, match="use it with sym_int8"):
        optimize_model(nn.Sequential(nn.Linear(64, 64)), "sym_int4", row_int8=True)
    for make in (lambda: scaled_linear(32, 64), lambda: FusedExperts(2, 64, 32)):
        with pytest.raises(RuntimeError, match="sym_int8"):
            ggml_convert_low_bit(nn.Sequential(make()), 2)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ri.RowInt8Linear(24, 16)
    with pytest.raises(RuntimeError, match="at most"):
        ri.RowInt8Linear(ri.MOST_K + 16, 16)


def test_shape_only_conversion_of_dense_layers():
    with torch.device("meta"):
        model = nn.ModuleDict({"a": nn.Linear(272, 200), "b": nn.Linear(200, 100), "long": nn.Linear(ri.MOST_K + 16, 8),
                               "e": FusedExperts(3, 64, 48, rows=False), "f": FusedExperts(3, 64, 40, rows=False),
                               "biased": held(FusedExperts(2, 64, 32, rows=False), gate_up_proj_bias=torch.ones(2, 64)),
                               "grouped": held(nn.Linear(64, 32), n_groups=2)})
    model = model.to("meta")
    model = ggml_convert_low_bit(model, INT8, convert_shape_only=True, row_int8=True)
    assert type(model["a"]) is ri.RowInt8Linear and model["a"].weight.shape == (200, 272) and model["a"].weight_scale.shape == (200,)
    assert type(model["b"]) is nn.Linear and type(model["long"]) is nn.Linear and type(model["f"]) is FusedExperts
    assert type(model["e"]) is ri.RowInt8Experts and model["e"].gate_up_proj_scale.shape == (3, 96) and model["e"].down_proj.shape == (3, 64, 48)
    assert type(model["biased"]) is FusedExperts and type(model["grouped"]) is nn.Linear
    with torch.device("meta"):
        model = nn.Sequential(nn.Linear(256, 64), nn.Linear(256, 64))
    model = ggml_convert_low_bit(model, INT8, convert_shape_only=True, row_int8={"1"})
    assert type(model[1]) is ri.RowInt8Linear and type(model[0]).__name__ == "LowBitLinear"
    with torch.device("meta"):
        model = nn.Sequential(nn.Linear(256, 64))
    assert type(ggml_convert_low_bit(model, INT8, convert_shape_only=True)[0]).__name__ == "LowBitLinear"      # the format that was there


def test_codes_and_scales_keep_their_format_when_a_model_moves():
    for new in (ri.RowInt8Linear.from_linear(scaled_linear(130, 144, True)), ri.RowInt8Experts.from_fused(FusedExperts(2, 64, 32, column=True))):
        want = {n: p.data.clone() for n, p in new.named_parameters() if n != "bias"}
        for move in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu"), lambda m: m.float()):
            m = move(new)
            for n, v in want.items():
                assert m._parameters[n].dtype == v.dtype and torch.equal(m._parameters[n], v)
        assert all(p.dtype == (torch.float16 if n == "bias" else want[n].dtype) for n, p in new.half().named_parameters())
        assert all(p.device.type == "meta" for p in new.to("meta").parameters())


@pytest.mark.parametrize("limit", [None, 3.0])
def test_experts_keep_their_scales_and_a_gate_of_their_own(limit, monkeypatch):
    module = FusedExperts(3, 64, 32, limit, column=True).eval()
    new = ggml_convert_low_bit(nn.Sequential(module).eval(), INT8)[0]
    assert type(new) is ri.RowInt8Experts and not new.training and (new.own_gate is None) == (limit is None)
    assert torch.equal(new.down_proj, module.down_proj) and torch.equal(new.down_proj_scale, module.down_proj_scale[..., 0])
    # (the products by the formula: there is no GPU here)
    monkeypatch.setattr(ri, "row_int8_linear", lambda x, w, s: u.product(x, w, s))
    x, picks = torch.randn((6, 64), generator=torch.Generator().manual_seed(3)) * 8, torch.tensor([[0, 2]] * 5 + [[1, 7]])
    p, want = torch.full((6, 2), 0.5), torch.zeros((6, 64))
    for e in range(3):
        t, j = torch.where(picks == e)
        gu = u.product(x[t], module.gate_up_proj[e], module.gate_up_proj_scale[e, :, 0])
        want.index_add_(0, t, u.product(module._apply_gate(gu), module.down_proj[e], module.down_proj_scale[e, :, 0]) * 0.5)
    got = ri._expert_loop(x, picks, p, new.gate_up_proj, new.gate_up_proj_scale, new.down_proj, new.down_proj_scale, new.own_gate or ri._gated(new.act_fn))
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    if limit is not None:
        assert torch.equal(new(x, picks, p), got)
    assert new(x[:0], picks[:0], p[:0]).shape == (0, 64)


def test_projections_of_a_checkpoint_are_not_merged():
    from ipex_llm.transformers.models.common import merge_linear
    assert merge_linear([scaled_linear(32, 64), scaled_linear(32, 64)]) is None
    assert merge_linear([nn.Linear(64, 32), scaled_linear(32, 64)]) is None
    assert merge_linear([nn.Linear(32, 16), nn.Linear(32, 16)]) is not None


def tiny_llama():
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(4)
    return LlamaForCausalLM(LlamaConfig(hidden_size=256, intermediate_size=384, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                                        vocab_size=64)).eval()


@pytest.mark.parametrize("apart", [False, True], ids=["merged", "disable_optimize_pre"])
def test_a_model_with_some_layers_of_a_checkpoint_saves_and_loads(apart, tmp_path):
    model = tiny_llama()
    for part in (model.model.layers[1].self_attn, model.model.layers[1].mlp):
        for name, lin in list(part.named_children()):
            if isinstance(lin, nn.Linear):
                setattr(part, name, scaled_linear(*lin.weight.shape))
    model = optimize_model(model, "sym_int8", modules_to_not_convert=["layers.0", "layers.2", "lm_head"], disable_optimize_pre=apart)
    assert hasattr(model.model.layers[0].self_attn, "qkv_proj") != apart and not hasattr(model.model.layers[1].self_attn, "qkv_proj")
    model.save_low_bit(str(tmp_path))
    again = load_low_bit(tiny_llama(), str(tmp_path))
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got) and all(torch.equal(got[k], v) and got[k].dtype == v.dtype for k, v in want.items())
    assert type(again.model.layers[1].self_attn.q_proj) is ri.RowInt8Linear and type(again.model.layers[2].mlp.up_proj) is nn.Linear
    assert again.half().model.layers[1].mlp.up_proj.weight_scale.dtype == torch.float32


def test_saved_layers_are_found_again():
    state = nn.ModuleDict({"q": ri.RowInt8Linear.from_linear(scaled_linear(32, 64)), "head": nn.Linear(16, 16),
                           "experts": ri.RowInt8Experts.from_fused(FusedExperts(2, 64, 32))}).state_dict()
    assert row_int8_layers(state, "sym_int8") == {"q", "experts"} and row_int8_layers(state, "fp8_e4m3") == set()
    assert [n for n in unconverted_linears(state) if n not in row_int8_layers(state, "sym_int8")] == ["head"]


def test_a_hugging_face_model_saves_and_loads(tmp_path, monkeypatch):
    """from_pretrained with row_int8, and back; the quantizer by the formula: there is no GPU here."""
    from ipex_llm.transformers import AutoModelForCausalLM
    monkeypatch.setattr(ri, "_pack_weight", lambda w, shape_only=False: tuple(
        t.to(d) for t, d in zip(u.quantize(w), (torch.int8, torch.float32))) if w.device.type != "meta" else (
            torch.empty(w.shape, dtype=torch.int8, device="meta"), torch.empty(w.shape[:-1], device="meta")))
    tiny_llama().save_pretrained(str(tmp_path / "dense"))
    model = AutoModelForCausalLM.from_pretrained(str(tmp_path / "dense"), load_in_low_bit="sym_int8", row_int8=True, torch_dtype=torch.bfloat16)
    attention = model.model.layers[0].self_attn
    assert type(attention.qkv_proj) is ri.RowInt8Linear and attention.qkv_proj.weight_scale.dtype == torch.float32
    assert type(model.lm_head) is ri.RowInt8Linear
    model.save_low_bit(str(tmp_path / "low"))
    again = AutoModelForCausalLM.load_low_bit(str(tmp_path / "low"))
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got) and all(torch.equal(got[k], v) and got[k].dtype == v.dtype for k, v in want.items())


def test_layers_left_out_of_another_format_stay_left_out(tmp_path):
    """int8 codes among the layers of a model in another format, as they were."""
    def model():
        return nn.ModuleDict({"left": scaled_linear(32, 128), "other": nn.Linear(64, 32)}).eval()
    want = optimize_model(model(), "bf16", modules_to_not_convert=["left"])
    want.save_low_bit(str(tmp_path))
    again = load_low_bit(model(), str(tmp_path))
    assert type(again["left"]) is nn.Linear and again["left"].weight.dtype == torch.int8 and torch.equal(again["left"].weight, want["left"].weight)


LEFT_OUT = {
    "a column of scales": lambda: scaled_linear(32, 128, column=True),
    "a row of scales": lambda: scaled_linear(32, 128, True),
    "16-bit scales": lambda: scaled_linear(32, 128, dtype=torch.float16),
    "fixed scale of the activations": lambda: held(scaled_linear(32, 128), activation_scheme="static"),
    "zero points": lambda: held(scaled_linear(32, 128), weight_zero_point=torch.zeros(32)),
    "experts": lambda: FusedExperts(2, 64, 32),
    "experts with columns": lambda: FusedExperts(2, 64, 32, column=True),
}


def saved_and_loaded(model, folder, **kwargs):
    want = optimize_model(model(), "sym_int8", modules_to_not_convert=["left"], **kwargs)
    want.save_low_bit(str(folder))
    return want, lambda: load_low_bit(model(), str(folder))


@pytest.mark.parametrize("what", LEFT_OUT)
def test_layers_left_out_of_a_sym_int8_model_stay_left_out(what, tmp_path):
    """A checkpoint's int8 layers, some of them left out of the conversion: as they were after a model is saved and loaded, also where they hold the
    tensors of a converted one."""
    want, load = saved_and_loaded(lambda: nn.ModuleDict({"left": LEFT_OUT[what](), "other": scaled_linear(32, 64), "experts": FusedExperts(2, 64, 32)}).eval(),
                                  tmp_path)
    again = load()
    assert type(again["left"]) is type(LEFT_OUT[what]()) and type(again["other"]) is ri.RowInt8Linear and type(again["experts"]) is ri.RowInt8Experts
    assert want.state_dict().keys() == again.state_dict().keys()
    for name, v in want.state_dict().items():
        assert torch.equal(again.state_dict()[name], v) and again.state_dict()[name].dtype == v.dtype, name


@pytest.mark.parametrize("what", ["a column of scales", "zero points", "experts with columns"])
def test_models_saved_without_a_list_of_layers_load(what, tmp_path):
    """What no converted layer holds was left out."""
    import json
    _, load = saved_and_loaded(lambda: nn.ModuleDict({"left": LEFT_OUT[what](), "other": scaled_linear(32, 64, True), "experts": FusedExperts(2, 64, 32)}).eval(),
                               tmp_path)
    config = json.loads((tmp_path / "bigdl_config.json").read_text())
    assert config.pop("row_int8_layers") == ["other", "experts"]
    (tmp_path / "bigdl_config.json").write_text(json.dumps(config))
    again = load()
    assert type(again["left"]) is type(LEFT_OUT[what]()) and type(again["other"]) is ri.RowInt8Linear and type(again["experts"]) is ri.RowInt8Experts


def test_a_list_of_layers_goes_before_what_they_hold():
    state = {"low.weight": torch.zeros(8, dtype=torch.uint8), "left.weight": torch.zeros(4, 4), "q.weight": torch.zeros((4, 16), dtype=torch.int8),
             "q.weight_scale": torch.zeros(4)}
    assert row_int8_layers(state, "sym_int8") == {"q"} and row_int8_layers(state, "sym_int8", []) == set()
    assert row_int8_layers(state, "sym_int8", ["q"]) == {"q"} and row_int8_layers(state, "bf16", ["q"]) == set()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_layers_left_out_of_the_conversion_keep_their_scales(dtype, tmp_path):
    """Scales that 16 bits do not hold, of a linear, of one with fixed scales of its activations and zero points, and of experts with and without a
    module for their gate."""
    def model():
        def small(module):
            for name, p in module.named_parameters():
                if name.endswith("_scale"):
                    p.data = torch.arange(1, p.numel() + 1).view(p.shape) * 1.234567e-8
            return module
        bare = FusedExperts(2, 64, 32)
        bare.act_fn = None
        del bare._modules["act_fn"]
        static = held(scaled_linear(32, 128), input_scale=torch.tensor([1.234567e-3]), weight_zero_point=torch.full((32,), 0.1))
        return nn.ModuleDict({"left": small(scaled_linear(32, 128, True)), "left_static": small(static), "left_experts": small(FusedExperts(2, 64, 32)),
                              "left_bare": small(bare), "other": scaled_linear(32, 64), "norm": nn.LayerNorm(64)}).eval()
    before = model()
    after = optimize_model(model(), "sym_int8", modules_to_not_convert=["left"], torch_dtype=dtype)
    assert after["norm"].weight.dtype == dtype and type(after["other"]) is ri.RowInt8Linear and after["left"].bias.dtype == dtype
    after.save_low_bit(str(tmp_path))
    for m in (after, load_low_bit(model(), str(tmp_path))):
        for name, v in before.state_dict().items():
            if name.startswith("left") and not name.endswith("bias"):
                assert m.state_dict()[name].dtype == v.dtype and torch.equal(m.state_dict()[name], v), name
