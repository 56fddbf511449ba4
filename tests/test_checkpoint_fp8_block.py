"""CPU-only: checkpoints of block-scaled FP8 modules."""
import json

import pytest
import torch
from safetensors.torch import save_file

E4M3 = torch.float8_e4m3fn


def model(*names, experts=0):
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    make = (lambda: FP8BlockGroupedLinear(experts, 256, 200, dev="cpu")) if experts else (lambda: FP8BlockLinear(256, 200, False, dev="cpu"))
    return torch.nn.ModuleDict({n: make() for n in names})


def codes(shape, seed):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * 100).clamp(-448, 448).to(E4M3)


@pytest.mark.parametrize("experts", [0, 3])
def test_only_codes_become_codes(tmp_path, experts):
    """Codes may be stored in a wider type; values that 8 bits do not hold are refused, and the module keeps what it had."""
    from llmqrt_amd.checkpoint import load_quantized_weights
    m = model("up", experts=experts)
    shape, scale = m["up"].weight.shape, torch.rand(m["up"].weight_scale.shape) + 0.5
    q = codes(shape, 1)
    for dtype in (E4M3, torch.bfloat16, torch.float16, torch.float32, torch.float8_e5m2):
        q = (q.float().sign() * 2).to(E4M3) if dtype == torch.float8_e5m2 else q
        m["up"].weight.zero_()
        save_file({"up.weight": q.to(dtype), "up.weight_scale": scale}, str(tmp_path / "m.safetensors"))
        assert load_quantized_weights(m, str(tmp_path)) == ([], [])
        assert torch.equal(m["up"].weight.view(torch.uint8), q.view(torch.uint8)) and torch.equal(m["up"].weight_scale, scale)
    for values in (torch.randn(shape) * 1000, torch.randn(shape) * 0.02, torch.full(shape, float("nan")), torch.full(shape, 480.0)):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            save_file({"up.weight": values.to(dtype), "up.weight_scale": scale}, str(tmp_path / "m.safetensors"))
            with pytest.raises(RuntimeError, match="codes"):
                load_quantized_weights(m, str(tmp_path))
            assert torch.equal(m["up"].weight.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("experts", [0, 3])
def test_codes_without_scales(tmp_path, experts):
    """A directory has to hold both; one file of several may hold either, and the rest is listed as missing."""
    from llmqrt_amd.checkpoint import load_quantized_weights
    m = model("up", "down", experts=experts)
    weight, scale = codes(m["up"].weight.shape, 2), torch.ones(m["up"].weight_scale.shape)
    save_file({"up.weight": weight, "up.weight_scale": scale, "down.weight": weight.clone()}, str(tmp_path / "a.safetensors"))
    with pytest.raises(RuntimeError, match="down.weight_scale"):
        load_quantized_weights(m, str(tmp_path))
    assert load_quantized_weights(m, str(tmp_path / "a.safetensors")) == (["down.weight_scale"], [])
    save_file({"down.weight_scale": scale}, str(tmp_path / "b.safetensors"))
    assert load_quantized_weights(m, str(tmp_path)) == ([], [])
    one = m["up"]  # a module by itself, whose names have no prefix
    (tmp_path / "c").mkdir()
    save_file({"weight": weight}, str(tmp_path / "c" / "m.safetensors"))
    with pytest.raises(RuntimeError, match="weight_scale"):
        load_quantized_weights(one, str(tmp_path / "c"))


def test_experts_are_named(tmp_path):
    from llmqrt_amd.checkpoint import named_quantized_linears
    m = torch.nn.ModuleDict({"a": model("up", experts=2), "b": model("up"), "c": torch.nn.Linear(16, 16)})
    assert [n for n, _ in named_quantized_linears(m)] == ["a.up", "b.up"]


class Expert(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.down_proj = torch.nn.Linear(144, 200, bias=False), torch.nn.Linear(208, 144, bias=False)


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.mlp = torch.nn.Module()
        self.mlp.gate = torch.nn.Linear(144, 2, bias=False)
        self.mlp.experts = torch.nn.ModuleList([Expert(), Expert()])
        self.lm_head = torch.nn.Linear(144, 16, bias=False)


def published(**config):
    return {"quantization_config": {"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [128, 128],
                                    "modules_to_not_convert": ["lm_head", "mlp.gate"], **config}}


def test_published_names(tmp_path):
    """quant_method "fp8" with weight_block_size, scales in weight_scale_inv, and a list of experts: replaced, filled, joined."""
    from llmqrt_amd.checkpoint import QuantConfig, load_quantized_weights, replace_linears
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    (tmp_path / "config.json").write_text(json.dumps(published()))
    cfg = QuantConfig.from_pretrained(str(tmp_path))
    assert (cfg.quant_method, cfg.q_group_size, cfg.w_bit) == ("fp8_dynamic_quant", 128, 8)
    assert QuantConfig.from_transformers_dict(cfg.to_transformers_dict()) == cfg
    m = Layer()
    names = [f"mlp.experts.{e}.{p}" for e in range(2) for p in ("gate_proj", "down_proj")]
    assert replace_linears(m, cfg) == names and all(isinstance(m.get_submodule(n), FP8BlockLinear) for n in names)
    sd = {"mlp.gate.weight": torch.randn(2, 144), "lm_head.weight": torch.randn(16, 144).bfloat16(), "other.weight_scale_inv": torch.ones(1)}
    for i, n in enumerate(names):
        sub = m.get_submodule(n)
        sd[f"{n}.weight"], sd[f"{n}.weight_scale_inv"] = codes(sub.weight.shape, i), torch.rand(sub.weight_scale.shape) + 0.5
    save_file(sd, str(tmp_path / "model.safetensors"))
    assert load_quantized_weights(m, str(tmp_path)) == ([], ["other.weight_scale_inv"])
    joined = FP8BlockGroupedLinear.from_linears([e.gate_proj for e in m.mlp.experts])
    for e in range(2):
        n = f"mlp.experts.{e}.gate_proj"
        assert torch.equal(joined.weight[e].view(torch.uint8), sd[f"{n}.weight"].view(torch.uint8)) and torch.equal(joined.weight_scale[e], sd[f"{n}.weight_scale_inv"])
    assert torch.equal(m.mlp.gate.weight, sd["mlp.gate.weight"])


@pytest.mark.parametrize("config", [dict(weight_block_size=None), dict(weight_block_size=[64, 64]), dict(activation_scheme="static")])
def test_other_fp8_checkpoints_are_refused(tmp_path, config):
    from llmqrt_amd.checkpoint import QuantConfig, replace_linears
    (tmp_path / "config.json").write_text(json.dumps(published(**config)))
    m = Layer()
    with pytest.raises(RuntimeError, match="quant_method 'fp8'"):
        replace_linears(m, QuantConfig.from_pretrained(str(tmp_path)))
    assert type(m.mlp.experts[0].gate_proj) is torch.nn.Linear


def test_codes_do_not_become_plain_weights(tmp_path):
    from llmqrt_amd.checkpoint import load_quantized_weights
    m = Layer()
    q = codes((2, 144), 1)
    for name in ("weight_scale_inv", "weight_scale"):
        save_file({"mlp.gate.weight": q, f"mlp.gate.{name}": torch.ones(1, 2)}, str(tmp_path / "m.safetensors"))
        with pytest.raises(RuntimeError, match="not quantized"):
            load_quantized_weights(m, str(tmp_path))
    save_file({"mlp.gate.weight": q}, str(tmp_path / "m.safetensors"))  # 8-bit values as they are, without scales
    assert "mlp.gate.weight" not in load_quantized_weights(m, str(tmp_path))[0] and torch.equal(m.mlp.gate.weight, q.float())


def test_other_names_stay_unexpected(tmp_path):
    from llmqrt_amd.checkpoint import load_quantized_weights
    m = model("up")
    save_file({"up.my_weight_scale_inv": torch.ones(2, 2)}, str(tmp_path / "m.safetensors"))
    assert load_quantized_weights(m, str(tmp_path)) == (["up.weight", "up.weight_scale"], ["up.my_weight_scale_inv"])
