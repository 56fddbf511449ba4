"""CPU-only: checkpoints of block-scaled FP8 modules."""
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
