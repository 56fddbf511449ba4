"""CPU-only checks of the modules by experts: interfaces, conversions, experts of quantized modules, refusals."""
import pytest
import torch


def linears(n, k, m, bias, seed=0):
    torch.manual_seed(seed)
    return [torch.nn.Linear(k, m, bias=bias) for _ in range(n)]


@pytest.mark.parametrize("bias", [False, True])
def test_experts_of_linears_and_of_quantized_modules(bias):
    from llmqrt_amd.linear import SqW8A8BBF16OBF16PerChannel, SqW8A8GroupedLinear
    mods = linears(3, 64, 40, bias)
    lin = SqW8A8GroupedLinear.from_linears(mods)
    singles = [SqW8A8BBF16OBF16PerChannel.from_linear(m, 8, 0, init_only=False, dtype=torch.bfloat16) for m in mods]
    same = SqW8A8GroupedLinear.from_linears(singles)
    for a in (lin, same):
        assert a.qweight.shape == (3, 40, 64) and a.qweight.dtype == torch.int8 and a.weight_scale.shape == (3, 40) and a.weight_scale.dtype == torch.float32
        assert (a.bias is not None) == bias and a.dtype == torch.bfloat16
        for e, s in enumerate(singles):
            assert torch.equal(a.qweight[e], s.qweight) and torch.equal(a.weight_scale[e], s.weight_scale)
            if bias:
                assert torch.equal(a.bias[e], s.bias)
            w = mods[e].weight.detach()
            assert ((a.qweight[e].float() * a.weight_scale[e][:, None] - w).abs() <= a.weight_scale[e][:, None] * 0.5001).all()
    assert sorted(lin.state_dict()) == (["bias"] if bias else []) + ["qweight", "weight_scale"]
    again = SqW8A8GroupedLinear(3, 64, 40, bias, dev="cpu")
    again.load_state_dict(lin.state_dict())
    assert torch.equal(again.qweight, lin.qweight)


@pytest.mark.parametrize("bias", [False, True])
def test_conversions(bias):
    from llmqrt_amd.linear import SqW8A8GroupedLinear
    m = SqW8A8GroupedLinear(2, 32, 16, bias, dev="cpu")
    for dtype, f in ((torch.float16, lambda: m.half()), (torch.bfloat16, lambda: m.bfloat16()), (torch.float16, lambda: m.to(torch.float16))):
        f()
        assert m.dtype == dtype and m.qweight.dtype == torch.int8 and m.weight_scale.dtype == torch.float32
        assert m.bias is None or m.bias.dtype == dtype
    assert "num_experts=2" in repr(m)


def test_refusals():
    from llmqrt_amd.linear import SqW8A8BBF16OBF16PerChannel, SqW8A8GroupedLinear
    plain = linears(2, 64, 40, False)
    single = SqW8A8BBF16OBF16PerChannel.from_linear(plain[0], 8, 0, init_only=False)
    other = SqW8A8BBF16OBF16PerChannel.from_linear(plain[0], 8, 0, init_only=False, dtype=torch.bfloat16)
    for bad in ([], [plain[0], single], [single, other], [plain[0], linears(1, 64, 48, False)[0]], [plain[0], linears(1, 64, 40, True)[0]], [torch.nn.Conv1d(1, 1, 1)]):
        with pytest.raises((RuntimeError, AttributeError)):
            SqW8A8GroupedLinear.from_linears(bad)
    for k in (24, 1 << 17):
        with pytest.raises(RuntimeError):
            SqW8A8GroupedLinear(1, k, 8, dev="meta")
    with pytest.raises(RuntimeError):
        SqW8A8GroupedLinear(1, 32, 8, dev="cpu", dtype=torch.float32)
    m = SqW8A8GroupedLinear(2, 64, 40, dev="cpu")
    for x in (torch.zeros(3, 64), torch.zeros(3, 48, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError):
            m(x, torch.zeros(3, dtype=torch.int32))


def test_gated_experts_interface():
    from llmqrt_amd.linear import FP8BlockGroupedLinear, GatedExperts, SqW8A8GroupedLinear
    up, down = SqW8A8GroupedLinear(4, 64, 96, dev="cpu"), SqW8A8GroupedLinear(4, 48, 64, dev="cpu")
    m = GatedExperts(up, down, 2, torch.zeros(4), scoring="sigmoid", num_groups=2, group_score="top2")
    assert {"gate_up.qweight", "down.qweight", "score_bias"} <= set(m.state_dict())
    m.half()
    assert m.score_bias.dtype == torch.float32 and m.gate_up.dtype == torch.float16 and m.gate_up.weight_scale.dtype == torch.float32
    assert "score_bias" in m.state_dict() and "sigmoid" in repr(m)
    with pytest.raises(RuntimeError):
        m(torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 4))
    with pytest.raises(RuntimeError):
        m(torch.zeros(3, 64, dtype=torch.float16), torch.zeros(2, 4))
    for args, kw in (((up, SqW8A8GroupedLinear(3, 48, 64, dev="cpu"), 2), {}), ((up, SqW8A8GroupedLinear(4, 96, 64, dev="cpu"), 2), {}),
                     ((up, FP8BlockGroupedLinear(4, 48, 64, dev="cpu"), 2), {}), ((torch.nn.Linear(2, 2), down, 2), {}), ((up, down, 2), {"temperature": 1.0}),
                     ((up, SqW8A8GroupedLinear(4, 48, 64, dev="cpu"), 2), {})):  # the last: bf16 beside fp16
        with pytest.raises(RuntimeError):
            GatedExperts(*args, **kw)
