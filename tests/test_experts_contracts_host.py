"""CPU-only checks of what the modules and entries by experts promise beyond their results: conversions, constructor refusals, size queries."""
import pytest
import torch


def layer(dev="cpu", bias=True):
    from llmqrt_amd.linear import GatedExperts, SqW8A8GroupedLinear
    up, down = SqW8A8GroupedLinear(4, 64, 96, dev=dev), SqW8A8GroupedLinear(4, 48, 64, dev=dev)
    return GatedExperts(up, down, 2, torch.arange(4.0, device=dev) if bias else None)


@pytest.mark.parametrize("bias", [True, False])
def test_layer_from_the_meta_device(bias):
    """A layer that was built without memory takes memory and then its values, the scores' bias among them."""
    m = layer("meta", bias).to_empty(device="cpu")
    assert m.gate_up.qweight.device.type == "cpu" and (m.score_bias is None) == (not bias)
    m.load_state_dict(layer("cpu", bias).state_dict())
    if bias:
        assert m.score_bias.dtype == torch.float32 and torch.equal(m.score_bias, torch.arange(4.0))


def test_conversions_keep_the_scores_bias():
    for f in (lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.bfloat16), lambda m: m.to("meta").half()):
        m = f(layer())
        assert m.score_bias.dtype == torch.float32 and "score_bias" in m.state_dict() and m.gate_up.dtype in (torch.float16, torch.bfloat16)


def test_a_failed_conversion_leaves_the_layer_whole():
    m = layer()

    def fails(t):
        if t is m.score_bias:
            raise NotImplementedError("no")
        return t
    with pytest.raises(NotImplementedError):
        m._apply(fails)
    assert torch.equal(m.score_bias, torch.arange(4.0)) and "score_bias" in m.state_dict()


def test_a_layer_whose_sum_cannot_be_formed_is_refused():
    """combine_from_experts takes multiples of 8 channels: said when the layer is built, not behind four of its steps."""
    from llmqrt_amd.linear import FP8BlockGroupedLinear, GatedExperts, SqW8A8GroupedLinear
    for kind in (SqW8A8GroupedLinear, FP8BlockGroupedLinear):
        up = kind(4, 64, 96, dev="cpu")
        for n in (100, 4, 65):
            with pytest.raises(RuntimeError, match="multiple of 8"):
                GatedExperts(up, kind(4, 48, n, dev="cpu"), 2)
        GatedExperts(up, kind(4, 48, 104, dev="cpu"), 2)


def test_named_quantized_linears_names_the_modules_by_experts():
    from llmqrt_amd.checkpoint import named_quantized_linears
    from llmqrt_amd.linear import FP8BlockGroupedLinear, GatedExperts
    model = torch.nn.ModuleDict({"a": layer(), "b": GatedExperts(FP8BlockGroupedLinear(2, 64, 96, dev="cpu"), FP8BlockGroupedLinear(2, 48, 64, dev="cpu"), 1),
                                 "router": torch.nn.Linear(64, 4)})
    assert [n for n, _ in named_quantized_linears(model)] == ["a.gate_up", "a.down", "b.gate_up", "b.down"]


def test_dispatch_workspace_bound_of_the_header():
    """The header names a number of rows up to which no workspace is needed, whatever the experts; it says nothing that the size query does not."""
    import pathlib
    import re
    from llmqrt_amd import _abi
    need = _abi.lib().llmq_dispatch_experts_workspace_bytes
    text = (pathlib.Path(__file__).resolve().parent.parent / "include" / "llmq.h").read_text()
    rows = int(re.search(r"none is needed for up to (\d+) rows, whatever the experts", text)[1])
    for experts in (1, 60, 255, 256, 257, 512, 1000, 1024, 2048, 4095, 4096):
        for top in (1, 2, 7, 8, 64):
            for n in range(max(1, rows // top - 300), rows // top + 1):
                assert need(n, top, experts) == 0
    assert need(14200, 1, 4096) > 0 and need(18200, 1, 1024) > 0  # near the bound: another figure would not do


def test_rows_are_quantized_on_their_own_device(monkeypatch):
    """The current device may be another than the activations': the quantizer in front of the product launches with theirs as the current one."""
    import contextlib
    from torch._subclasses.fake_tensor import FakeTensorMode
    from llmqrt_amd.linear import SqW8A8GroupedLinear
    from llmqrt_amd.linear import linear_sq_grouped as mod
    current, seen = [torch.device("cuda:0")], []

    @contextlib.contextmanager
    def device(d):
        current.append(torch.device(d))
        yield
        current.pop()

    def quantizer(x):
        seen.append((x.device, current[-1]))
        return x, x
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(mod, "quantize_activation_per_token_absmax_f32", quantizer)
    monkeypatch.setattr(mod, "w8a8_int8_linear_per_channel_grouped", lambda *a: a[0])
    m = SqW8A8GroupedLinear(2, 64, 40, dev="cpu")
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(3, 64, dtype=torch.bfloat16, device="cuda:1")
        m(x, None)
    assert seen == [(torch.device("cuda:1"), torch.device("cuda:1"))] and current == [torch.device("cuda:0")]
    with pytest.raises(RuntimeError):
        m(torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32))
