"""CPU-only checks of the block-scaled FP8 modules: conversions, and what a module may be made from."""
import copy

import pytest
import torch

E4M3 = torch.float8_e4m3fn


def module(grouped, bias):
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    g = torch.Generator().manual_seed(1)
    m = FP8BlockGroupedLinear(3, 256, 200, bias, dev="cpu") if grouped else FP8BlockLinear(256, 200, bias, dev="cpu")
    m.set_weight(torch.randn(m.weight.shape, generator=g), torch.randn(m.bias.shape, generator=g) if bias else None)
    return m


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("grouped", [True, False])
def test_conversions(grouped, bias):
    """A conversion changes the type of the bias and of the outputs, whether there is a bias or not; codes and scales keep theirs."""
    m = module(grouped, bias)
    w, s = m.weight.clone(), m.weight_scale.clone()

    def holds(dtype, bias_dtype=None):
        assert m.dtype == dtype
        assert m.weight.dtype == E4M3 and torch.equal(m.weight.view(torch.uint8), w.view(torch.uint8))
        assert m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, s)
        assert m.bias is None if not bias else m.bias.dtype == (bias_dtype or dtype)
    holds(torch.bfloat16)
    assert m.half() is m
    holds(torch.float16)
    m.to(torch.bfloat16)
    holds(torch.bfloat16)
    m.to("cpu")
    holds(torch.bfloat16)
    m.float()  # outputs are bf16 or fp16; an fp32 bias is one that the products take
    holds(torch.bfloat16, torch.float32)
    m.half()
    holds(torch.float16)
    m = copy.deepcopy(torch.nn.Sequential(m)).to(torch.bfloat16)[0]
    holds(torch.bfloat16)
    m.to("meta")
    assert m.weight.device.type == "meta" and m.weight.dtype == E4M3 and m.weight_scale.dtype == torch.float32 and m.dtype == torch.bfloat16


def test_tensors_that_require_grad_are_not_written():
    """(Refused before anything else is looked at, so also without a GPU.)"""
    from llmqrt_amd import norm as N
    from llmqrt_amd.linear import FP8BlockGroupedLinear
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise_grouped
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    leaf = torch.zeros(4, 64, dtype=torch.bfloat16, requires_grad=True)
    for r in (leaf, leaf * 2, (leaf * 2)[:]):
        for f in (N.add_rmsnorm, N.add_rmsnorm_quantize_activation_per_token_absmax, N.add_rmsnorm_per_token_quantize, N.add_rmsnorm_per_group_quantize):
            with pytest.raises(RuntimeError, match="requires grad"):
                f(x, r, w, inplace=True)
        with pytest.raises(RuntimeError, match="requires grad"):
            N.RMSNorm(w).forward_add(x, r, inplace=True)
    with torch.inference_mode():
        made = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="inference"):
        N.add_rmsnorm(x, made, w, inplace=True)
    out = torch.zeros(4, 200, dtype=torch.bfloat16, requires_grad=True)
    m, off = FP8BlockGroupedLinear(1, 64, 200, dev="cpu"), torch.tensor([0, 4], dtype=torch.int32)
    q, s = torch.zeros(4, 64, dtype=E4M3), torch.ones(4, 1)
    with pytest.raises(RuntimeError, match="requires grad"):
        f8f8_blockwise_grouped(q, m.weight, None, s, m.weight_scale, off, out=out)
    with pytest.raises(RuntimeError, match="requires grad"):
        m.forward_quantized(q, s, off, out)


def test_rows_that_partly_overlap():
    """The rule on addresses against the sets of elements, for rows anywhere in one buffer."""
    from llmqrt_amd.norm import _partly_over
    buf = torch.arange(200, dtype=torch.int16)
    for m in (1, 2, 5):
        for k in (1, 4, 7):
            for ld in (k, k + 1, 2 * k, 2 * k + 3):
                b = buf.as_strided((m, k), (ld, 1), 40)
                mine = set(b.flatten().tolist())
                for at in range(0, 120):
                    a = buf.as_strided((m, k), (ld, 1), at)
                    want = a.data_ptr() != b.data_ptr() and bool(mine & set(a.flatten().tolist()))
                    assert _partly_over(a, b) == want and _partly_over(b, a) == want, (m, k, ld, at)
    a, b = buf.as_strided((3, 4), (8, 1), 0), buf.as_strided((3, 4), (12, 1), 0)
    assert _partly_over(a, b) and not _partly_over(a, buf.as_strided((3, 4), (12, 1), 20))


@pytest.mark.parametrize("bias", [True, False])
def test_experts_of_quantized_modules(bias):
    """The codes, scales and biases of FP8BlockLinear modules, as they are."""
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    g = torch.Generator().manual_seed(3)
    plain = [torch.nn.Linear(144, 200, bias=bias) for _ in range(3)]
    for p in plain:
        p.weight.data = torch.randn(200, 144, generator=g)
    parts = [FP8BlockLinear.from_linear(p, init_only=False, dtype=torch.float16) for p in plain]
    m = FP8BlockGroupedLinear.from_linears(torch.nn.ModuleList(parts))
    assert m.dtype == torch.float16 and m.num_experts == 3
    for e, p in enumerate(parts):
        assert torch.equal(m.weight[e].view(torch.uint8), p.weight.view(torch.uint8)) and torch.equal(m.weight_scale[e], p.weight_scale)
        assert m.bias is None if not bias else torch.equal(m.bias[e], p.bias)
    quantized_here = FP8BlockGroupedLinear.from_linears(plain)
    assert quantized_here.dtype == torch.bfloat16 and torch.equal(quantized_here.weight.view(torch.uint8), m.weight.view(torch.uint8))
    assert FP8BlockGroupedLinear.from_linears(parts, torch.bfloat16).dtype == torch.bfloat16
    other = FP8BlockLinear.from_linear(plain[0], init_only=False)
    for bad in ([], [parts[0], plain[1]], [plain[0], parts[1]], [parts[0], other], [parts[0], FP8BlockLinear(144, 72, bias, dev="cpu", dtype=torch.float16)],
                [parts[0], FP8BlockLinear(144, 200, not bias, dev="cpu", dtype=torch.float16)]):
        with pytest.raises(RuntimeError):
            FP8BlockGroupedLinear.from_linears(bad)


def test_codes_are_not_quantized_again():
    """Codes without their scales are no weight: the result would be right but for factors that nobody sees."""
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear, FP8DynamicLinear
    lin = torch.nn.Linear(64, 72)
    block, token = FP8BlockLinear.from_linear(lin, init_only=False), FP8DynamicLinear.from_linear(lin, init_only=False, per_tensor=False)
    for m in (block, token):
        with pytest.raises(RuntimeError, match="quantized already"):
            FP8BlockLinear.from_linear(m, init_only=False)
    with pytest.raises(RuntimeError, match="quantized already"):
        FP8BlockGroupedLinear.from_linears([token, token])
    with pytest.raises(RuntimeError):
        block.set_weight(block.weight, block.bias)
    for bias in (torch.zeros(1), torch.zeros(1, 72), torch.zeros(())):
        with pytest.raises(RuntimeError):
            block.set_weight(lin.weight, bias)
    empty = FP8BlockLinear.from_linear(token)  # sizes only
    assert empty.weight.shape == (72, 64)
