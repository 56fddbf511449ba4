"""GPU: what the block-scaled operators promise beside their sums: types after a conversion, writes that autograd sees, infinite scales, channels of any
number."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def same(a, b):
    return bool(torch.equal(a, b))


@pytest.mark.parametrize("bias", [True, False])
def test_converted_modules_agree_on_their_type(cuda, bias):
    """After .half() both forward passes of a module return fp16 (the same bits: the same codes, scales and sums), plain and by experts."""
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    from llmqrt_amd.quantize import per_group_quantize
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 256, generator=g).half().to(cuda)
    q, s = per_group_quantize(x)
    offsets = torch.tensor([0, 4, 9], dtype=torch.int32, device=cuda)
    one, two = FP8BlockLinear(256, 200, bias, dev=cuda), FP8BlockGroupedLinear(2, 256, 200, bias, dev=cuda)
    for m, args in ((one, ()), (two, (offsets,))):
        m.set_weight(torch.randn(m.weight.shape, generator=g), torch.randn(m.bias.shape, generator=g) if bias else None)
        m = torch.nn.Sequential(m).half()[0]
        y = m.forward_quantized(q, s, *args)
        assert y.dtype == torch.float16 and same(m(x, *args), y)
