"""GPU: the block-scaled product for a few tokens and many channels, where a block takes one group of 64 channels after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
MANY = 14    # the configuration: up to 16 tokens, 64 channels at a time, 256 blocks resident
RESIDENT, CHANNELS, MOST = 256, 64, 16


def groups(n):
    """Groups of channels of the first block."""
    parts = -(-n // CHANNELS)
    each = min(MOST, -(-parts // RESIDENT))
    return -(-parts // -(-parts // each))


@pytest.fixture
def force():
    from llmqrt_amd import _abi
    yield _abi.lib().llmq_gemm_fp8_block_force_plan
    assert _abi.lib().llmq_gemm_fp8_block_force_plan(-1, 0) == 0


def test_the_most_channels(cuda, force):
    """Nearly 2^31 channels, the most that the product takes: 34 GB of weights, a step from group to group that ends past 2^31 behind the last one."""
    from llmqrt_amd import _abi
    N, K = 0x7FFFFF00, 16
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of GPU memory")
    assert groups(N) == MOST
    step = -(-(-(-N // CHANNELS)) // MOST) * CHANNELS
    at = torch.tensor([0, 63, 64, step - 1, step, 7 * step + 5, 15 * step, N - 65, N - 1], device=cuda)
    a = torch.ones(1, K, device=cuda).to(E4M3)
    w = torch.zeros(N, K, dtype=torch.uint8, device=cuda)
    w[at] = torch.full((K,), 2.0, device=cuda).to(E4M3).view(torch.uint8)
    sa, sw = torch.ones(1, 1, device=cuda), torch.ones(N // 128, 1, device=cuda)
    out = torch.full((1, N), 7.0, dtype=torch.bfloat16, device=cuda)
    assert force(MANY, 0) == 0
    _abi.check(_abi.lib().llmq_gemm_fp8_block(a.data_ptr(), K, sa.data_ptr(), w.data_ptr(), K, sw.data_ptr(), None, _abi.BF16, out.data_ptr(), _abi.BF16, N, 1, N, K,
                                              None, 0, torch.cuda.current_stream().cuda_stream), "llmq_gemm_fp8_block")
    assert (out[0, at] == 2 * K).all()
    out[0, at] = 0
    assert not any(bool(part.any()) for part in out.view(-1).split(1 << 28))
    del w, out
    torch.cuda.empty_cache()
