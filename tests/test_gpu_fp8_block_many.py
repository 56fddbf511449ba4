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


def exact_operands(m, n, k, seed, dev):
    """Whole numbers and powers of two: every sum is exact in fp32, so the output's rounding is the only one."""
    g = torch.Generator().manual_seed(seed)
    b = -(-k // 128)
    a, w = torch.randint(-3, 4, (m, k), generator=g).float().to(E4M3), torch.randint(-2, 3, (n, k), generator=g).float().to(E4M3)
    sa, sw = torch.pow(2.0, torch.randint(-1, 2, (m, b), generator=g).float()), torch.pow(2.0, torch.randint(-1, 2, (-(-n // 128), b), generator=g).float())
    return a.to(dev), w.to(dev), sa.to(dev), sw.to(dev)


def product64(a, w, sa, sw):
    k, n = a.shape[1], w.shape[0]
    x = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    return x @ (w.double() * sw.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(128, 0)[:n]).t()


@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("N", [16384, 16385, 24001, 37888, 49300])
@pytest.mark.parametrize("K", [16, 144, 512, 912, 1040, 2064])
def test_group_after_group(cuda, force, M, N, K):
    """One to five stages of K per group, whole and ragged, in a ring of three; last blocks with fewer groups than the others, a last group of one channel;
    with and without a bias, which is indexed by group; the configuration forced and the planner's choice."""
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise
    if N > 16384:
        assert groups(N) > 1
    a, w, sa, sw = exact_operands(M, N, K, M + N + K, cuda)
    ref = product64(a, w, sa, sw)
    for bias in (None, torch.bfloat16, torch.float16, torch.float32):
        b = None if bias is None else torch.randint(-8, 9, (N,), generator=torch.Generator().manual_seed(K)).to(bias).to(cuda)
        want = ref if b is None else ref + b.double()
        for cfg in (MANY, -1):
            assert force(cfg, 0) == 0
            for dtype, name in ((torch.bfloat16, "bfloat16"), (torch.float16, "float16")):
                y = f8f8_blockwise(a, w.t(), b, sa, sw, name)
                assert bool(torch.equal(y, want.to(dtype))), f"configuration {cfg}, bias {bias}, {name}"


def test_groups_in_a_graph_and_on_two_streams(cuda, force):
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise
    cases = [exact_operands(7, 24001, 1040, s, cuda) for s in (1, 2)]
    run = lambda c: f8f8_blockwise(c[0], c[1].t(), None, c[2], c[3])  # noqa: E731
    assert force(MANY, 0) == 0
    for c in cases:
        run(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [run(c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(3):
        cases[0][2].mul_(2.0)
        torch.cuda.synchronize()
        graph.replay()
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(run(c))
        torch.cuda.synchronize()
        for c, y, z in zip(cases, ys, got):
            ref = product64(c[0], c[1], c[2], c[3]).bfloat16()
            assert bool(torch.equal(y, ref)) and bool(torch.equal(z, ref))
