"""GPU: NaN and infinities in block-scaled products, on every configuration: in the whole and the ragged blocks of K, in codes and in scales, shared by groups
of wavefronts, K splits and experts.

Codes are small whole numbers and scales powers of two or infinite, so that every finite sum is exact in fp32; what is not finite is the same in any order of
the sum (inf + inf = inf, inf - inf = NaN, inf * 0 = NaN).  Results have to be the definition's bits, a NaN for each NaN."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
TILES = range(8)
ROWS = {8: 16, 9: 16, 10: 32, 11: 48, 12: 48, 13: 64, 14: 16}  # the row-streaming configurations, and how many tokens each takes


def blocks(n):
    return (n + 127) // 128


def operands(M, N, K, seed, dev, positive):
    g = torch.Generator().manual_seed(seed)
    a, w = torch.randint(1 if positive else -3, 4, (M, K), generator=g).float(), torch.randint(1 if positive else -2, 3, (N, K), generator=g).float()
    sa = torch.pow(2.0, torch.randint(-1, 2, (M, blocks(K)), generator=g).float())
    sw = torch.pow(2.0, torch.randint(-1, 2, (blocks(N), blocks(K)), generator=g).float())
    return a.to(E4M3).to(dev), w.to(E4M3).to(dev), sa.to(dev), sw.to(dev)


def definition(a, w, sa, sw):
    y = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=a.device)
    for b in range(sa.shape[1]):
        part = slice(128 * b, min(128 * (b + 1), a.shape[1]))
        p = a[:, part].double() @ w[:, part].double().t()
        y += sa[:, b:b + 1].double() * sw[:, b].double().repeat_interleave(128)[:w.shape[0]] * p
    return y.bfloat16()


def same(y, ref):
    return bool(torch.equal(y.isnan(), ref.isnan())) and bool(torch.equal(y.nan_to_num(0.0, posinf=3e38, neginf=-3e38), ref.nan_to_num(0.0, posinf=3e38, neginf=-3e38)))


def check_all(a, w, sa, sw, what):
    from llmqrt_amd import _abi
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
    M, K = a.shape
    ref = definition(a, w, sa, sw)
    off = torch.tensor([0, 1, max(M - 3, 1), max(M - 3, 1), M], dtype=torch.int32, device=a.device)
    wg, swg = w.expand(4, *w.shape).contiguous(), sw.expand(4, *sw.shape).contiguous()
    force = _abi.lib().llmq_gemm_fp8_block_force_plan
    try:
        for cfg in [-1, *TILES, *(c for c, most in ROWS.items() if M <= most)]:
            for splits in (1, 2, 3) if cfg in TILES else (1,):
                assert force(cfg, splits) == 0
                print(what, "configuration", cfg, "splits", splits, tuple(a.shape), tuple(w.shape), flush=True)
                assert same(f8f8_blockwise(a, w.t(), None, sa, sw), ref), f"{what}: configuration {cfg}, {splits} splits"
            if cfg < 8:
                assert same(f8f8_blockwise_grouped(a, wg, None, sa, swg, off), ref), f"{what}: configuration {cfg}, by experts"
    finally:
        force(-1, 0)


SIZES = [(M, N, K) for M, N in ((3, 260), (70, 200)) for K in (16, 144, 256, 400, 528, 656, 912, 1040, 1296)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_infinite_scales(cuda, M, N, K):
    """A scale of a token or of a block of weights that is infinite, in the first, a middle and the last block of K."""
    KB = blocks(K)
    for b in sorted({0, KB // 2, KB - 1}):
        a, w, sa, sw = operands(M, N, K, K + b, cuda, True)
        sa[M - 1, b] = float("inf")
        check_all(a, w, sa, sw, f"token's scale {b}")
        a, w, sa, sw = operands(M, N, K, K + b + 1, cuda, True)
        sw[-1, b] = float("inf")
        check_all(a, w, sa, sw, f"weights' scale {b}")
    a, w, sa, sw = operands(M, N, K, K + 7, cuda, False)  # products of both signs, and zeros: infinities of both signs, and NaN
    sa[0, KB - 1], sw[0, 0] = float("inf"), float("inf")
    check_all(a, w, sa, sw, "both signs")


@pytest.mark.parametrize("M,N,K", SIZES)
def test_nan_in_codes_and_scales(cuda, M, N, K):
    """A NaN reaches its token or channel (a scale's: its token, or its block of channels) and nothing else."""
    KB = blocks(K)
    for k in sorted({0, K // 2, 128 * (KB - 1), K - 1}):
        a, w, sa, sw = operands(M, N, K, K + k, cuda, False)
        a.view(torch.uint8)[M - 1, k] = 0x7F
        w.view(torch.uint8)[N - 1, K - 1 - k] = 0xFF
        check_all(a, w, sa, sw, f"codes {k}")
    a, w, sa, sw = operands(M, N, K, K + 3, cuda, False)
    sa[0, KB - 1], sw[-1, 0] = float("nan"), float("nan")
    check_all(a, w, sa, sw, "scales")
