"""GPU: block-scaled fp8 - the group quantizer, the product, the product by experts - against plain forms in 64 bits.

Two kinds of comparison.  Exact: codes that are small whole numbers and scales that are powers of two, so that every sum is exact in fp32 and the
only rounding is the output's; results have to be the same bits.  (The matrix instruction adds each run of 8 products in fixed point and keeps those down
to 2^-13 of the largest, test_gpu_gemm.py; products of whole numbers up to 3 lie closer together.)  General: |error| <= (eps(out) / 2) |y| +
c S with S = sum |a b| of the dequantized operands; c = 7 2^-14 for the other seven products of a run, each cut by at most 2^-14 of the largest, and
2 u (K + 3 KB + 2), u = 2^-24: each of the K additions of a sum, each scale product, each scaled addition and the bias loses at most u
of what it adds, doubled for matrix cores that cut instead of rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}


def same(a, b):
    return bool(torch.equal(a, b))  # (a plain bool: a failed assertion prints no tensors)


def blocks(n):
    return (n + 127) // 128


def spread(scale, k, n=None):
    s = scale.double().repeat_interleave(128, dim=-1)[..., :k]
    return s if n is None else s.repeat_interleave(128, dim=-2)[..., :n, :]


def exact_operands(m, n, k, seed, dev, lead=()):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-3, 4, (m, k), generator=g).float().to(E4M3)
    w = torch.randint(-2, 3, (*lead, n, k), generator=g).float().to(E4M3)
    sa = torch.pow(2.0, torch.randint(-1, 2, (m, blocks(k)), generator=g).float())
    sw = torch.pow(2.0, torch.randint(-1, 2, (*lead, blocks(n), blocks(k)), generator=g).float())
    return a.to(dev), w.to(dev), sa.to(dev), sw.to(dev)


def general_operands(m, n, k, seed, dev, lead=()):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(m, k, generator=g) * 90).clamp(-448, 448).to(E4M3)
    w = (torch.randn(*lead, n, k, generator=g) * 90).clamp(-448, 448).to(E4M3)
    sa = torch.rand(m, blocks(k), generator=g) * 0.05 + 1e-4
    sw = torch.rand(*lead, blocks(n), blocks(k), generator=g) * 1e-3 + 1e-6
    return a.to(dev), w.to(dev), sa.to(dev), sw.to(dev)


def product64(a, w, sa, sw, bias=None):
    k, n = a.shape[1], w.shape[0]
    x, y = a.double() * spread(sa, k), w.double() * spread(sw, k, n)
    out, s = x @ y.t(), x.abs() @ y.abs().t()
    return (out, s) if bias is None else (out + bias.double(), s + bias.double().abs())


def check_general(y, ref, s, k):
    c = 7 * 2.0 ** -14 + 2.0 ** -23 * (k + 3 * blocks(k) + 2)
    err = (y.double() - ref).abs()
    bound = torch.finfo(y.dtype).eps / 2 * ref.abs() * (1 + 1e-6) + c * s + 2.0 ** -25  # the last: fp16 results below the normal range
    assert torch.isfinite(y).all()
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3g} of the bound"


def gemm(a, w, sa, sw, bias=None, dtype=torch.bfloat16):
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise
    return f8f8_blockwise(a, w.t(), bias, sa, sw, NAMES[dtype])


# ---- group quantizer

def groups_ref(x):
    rows, k = x.shape
    full = torch.nn.functional.pad(x.float(), (0, blocks(k) * 128 - k)).view(rows, -1, 128)
    s = full.abs().amax(-1).clamp(min=1e-12) / 448.0
    q = (full / s[..., None]).clamp(-448, 448).to(E4M3)
    return q.view(rows, -1)[:, :k], s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 8), (1, 128), (3, 136), (5, 3584), (17, 120), (64, 264), (37, 18944), (700, 1000), (1030, 3584), (2100, 2056)])
def test_group_quantizer_bits(cuda, M, K, dtype):
    from llmqrt_amd.quantize import per_group_quantize
    from llmqrt_amd import workloads as W
    x = W.activations(M, K, M + K, dtype=dtype)
    x[0, : min(K, 128)] = 0                       # a group of zeros
    x[-1, -8:] *= 1e-3 if dtype == torch.float16 else 1e-30  # (a short last group of tiny values)
    q, s = per_group_quantize(x.to(cuda))
    qr, sr = groups_ref(x)
    assert q.dtype == E4M3 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == (M, blocks(K))
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu().view(torch.uint8), qr.view(torch.uint8))


def test_group_quantizer_strides_and_shapes(cuda):
    from llmqrt_amd.quantize import per_group_quantize
    big = torch.randn(40, 2048, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    for view in (big[:, :1000], big[:, 8:648], big[::3, 128:1152], big[:, 3:1003], big[:, ::2], big[7:8, :136], big.view(4, 10, 2048)):
        q, s = per_group_quantize(view)
        flat = view.reshape(-1, view.shape[-1]).cpu()
        qr, sr = groups_ref(flat)
        assert q.shape == view.shape and s.shape == (*view.shape[:-1], blocks(view.shape[-1]))
        assert torch.equal(q.cpu().view(torch.uint8).reshape(flat.shape), qr.view(torch.uint8)) and torch.equal(s.cpu().reshape(sr.shape), sr)
    q, s = per_group_quantize(big[:0])
    assert q.shape == (0, 2048) and s.shape == (0, 16)


def test_group_quantizer_infinities_stay_in_their_group(cuda):
    from llmqrt_amd.quantize import per_group_quantize
    x = torch.randn(6, 512, generator=torch.Generator().manual_seed(2)).bfloat16()
    x[1, 130], x[2, 5], x[4, 511] = float("inf"), float("nan"), float("-inf")
    q, s = per_group_quantize(x.to(cuda))
    qr, sr = groups_ref(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(sr)) and torch.equal(s.cpu().nan_to_num(1.0), sr.nan_to_num(1.0))
    assert torch.equal(q.cpu().float().isnan(), qr.float().isnan())
    assert torch.equal(q.cpu().float().nan_to_num(0.0), qr.float().nan_to_num(0.0))


# ---- the product

SIZES = [(1, 1, 16), (1, 128, 128), (2, 3, 144), (7, 130, 256), (16, 512, 384), (17, 96, 3584), (33, 257, 272), (64, 64, 2048), (65, 640, 640),
         (100, 129, 1040), (128, 256, 128), (200, 300, 400), (257, 513, 768), (300, 1000, 512), (1, 3584, 3584), (48, 1152, 896), (513, 260, 1168)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_exact(cuda, M, N, K, dtype):
    a, w, sa, sw = exact_operands(M, N, K, M * 3 + N * 5 + K, cuda)
    ref, _ = product64(a, w, sa, sw)
    assert same(gemm(a, w, sa, sw, None, dtype), ref.to(dtype))


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float16, torch.float32])
def test_product(cuda, M, N, K, bias):
    dtype = torch.float16 if bias == torch.float16 else torch.bfloat16
    a, w, sa, sw = general_operands(M, N, K, M + N + K, cuda)
    b = None if bias is None else torch.randn(N, generator=torch.Generator().manual_seed(N)).to(bias).to(cuda)
    check_general(gemm(a, w, sa, sw, b, dtype), *product64(a, w, sa, sw, b), K)


@pytest.fixture
def force():
    from llmqrt_amd import _abi
    yield _abi.lib().llmq_gemm_fp8_block_force_plan
    assert _abi.lib().llmq_gemm_fp8_block_force_plan(-1, 0) == 0


def all_configs():
    """The configurations that the hook accepts (a number past the last is refused)."""
    from llmqrt_amd import _abi
    f = _abi.lib().llmq_gemm_fp8_block_force_plan
    n = 0
    while f(n, 0) == 0:
        n += 1
    f(-1, 0)
    return range(n)


@pytest.mark.parametrize("M,N,K", [(1, 40, 16), (5, 128, 128), (40, 200, 384), (300, 520, 1296), (64, 1300, 640), (257, 257, 2064)])
@pytest.mark.parametrize("splits", [1, 3])
def test_every_plan_exact(cuda, force, M, N, K, splits):
    a, w, sa, sw = exact_operands(M, N, K, M + N + K + splits, cuda)
    bias = torch.randint(-8, 8, (N,), generator=torch.Generator().manual_seed(3)).float().to(cuda)
    ref, _ = product64(a, w, sa, sw, bias)
    for cfg in all_configs():
        print("plan", cfg, splits, M, N, K, flush=True)
        assert force(cfg, splits) == 0
        assert same(gemm(a, w, sa, sw, bias), ref.bfloat16()), f"configuration {cfg}, {splits} splits"


@pytest.mark.parametrize("K", [16, 112, 144, 256, 272, 400, 512, 528, 656, 784, 896, 912, 1040, 1280, 1424])
def test_every_plan_at_the_end_of_k(cuda, force, K):
    """Every number of blocks around the stages of a ring, whole ones and with a partial last one, shared by groups of wavefronts and by splits."""
    for M, N in ((130, 200), (33, 72)):
        a, w, sa, sw = exact_operands(M, N, K, K, cuda)
        ref = product64(a, w, sa, sw)[0].bfloat16()
        off = torch.tensor([0, 1, M - 20, M - 20, M], dtype=torch.int32, device=cuda)
        wg, swg = w.expand(4, N, K).contiguous(), sw.expand(4, *sw.shape).contiguous()
        for cfg in all_configs():
            for splits in (1, 2, 4):
                print("plan", cfg, splits, M, N, K, flush=True)
                assert force(cfg, splits) == 0
                assert same(gemm(a, w, sa, sw), ref), f"configuration {cfg}, {splits} splits"
            assert same(grouped(a, wg, sa, swg, off), ref), f"configuration {cfg}, by experts"


def test_product_strides(cuda):
    """Operands inside larger tensors, 16-byte aligned or not, and outputs of odd widths."""
    a, w, sa, sw = exact_operands(20, 50, 512, 9, cuda)
    ref = product64(a, w, sa, sw)[0].bfloat16()
    wide_a = torch.zeros(20, 1024, dtype=E4M3, device=cuda)
    wide_w = torch.zeros(50, 528, dtype=E4M3, device=cuda)
    for at in (0, 16, 5):
        va, vw = wide_a[:, at:at + 512], wide_w[:, min(at, 16):min(at, 16) + 512]
        va.copy_(a), vw.copy_(w)
        assert same(gemm(va, vw, sa, sw), ref)
    assert same(gemm(a, w, sa.t().contiguous().t(), sw), ref)
    assert same(gemm(a[3:4], w[:1], sa[3:4], sw[:1]), product64(a[3:4], w[:1], sa[3:4], sw[:1])[0].bfloat16())


def test_product_of_nothing(cuda):
    a, w, sa, sw = exact_operands(4, 130, 256, 1, cuda)
    assert gemm(a[:0], w, sa[:0], sw).shape == (0, 130)
    assert gemm(a, w[:0], sa, sw[:0]).shape == (4, 0)


def test_nan_stays_in_its_row_and_channel(cuda):
    for M, N in ((5, 260), (300, 520)):
        a, w, sa, sw = exact_operands(M, N, 400, 4, cuda)
        ref = product64(a, w, sa, sw)[0].bfloat16()
        a.view(torch.uint8)[M - 1, 399] = 0x7F  # NaN, in the ragged block
        w.view(torch.uint8)[130, 3] = 0x7F
        y = gemm(a, w, sa, sw)
        assert y[M - 1].isnan().all() and y[:, 130].isnan().all()
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[M - 1], keep[:, 130] = False, False
        assert torch.equal(y[keep], ref[keep])


# ---- by experts

def grouped(a, w, sa, sw, offsets, bias=None, dtype=torch.bfloat16, out=None):
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise_grouped
    return f8f8_blockwise_grouped(a, w, bias, sa, sw, offsets, NAMES[dtype], out)


def grouped64(a, w, sa, sw, at, bias=None, fill=None):
    ref = torch.full((a.shape[0], w.shape[1]), 0.0 if fill is None else fill, dtype=torch.float64, device=a.device)
    s = torch.zeros_like(ref)
    for e in range(w.shape[0]):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            ref[lo:hi], s[lo:hi] = product64(a[lo:hi], w[e], sa[lo:hi], sw[e], None if bias is None else bias[e])
    return ref, s


COUNTS = [[1], [0, 1], [5, 0, 0, 11], [1] * 70, [0] * 66 + [3, 0, 64], [16, 17, 0, 1, 33], [64, 65, 63, 128, 0], [257, 1, 130, 300], [700, 2, 0, 41]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("N,K", [(128, 128), (200, 400), (384, 1040)])
def test_grouped_exact(cuda, counts, N, K):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    a, w, sa, sw = exact_operands(at[-1], N, K, sum(counts) + N, cuda, lead=(len(counts),))
    off = torch.tensor(at, dtype=torch.int32, device=cuda)
    ref, _ = grouped64(a, w, sa, sw, at)
    for cfg in [-1, *all_configs()]:
        from llmqrt_amd import _abi
        print("grouped", cfg, counts[:6], N, K, flush=True)
        assert _abi.lib().llmq_gemm_fp8_block_force_plan(cfg, 0) == 0
        try:
            assert same(grouped(a, w, sa, sw, off), ref.bfloat16()), f"configuration {cfg}"
        finally:
            _abi.lib().llmq_gemm_fp8_block_force_plan(-1, 0)


@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_grouped(cuda, bias):
    counts = [40, 0, 3, 129, 1, 77, 300]
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    a, w, sa, sw = general_operands(at[-1], 300, 1168, 7, cuda, lead=(7,))
    b = None if bias is None else torch.randn(7, 300, generator=torch.Generator().manual_seed(1)).to(bias).to(cuda)
    y = grouped(a, w, sa, sw, torch.tensor(at, dtype=torch.int32, device=cuda), b, torch.float16)
    check_general(y, *grouped64(a, w, sa, sw, at, b), 1168)


@pytest.mark.parametrize("at", [[0, 5, 9], [3, 9, 20], [0, 0, 0], [40, 40, 40], [-7, 12, 900], [5, 30, 30]])
def test_rows_of_no_expert_stay(cuda, at):
    """Rows before the first and behind the last offset keep what `out` held; offsets outside the rows are taken as the nearest inside."""
    a, w, sa, sw = exact_operands(40, 140, 256, 3, cuda, lead=(2,))
    held = [min(max(v, 0), 40) for v in at]
    ref, _ = grouped64(a, w, sa, sw, held, fill=7.0)
    out = torch.full((40, 140), 7.0, dtype=torch.bfloat16, device=cuda)
    y = grouped(a, w, sa, sw, torch.tensor(at, dtype=torch.int32, device=cuda), out=out)
    assert y.data_ptr() == out.data_ptr() and torch.equal(out, ref.bfloat16())


def test_grouped_of_nothing(cuda):
    a, w, sa, sw = exact_operands(4, 130, 256, 1, cuda, lead=(2,))
    off = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert grouped(a[:0], w, sa[:0], sw, off).shape == (0, 130)
    out = torch.ones(4, 130, dtype=torch.bfloat16, device=cuda)
    assert grouped(a, w[:0], sa, sw[:0], off[:1], out=out) is out and (out == 1).all()


# ---- streams and graphs

def test_captured_calls_follow_their_inputs(cuda):
    from llmqrt_amd.quantize import per_group_quantize
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
    g = torch.Generator().manual_seed(5)
    x = torch.randn(96, 1024, generator=g).bfloat16().to(cuda)
    _, w, _, sw = general_operands(1, 512, 1024, 5, cuda, lead=(4,))
    off = torch.tensor([0, 20, 20, 50, 96], dtype=torch.int32, device=cuda)

    def run():
        q, s = per_group_quantize(x)
        return f8f8_blockwise(q, w[0].t(), None, s, sw[0]), f8f8_blockwise_grouped(q, w, None, s, sw, off)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = run()
    for k in range(3):
        x.copy_(torch.randn(96, 1024, generator=g).bfloat16())
        off.copy_(torch.tensor([0, 1 + k, 40, 60 + k, 96], dtype=torch.int32))
        graph.replay()
        other = run()  # eager work between the replays
        torch.cuda.synchronize()
        for y, z in zip(ys, other):
            assert torch.equal(y, z)


def test_two_streams_at_once(cuda):
    """Products with a K split share no scratch."""
    cases = [general_operands(70, 256, 8192, s, cuda) for s in (1, 2)]
    want = [gemm(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(gemm(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_captured_split(cuda):
    """A K split inside a graph: its partial sums are the graph's own, beside eager calls of the same size."""
    from llmqrt_amd import _abi
    a, w, sa, sw = general_operands(200, 512, 18944, 3, cuda)
    assert _abi.lib().llmq_gemm_fp8_block_workspace_bytes(200, 512, 18944) > 0
    gemm(a, w, sa, sw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm(a, w, sa, sw)
        z = gemm(a[:150], w, sa[:150], sw)
    for k in range(3):
        sa.mul_(1.25)
        graph.replay()
        y1, z1 = gemm(a, w, sa, sw), gemm(a[:150], w, sa[:150], sw)
        torch.cuda.synchronize()
        assert same(y, y1) and same(z, z1)


# ---- offsets past 32 bits

def test_many_rows(cuda):
    """1.25 million rows: 4.5 GB of codes, whose scales and products start past 2^32 bytes; compared on the last rows, and a block of rows in between."""
    from llmqrt_amd.quantize import per_group_quantize
    M, N, K = 1_250_000, 136, 3600
    x = torch.empty(M, K, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    for part in x.split(100_000):
        part.copy_(torch.randn(part.shape, generator=g, device=cuda))
    q, s = per_group_quantize(x)
    _, w, _, sw = general_operands(1, N, K, 2, cuda)
    y = gemm(q, w, s, sw)
    off = torch.tensor([0, 5, M - 40, M], dtype=torch.int32, device=cuda)
    z = grouped(q, torch.stack([w, w, w]), s, torch.stack([sw, sw, sw]), off)
    for lo, hi in ((M - 300, M), (1_193_000, 1_193_300)):
        qr, sr = groups_ref(x[lo:hi].cpu())
        assert same(s[lo:hi].cpu(), sr) and same(q[lo:hi].cpu().view(torch.uint8), qr.view(torch.uint8))
        ref, r = product64(q[lo:hi], w, s[lo:hi], sw)
        check_general(y[lo:hi], ref, r, K)
        check_general(z[lo:hi], ref, r, K)


def test_many_experts(cuda):
    """600 experts, 4.7 GB of weights: the last ones' lie past 2^32 bytes; more experts than a wavefront counts at once."""
    E, N, K = 600, 2200, 3584
    _, w1, _, sw1 = general_operands(1, N, K, 3, cuda)
    w, sw = torch.zeros(E, N, K, dtype=E4M3, device=cuda), torch.ones(E, blocks(N), blocks(K), device=cuda)
    for e in (0, 299, 598, 599):
        w[e].copy_(w1.view(torch.uint8).roll(e, 0).view(E4M3)), sw[e].copy_(sw1 * (1 + e / E))
    a, _, sa, _ = general_operands(50, 1, K, 4, cuda)
    counts = [0] * E
    counts[0], counts[299], counts[598], counts[599] = 3, 17, 1, 29
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    y = grouped(a, w, sa, sw, torch.tensor(at, dtype=torch.int32, device=cuda))
    for e in (0, 299, 598, 599):
        lo, hi = at[e], at[e + 1]
        check_general(y[lo:hi], *product64(a[lo:hi], w[e], sa[lo:hi], sw[e]), K)


def test_refusals_of_gpu_tensors(cuda):
    from llmqrt_amd.linear import FP8BlockLinear
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
    a, w, sa, sw = exact_operands(4, 130, 384, 1, cuda, lead=(2,))  # scales of [2, 3]: a transposed one shows
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda)
    bad = [dict(x_scale=sa.t().contiguous()), dict(x_scale=sa.half()), dict(x_scale=sa.cpu()), dict(w_scale=sw[0].t().contiguous()), dict(XQ=a.float()), dict(XQ=a[:, :128]),
           dict(WQ=w[0]), dict(bias=torch.zeros(129, device=cuda)), dict(bias=torch.zeros(130, dtype=torch.int32, device=cuda)), dict(dtype_str="float32")]
    for b in bad:
        with pytest.raises(RuntimeError):
            f8f8_blockwise(**{**dict(XQ=a, WQ=w[0].t(), bias=None, x_scale=sa, w_scale=sw[0]), **b})
    bad = [dict(x_scale=sa.t().contiguous()), dict(w_scale=sw[0]), dict(w_scale=sw.transpose(1, 2).contiguous()), dict(WQ=w[:1]), dict(offsets=off[:2]), dict(offsets=off.long()),
           dict(offsets=off.cpu()), dict(bias=torch.zeros(130, device=cuda)), dict(out=torch.zeros(4, 130, dtype=torch.float16, device=cuda)),
           dict(out=torch.zeros(130, 4, dtype=torch.bfloat16, device=cuda).t()), dict(out=torch.zeros(3, 130, dtype=torch.bfloat16, device=cuda))]
    for b in bad:
        with pytest.raises(RuntimeError):
            f8f8_blockwise_grouped(**{**dict(XQ=a, WQ=w, bias=None, x_scale=sa, w_scale=sw, offsets=off), **b})
    m = FP8BlockLinear(384, 130, False)
    for args in ((a, sa.t().contiguous()), (a.float(), sa), (a[:, :128], sa)):
        with pytest.raises(RuntimeError):
            m.forward_quantized(*args)
    for x in (torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda), torch.zeros(2, 384, device=cuda)):
        with pytest.raises(RuntimeError):
            m(x)
