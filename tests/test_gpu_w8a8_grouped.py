"""GPU: the W8A8 product by experts.  The sums are whole numbers that fp32 gets once, and the rest is the documented chain of roundings,
dtype((fp32(acc) * alpha) * beta + bias), so results have to be the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}
CONFIGS = list(range(4, 13))


def same(a, b):
    return bool(torch.equal(a, b))


@pytest.fixture(params=[-1] + CONFIGS)
def force(request):
    from llmqrt_amd import _abi
    _abi.check(_abi.lib().llmq_gemm_w8a8_grouped_force_plan(request.param), "force")
    yield request.param
    _abi.lib().llmq_gemm_w8a8_grouped_force_plan(-1)


def operands(M, E, N, K, dev, seed=0, extreme=False):
    g = torch.Generator().manual_seed(seed + M + N + K)
    lo, hi = (-128, 128)
    q = torch.randint(lo, hi, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(lo, hi, (E, N, K), generator=g, dtype=torch.int8)
    if extreme:
        q[:], w[:] = -128, -128
    alpha = torch.rand(M, 1, generator=g) * 0.02 + 1e-3
    beta = torch.rand(E, N, generator=g) * 0.01 + 1e-3
    return [t.to(dev) for t in (q, w, alpha, beta)]


def offsets_of(counts, dev):
    return torch.tensor([0] + list(counts), dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)


def rows_of(at, M):
    """First rows of the experts and the end of the last: the nearest in [0, M], none below an earlier one."""
    ends = []
    for v in at:
        ends.append(max(min(max(v, 0), M), ends[-1] if ends else 0))
    return ends


def reference(q, w, alpha, beta, bias, offsets, dtype):
    M, N = q.shape[0], w.shape[1]
    out = torch.zeros(M, N, dtype=dtype, device=q.device)
    at = rows_of(offsets.tolist(), M)
    for e in range(w.shape[0]):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            acc = (q[lo:hi].double() @ w[e].double().t()).float()  # exact in 64 bits, then rounded as an int32 is
            y = (acc * alpha[lo:hi]) * beta[e]
            out[lo:hi] = (y if bias is None else y + bias[e].float()).to(dtype)
    return out


def product(q, w, alpha, beta, bias, offsets, dtype=torch.bfloat16, out=None):
    from llmqrt_amd.sq_fp8_kernels import w8a8_int8_linear_per_channel_grouped
    return w8a8_int8_linear_per_channel_grouped(q, w, bias, alpha, beta, offsets, NAMES[dtype], out)


COUNTS = [[1], [0, 3, 0, 1], [5, 64, 33, 0, 129], [300, 1, 0, 257, 31], [0, 0, 600], [2] * 70]


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 144), (257, 272), (640, 640), (96, 3584), (512, 400), (100, 1040), (264, 112)])
@pytest.mark.parametrize("counts", COUNTS, ids=[str(sum(c)) + "x" + str(len(c)) for c in COUNTS])
def test_product(cuda, force, counts, N, K):
    q, w, alpha, beta = operands(sum(counts), len(counts), N, K, cuda)
    off = offsets_of(counts, cuda)
    dtype = torch.float16 if N % 2 else torch.bfloat16
    bias = torch.randn(len(counts), N, generator=torch.Generator().manual_seed(N)).to(cuda)
    bias = bias if K % 32 else bias.to(dtype)
    for b in (None, bias):
        assert same(product(q, w, alpha, beta, b, off, dtype), reference(q, w, alpha, beta, b, off, dtype))


@pytest.mark.parametrize("counts,N,K", [([700, 0, 1, 1300], 1152, 896), ([1000, 998], 3584, 1536), ([4] * 64, 2048, 2048), ([1500, 600, 0, 900], 2432, 18944)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_larger(cuda, counts, N, K, dtype):
    q, w, alpha, beta = operands(sum(counts), len(counts), N, K, cuda)
    off = offsets_of(counts, cuda)
    alpha *= 0.05
    assert same(product(q, w, alpha, beta, None, off, dtype), reference(q, w, alpha, beta, None, off, dtype))


def test_extreme_sums(cuda, force):
    """All products 16384, at the longest K that int32 sums take."""
    K = (1 << 17) - 16
    q, w, alpha, beta = operands(40, 2, 72, K, cuda, extreme=True)
    off = offsets_of([7, 33], cuda)
    alpha *= 1e-6
    assert same(product(q, w, alpha, beta, None, off), reference(q, w, alpha, beta, None, off, torch.bfloat16))


def test_rows_of_no_expert(cuda, force):
    """Rows outside every expert keep what `out` holds, its neighbours too; offsets that are no rows are taken as the nearest, those below an earlier one
    as that."""
    M, E, N, K = 200, 4, 136, 256
    q, w, alpha, beta = operands(M, E, N, K, cuda)
    for at in ([10, 40, 40, 150, 190], [-5, 20, 300, 100, 400], [50, 20, 90, 80, 120], [200, 200, 200, 200, 200], [0, 0, 0, 0, 0], [-9, -3, 5, 2 ** 31 - 1, -2 ** 31]):
        off = torch.tensor(at, dtype=torch.int32, device=cuda)
        for width in (N, N - 3):
            room = torch.full((M + 2, width), 7.0, dtype=torch.bfloat16, device=cuda)
            out = room[1:-1]
            ww, bb = w[:, :width].contiguous(), beta[:, :width].contiguous()
            want = torch.where(owned(at, M)[:, None].to(cuda), reference(q, ww, alpha, bb, None, off, torch.bfloat16), out)
            assert product(q, ww, alpha, bb, None, off, out=out) is out
            assert same(out, want) and (room[0] == 7).all() and (room[-1] == 7).all()


def owned(at, M):
    ends, has = rows_of(at, M), torch.zeros(M, dtype=torch.bool)
    has[ends[0]:ends[-1]] = True
    return has


def test_layouts_and_refusals(cuda):
    q, w, alpha, beta = operands(50, 3, 72, 128, cuda)
    off = offsets_of([20, 0, 30], cuda)
    want = product(q, w, alpha, beta, None, off)
    wide = torch.zeros(50, 256, dtype=torch.int8, device=cuda)
    wide[:, 16:144] = q
    odd = torch.zeros(50 * 128 + 1, dtype=torch.int8, device=cuda)[1:].view(50, 128)
    odd.copy_(q)
    for a in (wide[:, 16:144], odd, q.t().contiguous().t()):
        assert same(product(a, w, alpha, beta, None, off), want)
    assert same(product(q, w.permute(2, 0, 1).contiguous().permute(1, 2, 0), alpha, beta, None, off), want)
    assert same(product(q, w, alpha.view(-1), beta.t().contiguous().t(), None, off), want)
    assert same(product(q, w, alpha.double(), beta, None, torch.stack([off, off], 1)[:, 0]), want)
    assert product(q[:0], w, alpha[:0], beta, None, off).shape == (0, 72) and product(q, w[:, :0], alpha, beta[:, :0], None, off).shape == (50, 0)
    dt = torch.bfloat16
    for bad in (lambda: product(q.cpu(), w, alpha, beta, None, off), lambda: product(q, w.cpu(), alpha, beta, None, off), lambda: product(q.float(), w, alpha, beta, None, off),
                lambda: product(q, w.float(), alpha, beta, None, off), lambda: product(q, w[..., :112], alpha, beta, None, off),
                lambda: product(q[:, :120], w[..., :120], alpha, beta, None, off), lambda: product(q, w, alpha[:49], beta, None, off),
                lambda: product(q, w, alpha.view(1, 50), beta, None, off), lambda: product(q, w, alpha, beta[:2], None, off), lambda: product(q, w, alpha, beta.view(-1), None, off),
                lambda: product(q, w, alpha, beta.int(), None, off), lambda: product(q, w, alpha, beta, beta[0], off), lambda: product(q, w, alpha, beta, beta.double(), off),
                lambda: product(q, w, alpha, beta, None, off.long()), lambda: product(q, w, alpha, beta, None, off[:3]), lambda: product(q, w, alpha, beta, None, off.cpu()),
                lambda: product(q, w, alpha, beta, None, off, out=torch.empty(50, 72, device=cuda)), lambda: product(q, w, alpha, beta, None, off, out=torch.empty(49, 72, dtype=dt, device=cuda)),
                lambda: product(q, w, alpha, beta, None, off, out=torch.empty(50, 144, dtype=dt, device=cuda)[:, :72])):
        with pytest.raises(RuntimeError):
            bad()


def test_autograd_sees_out(cuda):
    q, w, alpha, beta = operands(6, 2, 64, 64, cuda)
    off = offsets_of([2, 4], cuda)
    want = product(q, w, alpha, beta, None, off)
    for a in (alpha, alpha.double()):  # the native path and the general one
        out = torch.ones(6, 64, dtype=torch.bfloat16, device=cuda)
        scale = torch.ones(6, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        saved = (scale * out).float().sum()
        assert same(product(q, w, a, beta, None, off, out=out), want) and out._version > 0
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
        leaf = torch.ones(6, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        with pytest.raises(RuntimeError, match="requires grad"):
            product(q, w, a, beta, None, off, out=leaf)
        assert (leaf == 1).all()
        with torch.no_grad():
            product(q, w, a, beta, None, off, out=leaf)
        assert same(leaf, want) and leaf._version > 0
