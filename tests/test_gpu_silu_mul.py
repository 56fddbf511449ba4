"""GPU: silu(gate) * up, as it is and in 8 bits, against the formula in 64 bits.

y is off by at most u (2 |g| + 8) |y|, u = 2^-24: exp takes 2 u |g| from its argument (the constant and the product, each off by u) and 2 u of its own, the sum
u, the reciprocal 2 u, the two products u each.  Below -88 exp(-g) is infinite and y is 0 instead of less than 1e-35 u.  Outputs add a rounding: eps / 2 of the value, or half a
step of the codes; scales carry the error of the largest value and two roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KINDS = ["same", "int8", "fp8", "group"]
SIZES = [(1, 8), (1, 3584), (3, 136), (37, 18944), (300, 896), (256, 1024), (255, 1024), (5, 2056), (399, 4096), (400, 4104), (401, 8192), (9, 24576), (7, 24584), (1030, 2432), (2100, 264), (9, 1024), (260, 1032), (17, 256), (300, 248), (9, 264), (31, 512), (2, 16384), (300, 16392), (3, 32768), (5, 32776)]


def call(kind, x):
    from llmqrt_amd import activation as A
    return {"same": A.silu_mul, "int8": A.silu_mul_quantize_activation_per_token_absmax, "fp8": A.silu_mul_per_token_quantize, "group": A.silu_mul_per_group_quantize}[kind](x)


def exact(x):
    g, u = x.double().chunk(2, dim=-1)
    y = g * torch.sigmoid(g) * u
    return y, U * (2 * g.abs() + 8) * y.abs() + 1e-35 * u.abs()


def check(kind, x):
    got = call(kind, x)
    y, off = exact(x)
    if kind == "same":
        assert got.dtype == x.dtype and got.shape == y.shape
        bound = torch.finfo(x.dtype).eps / 2 * y.abs() + off * 1.01 + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)
        assert ((got.double() - y).abs() <= bound).all()
        return
    q, s = got
    N = y.shape[-1]
    assert q.shape == y.shape and q.dtype == (torch.int8 if kind == "int8" else torch.float8_e4m3fn) and s.dtype == torch.float32
    most, floor = (127, 1e-5) if kind == "int8" else (448, 1e-12)
    if kind == "group":
        n = (N + 127) // 128
        pad = lambda t: torch.nn.functional.pad(t, (0, n * 128 - N)).view(*t.shape[:-1], n, 128)  # noqa: E731
        y, off, q = pad(y), pad(off), pad(q.double())
    else:
        n = 1
        y, off, q = y[..., None, :], off[..., None, :], q.double()[..., None, :]
    assert s.shape == (*x.shape[:-1], n)
    s = s.double()[..., None]
    top = y.abs().amax(-1, keepdim=True).clamp_min(floor)
    slack = off.amax(-1, keepdim=True) * 1.01
    assert ((s - top / most).abs() <= slack / most + 3 * U * s).all()
    v = y / s  # what is rounded, off by what y is; a code of the largest value may be past the range by that much
    half = 0.5 if kind == "int8" else torch.maximum(v.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64, device=v.device))
    assert ((q - v).abs() <= half * (1 + 1e-5) + off * 1.01 / s + 4 * U * v.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N", SIZES)
def test_silu_mul(cuda, M, N, kind, dtype):
    g = torch.Generator().manual_seed(M + N)
    x = torch.randn(M, 2 * N, generator=g) * 2
    x[:, :N] *= torch.where(torch.rand(N, generator=g) < 0.02, 12.0, 1.0)
    x[0, : N // 2] = 0
    check(kind, x.to(dtype).to(cuda))


@pytest.mark.parametrize("kind", KINDS)
def test_far_gates(cuda, kind):
    """Gates far out on both sides, rows of zeros, tiny rows."""
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.ones(6, 512, dtype=torch.float64)
        x[0, :256] = torch.linspace(-120, 120, 256)
        x[1, :256] = -90.0
        x[2] = 0
        x[3, :256], x[3, 256:] = 1e-3, 1e-3
        x[4, :256] = torch.linspace(-3e4, 3e4, 256)
        x[5, 256:] = -1e4
        check(kind, x.to(dtype).to(cuda))


@pytest.mark.parametrize("kind", KINDS)
def test_layouts(cuda, kind):
    big = torch.randn(40, 2048, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    for view in (big[:, :1008], big[:, 8:648], big[::3, 128:1152], big[:, 3:1011], big[:, ::2], big[7:8, :144], big.view(4, 10, 2048), big[3], big[:1, :512].expand(9, 512)):
        check(kind, view)
    empty = call(kind, big[:0])
    assert (empty if kind == "same" else empty[0]).shape == (0, 1024)
    for bad in (big[:, :24], big.float(), big.cpu()):
        with pytest.raises(RuntimeError):
            call(kind, bad)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N", [(6, 512), (300, 512), (9, 4096)])
def test_not_finite(cuda, M, N, kind):
    """An infinity or a NaN stays in its row (in its group, in its element): the others have the same bits."""
    x = torch.randn(M, 2 * N, generator=torch.Generator().manual_seed(2)).bfloat16().to(cuda)
    want = call(kind, x)
    bad = x.clone()
    bad[1, 130], bad[2, N + 5], bad[4, N - 1] = float("nan"), float("inf"), float("-inf")
    got = call(kind, bad)
    keep = [m for m in range(M) if m not in (1, 2, 4)]
    for a, b in zip((want,) if kind == "same" else want, (got,) if kind == "same" else got):
        assert torch.equal(a[keep].contiguous().view(torch.uint8), b[keep].contiguous().view(torch.uint8))
    if kind == "same":
        assert got[1, 130].isnan() and got[4, N - 1].isnan() and got[2, 5].isinf() and int((~got.isfinite()).sum()) == 3
    else:
        group = kind == "group"
        assert got[1][1, 1 if group else 0].isnan() and got[1][2, 0].isinf() and got[1][4, -1].isnan()
        assert int((~got[1].isfinite()).sum()) == 3


def test_many_rows(cuda):
    """Offsets past 32 bits of bytes and elements: the last rows are those of a call of their own."""
    M, N = 140000, 16384  # 2 M N elements: 4.6e9
    x = torch.empty(M, 2 * N, dtype=torch.bfloat16, device=cuda)
    x[:-8] = 0
    x[-8:] = torch.randn(8, 2 * N, generator=torch.Generator().manual_seed(3)).bfloat16().to(cuda)
    for kind in KINDS:
        got, want = call(kind, x), call(kind, x[-8:].clone())
        for a, b in zip((got,) if kind == "same" else got, (want,) if kind == "same" else want):
            assert torch.equal(a[-8:].contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        del got
