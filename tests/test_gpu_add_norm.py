"""GPU: the residual's addition + RMSNorm with an output in 16 or 8 bits, against the formula in 64 bits.

h is the same bits as torch's (x + residual).  The sum of squares is a chain of at most 8 x 10 FMAs per thread (rows of more than 20480: one per
chunk a thread visits) and at most 6 + 16 additions across threads, each off by u = 2^-24 relative to a sum of positive terms; halved by the root, with the
roundings of mean, eps, root, reciprocal and the two products: y is within Y_RTOL.  Codes may be off by half a step of their type (2^-4
of the value or 2^-10, the smallest step's half, for e4m3; 1/2 for int8) and by what y and the scale are off."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24
SHAPES = [(1, 8), (3, 120), (1, 896), (333, 896), (256, 1024), (300, 136), (5, 1032), (1, 3584), (32, 3584), (400, 3584), (9, 4104), (450, 8192), (7, 8200),
          (3, 18944), (2, 20488), (3, 40960)]


def y_rtol(k):
    chain = 8 * max(10, -(-k // (8 * 512))) + 22
    return (chain / 2 + 7) * U


def inputs(M, K, dtype, seed):
    from llmqrt_amd import workloads as W
    x = W.activations(M, K, seed, dtype=dtype)
    r = (2 * W.activations(M, K, seed + 1, dtype=torch.float32)).to(dtype)
    if M > 2:
        x[2], r[2] = 0, 0  # a row of zeros
    w = (1.0 + 0.2 * torch.randn(K, generator=torch.Generator().manual_seed(seed + 2))).to(dtype)
    return x, r, w


def norm64(h, w, eps):
    f = h.double()
    return f / torch.sqrt(f.square().mean(-1, keepdim=True) + eps) * w.double()


def grouped_amax(y):
    M, K = y.shape
    g = (K + 127) // 128
    return torch.nn.functional.pad(y.abs(), (0, g * 128 - K)).view(M, g, 128).amax(-1)


def check_codes(q, s, y, kind):
    K = y.shape[1]
    rt = y_rtol(K)
    if kind == "group":
        sr = grouped_amax(y).clamp_min(1e-12) / 448
        full = s.double().repeat_interleave(128, 1)[:, :K]
    else:
        sr = y.abs().amax(1, keepdim=True).clamp_min(1e-5 if kind == "int8" else 1e-12) / (127 if kind == "int8" else 448)
        full = s.double()
    assert s.dtype == torch.float32 and s.shape == sr.shape
    assert ((s.double() - sr).abs() <= (rt + 2 * U) * sr).all()
    v = y / full
    q64 = q.float().double()
    step = 0.5 if kind == "int8" else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10))
    err = (q64 - v).abs()
    assert (err <= step * (1 + 1e-5) + (rt + 4 * U) * v.abs() + 1e-30).all()


def fn(kind):
    from llmqrt_amd import norm
    return {"int8": norm.add_rmsnorm_quantize_activation_per_token_absmax, "fp8": norm.add_rmsnorm_per_token_quantize,
            "group": norm.add_rmsnorm_per_group_quantize}[kind]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_add_rmsnorm(cuda, M, K, dtype):
    from llmqrt_amd.norm import add_rmsnorm
    x, r, w = inputs(M, K, dtype, M + K)
    y, h = add_rmsnorm(x.to(cuda), r.to(cuda), w.to(cuda), 1e-6)
    href = x + r
    assert torch.equal(h.cpu(), href) and h.dtype == dtype and y.dtype == dtype and y.shape == x.shape
    ref = norm64(href, w, 1e-6)
    err = (y.cpu().double() - ref).abs()
    half = torch.finfo(dtype).eps / 2
    assert (err <= (half * (1 + 1e-4) + y_rtol(K)) * ref.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("kind", ["int8", "fp8", "group"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_add_rmsnorm_quantized(cuda, M, K, dtype, kind):
    x, r, w = inputs(M, K, dtype, 3 * M + K)
    args = x.to(cuda), r.to(cuda), w.to(cuda), 1e-5
    q, s, h = fn(kind)(*args)
    assert torch.equal(h.cpu(), x + r) and q.dtype == (torch.int8 if kind == "int8" else E4M3) and q.shape == x.shape
    y = norm64(x + r, w, 1e-5)
    check_codes(q.cpu(), s.cpu(), y, kind)
    # with the normalised row as well: the same codes, and the row of the form that does not quantize
    from llmqrt_amd.norm import add_rmsnorm
    q2, s2, y2, h2 = fn(kind)(*args, return_normed=True)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s) and torch.equal(h2, h)
    assert torch.equal(y2, add_rmsnorm(*args)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_rmsnorm_per_group(cuda, M, K, dtype):
    from llmqrt_amd.norm import add_rmsnorm_per_group_quantize, rmsnorm_per_group_quantize
    x, r, w = inputs(M, K, dtype, 5 * M + K)
    h = x + r
    q, s = rmsnorm_per_group_quantize(h.to(cuda), w.to(cuda))
    check_codes(q.cpu(), s.cpu(), norm64(h, w, 1e-6), "group")
    q2, s2, _ = add_rmsnorm_per_group_quantize(x.to(cuda), r.to(cuda), w.to(cuda))
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


@pytest.mark.parametrize("M,K", [(7, 3584), (300, 896), (3, 24576)])
def test_in_place_and_strides(cuda, M, K):
    from llmqrt_amd.norm import add_rmsnorm, add_rmsnorm_per_group_quantize
    x, r, w = (t.to(cuda) for t in inputs(M, K, torch.bfloat16, 77))
    y, h = add_rmsnorm(x, r, w)
    res = r.clone()
    y2, h2 = add_rmsnorm(x, res, w, inplace=True)
    assert h2 is res or h2.data_ptr() == res.data_ptr()
    assert torch.equal(res, h) and torch.equal(y2, y)
    # rows inside wider tensors, each with its own stride; the columns beside them stay
    wide_x, wide_r = torch.zeros(M, K + 24, dtype=x.dtype, device=cuda), torch.full((M, K + 64), 3.0, dtype=x.dtype, device=cuda)
    wide_x[:, 8:K + 8], wide_r[:, 16:K + 16] = x, r
    y3, h3 = add_rmsnorm(wide_x[:, 8:K + 8], wide_r[:, 16:K + 16], w, inplace=True)
    assert torch.equal(y3, y) and torch.equal(wide_r[:, 16:K + 16], h) and (wide_r[:, :16] == 3).all() and (wide_r[:, K + 16:] == 3).all()
    wide_r[:, 16:K + 16] = r
    q, s, h4 = add_rmsnorm_per_group_quantize(wide_x[:, 8:K + 8], wide_r[:, 16:K + 16], w)
    q5, s5, _ = add_rmsnorm_per_group_quantize(x, r, w)
    assert torch.equal(h4, h) and torch.equal(q.view(torch.uint8), q5.view(torch.uint8)) and torch.equal(s, s5) and torch.equal(wide_r[:, 16:K + 16], r)
    # an unaligned residual is copied, and refused where it would have to be written
    odd = torch.zeros(M, K + 8, dtype=x.dtype, device=cuda)[:, 3:K + 3]
    odd.copy_(r)
    assert torch.equal(add_rmsnorm(x, odd, w)[1], h)
    with pytest.raises(RuntimeError):
        add_rmsnorm(x, odd, w, inplace=True)
    assert torch.equal(odd, r)


@pytest.mark.parametrize("kind", ["int8", "fp8", "group"])
@pytest.mark.parametrize("M,K", [(7, 3584), (300, 896), (3, 24576)])
def test_a_nan_or_infinity_stays_in_its_row(cuda, M, K, kind):
    x, r, w = (t.to(cuda) for t in inputs(M, K, torch.bfloat16, 13))
    want = fn(kind)(x, r, w)
    x[1, 9] = float("nan")
    x[0, K - 1] = float("inf")
    q, s, h = fn(kind)(x, r, w)
    rest = torch.arange(M, device=cuda) > 1
    assert torch.equal(q[rest].view(torch.uint8), want[0][rest].view(torch.uint8)) and torch.equal(s[rest], want[1][rest])
    assert s[1].isnan().all() and h[1, 9].isnan() and h[0, K - 1].isinf()
    if kind == "int8":
        assert (q[1] == 0).all()
    else:
        assert q[1].float().isnan().all()
    # an infinite square: inv is 0, every finite element becomes 0 and the infinite one NaN
    other = torch.ones(K, dtype=torch.bool, device=cuda)
    other[(K - 1) // 128 * 128 if kind == "group" else 0:] = False
    if kind == "group":
        assert (q[0][other].float() == 0).all()
    assert s[0, -1].isnan()


def test_captured(cuda):
    from llmqrt_amd.norm import add_rmsnorm, add_rmsnorm_quantize_activation_per_token_absmax
    x, r, w = (t.to(cuda) for t in inputs(40, 3584, torch.bfloat16, 5))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        add_rmsnorm(x, r, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = add_rmsnorm(x, r, w)
        q, s, h2 = add_rmsnorm_quantize_activation_per_token_absmax(y, h, w)
    for k in range(3):
        x.normal_()
        graph.replay()
        y1, h1 = add_rmsnorm(x, r, w)
        q1, s1, h3 = add_rmsnorm_quantize_activation_per_token_absmax(y1, h1, w)
        torch.cuda.synchronize()
        assert torch.equal(y, y1) and torch.equal(h, h1) and torch.equal(q, q1) and torch.equal(s, s1) and torch.equal(h2, h3)


def test_no_rows_one_row_and_more_dimensions(cuda):
    from llmqrt_amd.norm import RMSNorm, add_rmsnorm, add_rmsnorm_per_group_quantize
    x, r, w = (t.to(cuda) for t in inputs(12, 904, torch.float16, 3))
    y, h = add_rmsnorm(x[:0], r[:0], w)
    assert y.shape == h.shape == (0, 904)
    q, s, h = add_rmsnorm_per_group_quantize(x[:0], r[:0], w)
    assert q.shape == (0, 904) and s.shape == (0, 8)
    want = add_rmsnorm(x, r, w)
    one = add_rmsnorm(x[5], r[5], w)
    assert all(torch.equal(a, b[5]) for a, b in zip(one, want))
    cube = add_rmsnorm_per_group_quantize(x.view(3, 4, 904), r.view(3, 4, 904), w)
    flat = add_rmsnorm_per_group_quantize(x, r, w)
    assert cube[1].shape == (3, 4, 8) and all(torch.equal(a.view(torch.uint8).flatten(), b.view(torch.uint8).flatten()) for a, b in zip(cube, flat))
    m = RMSNorm(w, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(m.forward_add(x, r), want))
    # the same row for every token, and x as its own residual
    assert torch.equal(add_rmsnorm(x, r[:1].expand(12, 904), w)[1], x + r[:1])
    with pytest.raises(RuntimeError):
        add_rmsnorm(x, r[:1].expand(12, 904), w, inplace=True)
    twice = x.clone()
    y2, h2 = add_rmsnorm(twice, twice, w, inplace=True)
    y3, h3 = add_rmsnorm(x, x, w)
    assert torch.equal(y2, y3) and torch.equal(twice, h3)


def test_many_rows(cuda):
    """2.2 million short rows: more than one grid's, and offsets past 2^32 bytes."""
    from llmqrt_amd.norm import add_rmsnorm_quantize_activation_per_token_absmax as f
    M, K = 2_200_000, 1032
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.empty(M, K, dtype=torch.bfloat16, device=cuda)
    for part in x.split(200_000):
        part.copy_(torch.randn(part.shape, generator=g, device=cuda))
    r = x.flip(0)
    w = torch.ones(K, dtype=torch.bfloat16, device=cuda)
    q, s, h = f(x, r, w)
    for rows in (slice(0, 50), slice(2_097_100, 2_097_200), slice(M - 50, M)):
        q1, s1, h1 = f(x[rows].contiguous(), r[rows].contiguous(), w)
        href = x[rows] + r[rows]
        assert torch.equal(h[rows], href) and torch.equal(h1, href)
        check_codes(q[rows].cpu(), s[rows].cpu(), norm64(href.cpu(), w.cpu(), 1e-6), "int8")
        check_codes(q1.cpu(), s1.cpu(), norm64(href.cpu(), w.cpu(), 1e-6), "int8")
