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


def norm_calls():
    from llmqrt_amd import norm as N
    return [N.add_rmsnorm, N.add_rmsnorm_quantize_activation_per_token_absmax, N.add_rmsnorm_per_token_quantize, N.add_rmsnorm_per_group_quantize]


@pytest.mark.parametrize("strided", [False, True])
def test_autograd_sees_a_residual_written_in_place(cuda, strided):
    """Both the native path (contiguous rows) and the general one (rows inside a wider tensor)."""
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)).bfloat16().to(cuda)
    w = torch.ones(256, dtype=torch.bfloat16, device=cuda)
    for f in norm_calls():
        room = torch.zeros(5, 512 if strided else 256, dtype=torch.bfloat16, device=cuda)
        r = room[:, :256]
        r.fill_(2)
        before = r._version
        scale = torch.ones(5, 256, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        saved = (scale * r).float().sum()  # keeps r for its backward pass
        f(x, r, w)
        assert r._version == before
        f(x, r, w, inplace=True)
        assert r._version > before and room._version == r._version and same(r, x + 2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
        # one that requires grad: left as it is, and written under no_grad
        leaf = torch.full((5, 512 if strided else 256), 2.0, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        for t in (leaf, leaf * 1):
            with pytest.raises(RuntimeError, match="requires grad"):
                f(x, t[:, :256] if strided else t, w, inplace=True)
            assert (t == 2).all()
        with torch.no_grad():
            part = leaf[:, :256] if strided else leaf
            before = leaf._version
            f(x, part, w, inplace=True)
            assert leaf._version > before and same(part, x + 2)
        with torch.inference_mode():
            made = torch.full((5, 512 if strided else 256), 2.0, dtype=torch.bfloat16, device=cuda)
            part = made[:, :256]
            assert f(x, part, w, inplace=True)[-1].data_ptr() == made.data_ptr() and same(part, x + 2)
        with pytest.raises(RuntimeError, match="inference"):
            f(x, part, w, inplace=True)


def test_autograd_sees_out_of_a_product_by_experts(cuda):
    from llmqrt_amd.linear import FP8BlockGroupedLinear
    from llmqrt_amd.quantize import per_group_quantize
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise_grouped
    g = torch.Generator().manual_seed(4)
    m = FP8BlockGroupedLinear(2, 256, 200, dev=cuda)
    m.set_weight(torch.randn(2, 200, 256, generator=g))
    x = torch.randn(6, 256, generator=g).bfloat16().to(cuda)
    wide = torch.cat([x, x], 1)[:, :256]  # rows inside a wider tensor: the general path
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device=cuda)
    q, s = per_group_quantize(x)
    calls = [lambda o: m(x, off, o), lambda o: m(wide, off, o), lambda o: m.forward_quantized(q, s, off, o),
             lambda o: f8f8_blockwise_grouped(q, m.weight, None, s.t().contiguous().t(), m.weight_scale, off, out=o)]
    want = m(x, off)
    for call in calls:
        out = torch.ones(6, 200, dtype=torch.bfloat16, device=cuda)
        scale = torch.ones(6, 200, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        saved = (scale * out).float().sum()
        assert call(out) is out or same(out, want)
        assert same(out, want) and out._version > 0
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
        leaf = torch.ones(6, 200, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        with pytest.raises(RuntimeError, match="requires grad"):
            call(leaf)
        assert (leaf == 1).all()
        with torch.no_grad():
            call(leaf)
        assert same(leaf, want) and leaf._version > 0


def test_a_residual_over_part_of_the_activations(cuda):
    """Refused in place, and left as it was; halves of the same rows, neighbours, and the activations themselves are fine, and so is any overlap otherwise."""
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda)
    buf = torch.randn(12, 128, generator=torch.Generator().manual_seed(5)).bfloat16().to(cuda)
    flat = buf.view(24, 64)
    bad = [(flat[1:9], flat[0:8]), (flat[0:8], flat[1:9]), (buf[1:9, :64], buf[0:8, :64]), (buf[:8, :64], buf[:8, 8:72]), (flat[:5], buf[:5, :64]),
           (buf.view(-1)[:64], buf.view(-1)[8:72])]
    for f in norm_calls():
        for x, r in bad:
            was = buf.clone()
            want = f(x.clone(), r.clone(), w)
            assert all(same(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(f(x, r, w), want))
            with pytest.raises(RuntimeError, match="apart"):
                f(x, r, w, inplace=True)
            assert same(buf, was)
        for x, r in ((flat[:8], flat[8:16]), (buf[:, :64], buf[:, 64:]), (buf[:, 64:], buf[:, :64]), (flat[:8], flat[:8]), (buf[:, :64], buf[:, :64])):
            was = buf.clone()
            want = f(x.clone(), r.clone(), w)
            got = f(x, r, w, inplace=True)
            assert got[-1].data_ptr() == r.data_ptr() and all(same(a.contiguous().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
            buf.copy_(was)


@pytest.mark.parametrize("wide", [False, True])
def test_scales_in_the_tokens_order(cuda, wide):
    """Scales with the dimensions of the codes, or one row per token; other dimensions of as many scales are refused.  Contiguous codes (the native path) and
    codes inside a wider tensor."""
    from llmqrt_amd.linear import FP8BlockLinear
    from llmqrt_amd.quantize import per_group_quantize
    g = torch.Generator().manual_seed(6)
    m = FP8BlockLinear(256, 72, False, dev=cuda)
    m.set_weight(torch.randn(72, 256, generator=g))
    x = torch.randn(2, 3, 256, generator=g).bfloat16().to(cuda)
    q, s = per_group_quantize(x)
    want = m(x)
    if wide:
        room = torch.zeros(2, 3, 512, dtype=torch.uint8, device=cuda)
        room[..., :256] = q.view(torch.uint8)
        q = room.view(E4M3)[..., :256]
    assert same(m.forward_quantized(q, s), want) and same(m.forward_quantized(q, s.view(6, 2)), want)
    for bad in (s.transpose(0, 1).contiguous(), s.view(3, 2, 2), s.view(1, 6, 2), s.view(1, 2, 3, 2), s.view(12), s.view(4, 3), s.view(6, 2)[:5]):
        with pytest.raises(RuntimeError):
            m.forward_quantized(q, bad)


def test_threads(cuda):
    """Four threads with a stream each, every one with its own sizes (split products among them): what each gets alone."""
    import threading
    from llmqrt_amd.norm import add_rmsnorm_per_group_quantize
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
    g = torch.Generator().manual_seed(7)
    cases = []
    for rows, n, k in ((1, 640, 896), (70, 256, 8192), (200, 512, 4096), (17, 1000, 400)):
        x, r = [torch.randn(rows, k, generator=g).bfloat16().to(cuda) for _ in range(2)]
        w = (torch.randn(2, n, k, generator=g) * 90).clamp(-448, 448).to(E4M3).to(cuda)
        sw = (torch.rand(2, -(-n // 128), -(-k // 128), generator=g) * 1e-3).to(cuda)
        off = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=cuda)
        cases.append((x, r, torch.ones(k, dtype=torch.bfloat16, device=cuda), w, sw, off))

    def run(x, r, weight, w, sw, off):
        q, s, h = add_rmsnorm_per_group_quantize(x, r, weight)
        return q.view(torch.uint8), s, h, f8f8_blockwise(q, w[0].t(), None, s, sw[0]), f8f8_blockwise_grouped(q, w, None, s, sw, off)
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = run(*cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(same(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


def test_a_captured_residual_in_place(cuda):
    """Each replay adds the activations to the residual as it then is, beside eager calls on another one."""
    for f in norm_calls():
        x = torch.ones(6, 256, dtype=torch.bfloat16, device=cuda)
        w = torch.ones(256, dtype=torch.bfloat16, device=cuda)
        r, other = torch.zeros_like(x), torch.zeros_like(x)
        f(x, r, w, inplace=True)
        r.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = f(x, r, w, inplace=True)
        for k in range(1, 4):
            graph.replay()
            eager = f(x, other, w, inplace=True)
            torch.cuda.synchronize()
            assert (r == k).all() and all(same(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs, eager))
