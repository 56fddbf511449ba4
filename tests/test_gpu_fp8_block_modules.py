"""GPU: the block-scaled FP8 modules, and the operators in a run: residual norm -> projections -> experts -> next residual norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def same(a, b):
    return bool(torch.equal(a, b))


def linear(k, n, bias, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(k, n, bias=bias)
    lin.weight.data = 0.02 * torch.randn(n, k, generator=g)
    if bias:
        lin.bias.data = torch.randn(n, generator=g)
    return lin.to(dtype).cuda()


def dequantized(w, s):
    n, k = w.shape[-2:]
    return w.double() * s.double().repeat_interleave(128, -1)[..., :k].repeat_interleave(128, -2)[..., :n, :]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N,bias", [(1, 896, 1152, True), (7, 3584, 200, False), (33, 400, 896, True), (300, 1040, 384, False)])
def test_module(cuda, M, K, N, bias, dtype):
    """The module is the quantizer and the product; against the unquantized Linear it is off by the two operands' e4m3 steps: every product by at most
    (1 + 2^-4)^2 - 1 < 2^-2.9 of its absolute value (2^-10 of the largest of the block below the normal range, far less here), so every output by
    that share of the sum of absolute products."""
    from llmqrt_amd.linear import FP8BlockLinear
    from llmqrt_amd.quantize import per_group_quantize
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise
    ref = linear(K, N, bias, K + N, dtype)
    m = FP8BlockLinear.from_linear(ref, init_only=False, dtype=dtype)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype).cuda()
    y = m(x)
    q, s = per_group_quantize(x)
    assert y.dtype == dtype and same(y, f8f8_blockwise(q, m.weight.t(), m.bias, s, m.weight_scale, {torch.bfloat16: "bfloat16", torch.float16: "float16"}[dtype]))
    assert same(m.forward_quantized(q, s), y)
    want = x.double() @ ref.weight.double().t() + (0 if ref.bias is None else ref.bias.double())
    room = 2.0 ** -2.9 * (x.double().abs() @ ref.weight.double().abs().t()) + torch.finfo(dtype).eps * want.abs() + 1e-3
    assert ((y.double() - want).abs() <= room).all()
    # other shapes of the same rows, and rows that are not contiguous
    assert same(m(x.view(1, M, K))[0], y) and same(m(torch.cat([x, x], 1)[:, :K]), y)
    assert m(x[:0]).shape == (0, N)


def test_outputs_of_one_call_are_apart(cuda):
    """Small outputs of a call share an allocation: writing one changes no other, and each counts its own versions."""
    from llmqrt_amd.norm import add_rmsnorm_per_group_quantize
    from llmqrt_amd.quantize import per_group_quantize
    x = torch.randn(3, 904).bfloat16().cuda()
    w = torch.ones(904, dtype=torch.bfloat16, device=cuda)
    for f in (lambda: add_rmsnorm_per_group_quantize(x, x, w, return_normed=True), lambda: per_group_quantize(x)):
        outs, ref = f(), f()
        assert all(t.data_ptr() % 256 == 0 and t.is_contiguous() and t._base is None for t in outs)
        for i, t in enumerate(outs):
            t.view(torch.uint8).fill_(255)
            assert t._version == 1 and all(same(a.view(torch.uint8), b.view(torch.uint8)) for a, b in list(zip(outs, ref))[i + 1:])
    with torch.inference_mode():
        q, s, y, h = add_rmsnorm_per_group_quantize(x, x, w, return_normed=True)
        assert h.is_inference() and same(h, x + x)
    h = add_rmsnorm_per_group_quantize(x, x, w)[-1]
    h.requires_grad_(True)
    (h.float() * 2).sum().backward()
    assert bool((h.grad == 2).all())


def test_module_moves_and_converts(cuda):
    from llmqrt_amd.linear import FP8BlockLinear
    m = FP8BlockLinear.from_linear(linear(256, 384, True, 1), init_only=False)
    x = torch.randn(5, 256).bfloat16().cuda()
    y = m(x)
    w, s = m.weight.clone(), m.weight_scale.clone()
    m = m.cpu().half().cuda()
    assert m.weight.dtype == E4M3 and m.weight_scale.dtype == torch.float32 and m.bias.dtype == torch.float16 and m.dtype == torch.float16
    assert same(m.weight.view(torch.uint8), w.view(torch.uint8)) and same(m.weight_scale, s)
    z = m(x.half())
    assert z.dtype == torch.float16 and torch.allclose(z.float(), y.float(), rtol=2 ** -6, atol=2 ** -6)


@pytest.mark.parametrize("sizes", [(256, 128, 128), (128, 384, 72)])
@pytest.mark.parametrize("bias", [True, False])
def test_fused_siblings(cuda, sizes, bias):
    """Exact inputs: the fused module has the separate ones' outputs whatever order its sizes give the sums."""
    from llmqrt_amd.fused_utils import fuse_linears
    from llmqrt_amd.linear import FP8BlockLinear
    g = torch.Generator().manual_seed(4)
    parts = []
    for n in sizes:
        m = FP8BlockLinear(512, n, bias, dev="cuda:0")
        m.weight.copy_(torch.randint(-2, 3, (n, 512), generator=g).float().to(E4M3))
        m.weight_scale.copy_(torch.pow(2.0, torch.randint(-1, 2, m.weight_scale.shape, generator=g).float()))
        if bias:
            m.bias.copy_(torch.randint(-4, 5, (n,), generator=g).float())
        parts.append(m)
    f = fuse_linears(parts)
    q = torch.randint(-3, 4, (9, 512), generator=g).float().to(E4M3).cuda()
    s = torch.ones(9, 4, device=cuda)
    assert same(f.forward_quantized(q, s), torch.cat([m.forward_quantized(q, s) for m in parts], -1))


def test_siblings_whose_blocks_straddle_stay_apart(cuda):
    from llmqrt_amd.fused_utils import fuse_linears
    from llmqrt_amd.linear import FP8BlockLinear
    parts = [FP8BlockLinear(128, n, False) for n in (72, 128)]
    assert fuse_linears(parts) == parts


def test_grouped_module(cuda):
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    from llmqrt_amd.quantize import per_group_quantize
    mods = [linear(400, 264, True, e) for e in range(5)]
    m = FP8BlockGroupedLinear.from_linears(mods)
    x = torch.randn(90, 400, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    at = [0, 20, 20, 61, 62, 90]
    off = torch.tensor(at, dtype=torch.int32, device=cuda)
    y = m(x, off)
    q, s = per_group_quantize(x)
    assert same(m.forward_quantized(q, s, off), y)
    a = q.double() * s.double().repeat_interleave(128, -1)[:, :400]
    for e in range(5):
        lo, hi = at[e], at[e + 1]
        w = dequantized(m.weight[e], m.weight_scale[e])
        want = a[lo:hi] @ w.t() + m.bias[e].double()
        # bf16's half step; 7 products of a run of 8 cut by 2^-14 of the largest each; 400 sums, 4 blocks (as in test_gpu_fp8_block.py)
        room = 2.0 ** -8 * want.abs() + (7 * 2.0 ** -14 + 2.0 ** -23 * 420) * (a[lo:hi].abs() @ w.abs().t() + m.bias[e].double().abs()) + 1e-30
        assert ((y[lo:hi].double() - want).abs() <= room * (1 + 1e-6)).all()
        one = FP8BlockLinear.from_linear(mods[e], init_only=False)
        assert same(one.weight.view(torch.uint8), m.weight[e].view(torch.uint8)) and same(one.weight_scale, m.weight_scale[e])
    strided = torch.cat([x, x], 1)[:, :400]
    assert same(m(strided, off), y)
    out = torch.full((90, 264), 3.0, dtype=torch.bfloat16, device=cuda)
    short = torch.tensor([0, 20, 20, 61, 62, 70], dtype=torch.int32, device=cuda)
    assert same(m(x, short, out)[:70], y[:70]) and (out[70:] == 3).all()


@pytest.mark.parametrize("tokens", [1, 19, 260])
def test_a_layer_of_experts(cuda, tokens):
    """residual norm -> gate_up of the experts of each token -> activation -> down -> weighted sum -> next residual norm, against the same run with
    every operator in plain fp32 torch.  The plain run quantizes the same values, but its own sums: codes next to a border may differ, by a step of 2^-3
    at most, in what is then a sum of hundreds; the norm of the difference stays under 2^-5 of the norm of the result (each of the two quantized
    tensors and of the three roundings to bf16 adds less than 2^-8 rms where a tenth of the codes differed)."""
    from llmqrt_amd.linear import FP8BlockGroupedLinear
    from llmqrt_amd.norm import RMSNorm
    g = torch.Generator().manual_seed(tokens)
    E, H, F, top = 8, 896, 640, 2
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, r = rnd(tokens, H).bfloat16().cuda(), (2 * rnd(tokens, H)).bfloat16().cuda()
    norm = RMSNorm((1 + 0.1 * rnd(H)).bfloat16().cuda())
    up, down = FP8BlockGroupedLinear(E, H, 2 * F, dev="cuda:0"), FP8BlockGroupedLinear(E, F, H, dev="cuda:0")
    up.set_weight(0.03 * rnd(E, 2 * F, H))
    down.set_weight(0.03 * rnd(E, F, H).transpose(1, 2).contiguous())
    gate = rnd(tokens, E).cuda()
    weight, expert = gate.softmax(-1).topk(top, -1)
    order = expert.view(-1).argsort(stable=True)
    token = order // top
    offsets = torch.cat([torch.zeros(1, device=cuda), torch.bincount(expert.view(-1), minlength=E).cumsum(0)]).to(torch.int32)

    q, s, h = norm.forward_add(x, r, quantize="fp8_block")
    ab = up.forward_quantized(q[token], s[token], offsets)
    a, b = ab.chunk(2, -1)
    y = down((torch.nn.functional.silu(a.float()) * b.float()).bfloat16(), offsets)
    mixed = torch.zeros(tokens, H, device=cuda).index_add_(0, token, y.float() * weight.view(-1)[order][:, None]).bfloat16()
    q2, s2, h2 = norm.forward_add(mixed, h, quantize="fp8_block")

    def groups(t):
        full = torch.nn.functional.pad(t, (0, -t.shape[1] % 128)).view(t.shape[0], -1, 128)
        sc = full.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 448
        return ((full / sc).to(E4M3).float() * sc).view(t.shape[0], -1)[:, :t.shape[1]]

    def plain_norm(t):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + norm.variance_epsilon) * norm.weight.float()
    hp = x + r
    ap = groups(plain_norm(hp.float()))[token]
    wu, wd = dequantized(up.weight, up.weight_scale).float(), dequantized(down.weight, down.weight_scale).float()
    of = expert.view(-1)[order]
    abp = torch.stack([wu[e] @ v for e, v in zip(of, ap)]).bfloat16()
    act = (torch.nn.functional.silu(abp[:, :F].float()) * abp[:, F:].float()).bfloat16()
    yp = torch.stack([wd[e] @ v for e, v in zip(of, groups(act.float()))]).bfloat16()
    mp = torch.zeros(tokens, H, device=cuda).index_add_(0, token, yp.float() * weight.view(-1)[order][:, None]).bfloat16()
    assert same(h, hp)
    assert (mixed.float() - mp.float()).norm() <= 2.0 ** -5 * mp.float().norm()
    assert same(h2, mixed + h)
    assert (q2.float() * s2.repeat_interleave(128, 1) - groups(plain_norm((mp + hp).float()))).norm() <= 2.0 ** -4 * (q2.float() * s2.repeat_interleave(128, 1)).norm()


def test_checkpoint(cuda, tmp_path):
    from safetensors.torch import save_file
    from llmqrt_amd.checkpoint import QuantConfig, load_quantized_weights, named_quantized_linears, replace_linears
    from llmqrt_amd.linear import FP8BlockLinear
    src = torch.nn.ModuleDict({"up": linear(256, 200, True, 1), "lm_head": linear(256, 64, False, 2)})
    made = FP8BlockLinear.from_linear(src["up"], init_only=False)
    save_file({f"up.{k}": v.cpu() for k, v in made.state_dict().items()}, str(tmp_path / "model.safetensors"))
    cfg = QuantConfig(quant_method="fp8_dynamic_quant", q_group_size=128)
    assert replace_linears(src, cfg) == ["up"] and isinstance(src["up"], FP8BlockLinear) and [n for n, _ in named_quantized_linears(src)] == ["up"]
    missing, unexpected = load_quantized_weights(src, str(tmp_path))
    assert unexpected == [] and missing == ["lm_head.weight"]
    x = torch.randn(3, 256).bfloat16().cuda()
    assert same(src["up"](x), made(x))
