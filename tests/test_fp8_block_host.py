"""CPU-only checks of the block-scaled fp8 operators: argument validation of the C entries before any HIP call, refusals of the Python ones, the weight
quantizer, and the modules' interfaces."""
import ctypes

import pytest
import torch

from llmqrt_amd import _abi

E4M3 = torch.float8_e4m3fn
OK, NULL, DTYPE, SHAPE, WORKSPACE, ALIGN = 0, -1, -2, -3, -4, -6


@pytest.fixture(scope="module")
def p16():
    buf = ctypes.create_string_buffer(4096)
    p16.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def quant(p, dt=0, M=4, K=64, ldx=64, q=None, s=None, x=None):
    return _abi.lib().llmq_quant_fp8_per_group(p if x is None else x, dt, M, K, ldx, p if q is None else q, p if s is None else s, None)


def test_group_quantizer_refusals(p16):
    assert quant(p16, dt=2) == DTYPE
    assert quant(p16, K=60) == SHAPE and quant(p16, ldx=56) == SHAPE and quant(p16, ldx=68) == SHAPE and quant(p16, M=-1) == SHAPE
    assert quant(p16, x=0) == NULL and quant(p16, q=0) == NULL and quant(p16, s=0) == NULL
    assert quant(p16, x=p16 + 8) == ALIGN and quant(p16, q=p16 + 4) == ALIGN
    assert quant(p16, M=0) == OK and quant(p16, K=0, ldx=0) == OK


def norm(p, out=0, dt=0, M=4, K=64, ldx=64, res=0, ldr=64, h=0, ldh=64, w=None, y=None, q=None, s=None, x=None):
    return _abi.lib().llmq_add_rmsnorm(out, p if x is None else x, dt, M, K, ldx, res, ldr, h, ldh, p if w is None else w, 1e-6, p if y is None else y,
                                       p if q is None else q, p if s is None else s, None)


def test_norm_refusals(p16):
    p = p16
    assert norm(p, out=4) == DTYPE and norm(p, out=-1) == DTYPE and norm(p, dt=2) == DTYPE
    assert norm(p, K=60) == SHAPE and norm(p, ldx=56) == SHAPE and norm(p, M=-1) == SHAPE and norm(p, K=0, ldx=0) == SHAPE
    assert norm(p, res=p, h=p, ldr=56) == SHAPE and norm(p, res=p, h=p, ldh=68) == SHAPE
    assert norm(p, x=0) == NULL and norm(p, w=0) == NULL and norm(p, res=p) == NULL and norm(p, y=0) == NULL
    for out in (1, 2, 3):
        assert norm(p, out=out, q=0) == NULL and norm(p, out=out, s=0) == NULL and norm(p, out=out, q=p + 4) == ALIGN
    assert norm(p, x=p + 8) == ALIGN and norm(p, w=p + 8) == ALIGN and norm(p, y=p + 8) == ALIGN and norm(p, res=p + 8, h=p) == ALIGN and norm(p, res=p, h=p + 8) == ALIGN
    assert norm(p, M=0) == OK


def gemm(p, lda=64, ldb=64, ldo=8, M=4, N=8, K=64, dt=0, bias=None, bdt=0, A=None, sa=None, B=None, sw=None, out=None, ws=0, wsb=0):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_gemm_fp8_block(d(A), lda, d(sa), d(B), ldb, d(sw), bias, bdt, d(out), dt, ldo, M, N, K, ws, wsb, None)


def grouped(p, off=None, E=2, lda=64, ldo=8, M=4, N=8, K=64, dt=0, bias=None, bdt=0, A=None, sa=None, B=None, sw=None, out=None):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_gemm_fp8_block_grouped(d(A), lda, d(sa), d(B), d(sw), d(off), E, bias, bdt, d(out), dt, ldo, M, N, K, None)


@pytest.mark.parametrize("call", [gemm, grouped])
def test_product_refusals(p16, call):
    p = p16
    assert call(p, dt=2) == DTYPE and call(p, bias=p, bdt=3) == DTYPE
    assert call(p, K=72, lda=80) == SHAPE and call(p, lda=48) == SHAPE and call(p, lda=72) == SHAPE and call(p, ldo=4) == SHAPE
    assert call(p, M=-1) == SHAPE and call(p, N=-1) == SHAPE and call(p, K=0) == SHAPE and call(p, lda=1 << 24) == SHAPE
    for name in ("A", "sa", "B", "sw", "out"):
        assert call(p, **{name: 0}) == NULL
    assert call(p, A=p + 8) == ALIGN and call(p, B=p + 8) == ALIGN
    assert call(p, M=0) == OK and call(p, N=0, ldo=0) == OK


def test_product_workspace_and_experts(p16):
    L = _abi.lib()
    assert gemm(p16, ldb=48) == SHAPE and gemm(p16, ldb=72) == SHAPE
    assert grouped(p16, off=0) == NULL and grouped(p16, E=-1) == SHAPE and grouped(p16, E=65537) == SHAPE and grouped(p16, E=0) == OK
    M, N, K = 300, 512, 18944  # a few tiles over a long K: split
    need = L.llmq_gemm_fp8_block_workspace_bytes(M, N, K)
    assert need > 0 and need % (M * N * 4) == 0
    assert gemm(p16, lda=K, ldb=K, ldo=N, M=M, N=N, K=K) == WORKSPACE
    assert gemm(p16, lda=K, ldb=K, ldo=N, M=M, N=N, K=K, ws=p16, wsb=need - 1) == WORKSPACE
    assert gemm(p16, lda=K, ldb=K, ldo=N, M=M, N=N, K=K, ws=p16 + 4, wsb=need) == ALIGN
    assert L.llmq_gemm_fp8_block_workspace_bytes(8192, 37888, 3584) == 0 and L.llmq_gemm_fp8_block_workspace_bytes(1, 3584, 3584) == 0
    for sizes in ((0, 1, 16), (1, 0, 16), (1, 1, 0), (-1, 5, 5), (2 ** 62, 2 ** 62, 2 ** 62), (0x7fffff00, 0x7fffff00, 1 << 23)):
        assert L.llmq_gemm_fp8_block_workspace_bytes(*sizes) >= 0  # answers for any sizes


def test_tuning_hook_refuses(p16):
    f = _abi.lib().llmq_gemm_fp8_block_force_plan
    assert f(0, -1) == SHAPE and f(1000, 0) == SHAPE and f(0, 1) == OK and f(-1, 0) == OK


def test_ops_refuse_wrong_tensors():
    from llmqrt_amd import norm as N
    from llmqrt_amd.quantize import per_group_quantize
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        per_group_quantize(x)  # not on the GPU
    with pytest.raises(RuntimeError):
        per_group_quantize(x.float())
    for f in (N.add_rmsnorm, N.add_rmsnorm_quantize_activation_per_token_absmax, N.add_rmsnorm_per_token_quantize, N.add_rmsnorm_per_group_quantize):
        with pytest.raises(RuntimeError):
            f(x, None, w)
        with pytest.raises(RuntimeError):
            f(x, x, w)
    with pytest.raises(RuntimeError):
        N.rmsnorm_per_group_quantize(x, w)
    norm = N.RMSNorm(w)
    with pytest.raises(RuntimeError):
        norm.forward_add(x, None)
    with pytest.raises(RuntimeError):
        norm.forward_add(x, x, quantize="fp4")
    q, s = torch.zeros(4, 64, dtype=E4M3), torch.ones(4, 1)
    wq, ws = torch.zeros(8, 64, dtype=E4M3), torch.ones(1, 1)
    for bad in (dict(dtype_str="float32"), dict()):  # the second: right but on the CPU
        with pytest.raises(RuntimeError):
            f8f8_blockwise(q, wq.t(), None, s, ws, **bad)
        with pytest.raises(RuntimeError):
            f8f8_blockwise_grouped(q, wq[None], None, s, ws[None], torch.zeros(2, dtype=torch.int32), **bad)


def test_weight_quantizer():
    from llmqrt_amd.quantize import quantize_weight_per_block
    g = torch.Generator().manual_seed(1)
    w = torch.randn(2, 300, 200, generator=g)
    w[0, :128, :128] = 0
    w[1, 256:, 128:] *= 1000
    q, s = quantize_weight_per_block(w)
    assert q.shape == w.shape and q.dtype == E4M3 and s.shape == (2, 3, 2) and s.dtype == torch.float32
    for e in range(2):
        for i in range(3):
            for j in range(2):
                b = w[e, 128 * i:128 * (i + 1), 128 * j:128 * (j + 1)]
                sc = b.abs().max().clamp_min(1e-12) / 448.0
                assert s[e, i, j] == sc
                assert torch.equal(q[e, 128 * i:128 * (i + 1), 128 * j:128 * (j + 1)].float(), (b / sc).to(E4M3).float())
    for bad in (torch.zeros(5), torch.zeros(4, 4, dtype=torch.int8)):
        with pytest.raises(RuntimeError):
            quantize_weight_per_block(bad)


def test_module_interfaces():
    from llmqrt_amd.checkpoint import QuantConfig, named_quantized_linears, replace_linears
    from llmqrt_amd.linear import FP8BlockGroupedLinear, FP8BlockLinear
    lin = torch.nn.Linear(48, 200, bias=True)
    m = FP8BlockLinear.from_linear(lin, init_only=False)
    assert {k: (tuple(v.shape), v.dtype) for k, v in m.state_dict().items()} == {
        "weight": ((200, 48), E4M3), "weight_scale": ((2, 1), torch.float32), "bias": ((200,), torch.bfloat16)}
    deq = m.weight.float() * m.weight_scale.repeat_interleave(128, 0)[:200].repeat_interleave(48, 1)
    # half a step of e4m3: 2^-4 of the value, or half of the smallest step, 2^-10, of the scale
    bound = 2.0 ** -4 * lin.weight.abs() + 2.0 ** -10 * m.weight_scale.max()
    assert ((deq - lin.weight).abs() <= bound * (1 + 1e-5)).all()
    h = m.half()
    assert h.weight.dtype == E4M3 and h.weight_scale.dtype == torch.float32 and h.bias.dtype == torch.float16 and h.dtype == torch.float16
    for bad in (dict(w_bit=4), dict(group_size=64)):
        with pytest.raises(RuntimeError):
            FP8BlockLinear.from_linear(lin, **bad)
    with pytest.raises(RuntimeError):
        FP8BlockLinear(40, 8, False, dev="cpu")
    with pytest.raises(RuntimeError):
        FP8BlockLinear(48, 8, False, dev="cpu", dtype=torch.float32)
    e = FP8BlockGroupedLinear.from_linears([torch.nn.Linear(48, 200, bias=False) for _ in range(3)])
    assert tuple(e.weight.shape) == (3, 200, 48) and tuple(e.weight_scale.shape) == (3, 2, 1) and e.bias is None
    with pytest.raises(RuntimeError):
        FP8BlockGroupedLinear.from_linears([torch.nn.Linear(48, 200), torch.nn.Linear(48, 100)])
    with pytest.raises(RuntimeError):
        e.set_weight(torch.zeros(3, 200, 32))
    model = torch.nn.Sequential(torch.nn.Linear(32, 16), torch.nn.Linear(16, 16))
    assert replace_linears(model, QuantConfig(quant_method="fp8_dynamic_quant", q_group_size=128)) == ["0", "1"]
    assert [n for n, _ in named_quantized_linears(model)] == ["0", "1"] and isinstance(model[0], FP8BlockLinear)
    with pytest.raises(RuntimeError):
        model[0](torch.zeros(2, 32, dtype=torch.bfloat16))  # on the CPU: refused
