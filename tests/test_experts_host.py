"""CPU-only checks of the operators around products by experts: argument validation of the C entries before any HIP call, and refusals of the Python ones."""
import ctypes

import pytest
import torch

from llmqrt_amd import _abi

OK, NULL, DTYPE, SHAPE, WORKSPACE, ALIGN = 0, -1, -2, -3, -4, -6


@pytest.fixture(scope="module")
def p16():
    buf = ctypes.create_string_buffer(4096)
    p16.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def route(p, scoring=0, dt=2, T=4, E=16, ld=16, bias=0, G=1, tg=1, gs=0, k=2, logits=None, w=None, ids=None):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_route_experts(scoring, d(logits), dt, T, E, ld, bias, G, tg, gs, k, 1, 1.0, d(w), d(ids), None)


def test_route_refusals(p16):
    p = p16
    assert route(p, scoring=2) == DTYPE and route(p, scoring=-1) == DTYPE and route(p, dt=3) == DTYPE and route(p, gs=2) == DTYPE
    assert route(p, T=-1) == SHAPE and route(p, E=0, ld=0) == SHAPE and route(p, E=1025, ld=1025) == SHAPE and route(p, ld=15) == SHAPE
    assert route(p, k=0) == SHAPE and route(p, k=17) == SHAPE and route(p, E=128, ld=128, k=65) == SHAPE
    assert route(p, G=0) == SHAPE and route(p, G=3) == SHAPE and route(p, G=4, tg=5) == SHAPE and route(p, G=4, tg=0) == SHAPE
    assert route(p, G=4, tg=1, k=5) == SHAPE and route(p, E=256, ld=256, G=128) == SHAPE and route(p, T=1 << 31, k=2) == SHAPE
    assert route(p, logits=0) == NULL and route(p, w=0) == NULL and route(p, ids=0) == NULL
    assert route(p, T=0, logits=0, w=0, ids=0) == OK


def dispatch(p, out=0, dt=0, T=4, K=64, ldx=64, k=2, first=0, E=4, x=None, ids=None, rows=None, scale=None, off=None, pl=None, ws=None, wsb=0):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_dispatch_experts(out, d(x), dt, T, K, ldx, d(ids), k, first, E, d(rows), d(scale), d(off), d(pl), ws, wsb, None)


def test_dispatch_refusals(p16):
    p = p16
    assert dispatch(p, out=2) == DTYPE and dispatch(p, out=4) == DTYPE and dispatch(p, dt=2) == DTYPE
    assert dispatch(p, T=-1) == SHAPE and dispatch(p, K=60) == SHAPE and dispatch(p, ldx=56) == SHAPE and dispatch(p, ldx=68) == SHAPE
    assert dispatch(p, k=0) == SHAPE and dispatch(p, k=65) == SHAPE and dispatch(p, E=0) == SHAPE and dispatch(p, E=4097) == SHAPE
    assert dispatch(p, first=-1) == SHAPE and dispatch(p, first=0x7fffffff) == SHAPE and dispatch(p, T=1 << 31) == SHAPE and dispatch(p, K=0, ldx=0) == SHAPE
    for name in ("x", "ids", "rows", "off", "pl"):
        assert dispatch(p, **{name: 0}) == NULL
    assert dispatch(p, out=1, scale=0) == NULL and dispatch(p, out=3, scale=0) == NULL and dispatch(p, T=0, off=0) == NULL
    need = _abi.lib().llmq_dispatch_experts_workspace_bytes
    assert need(48, 4, 64) == 0 and need(4000, 4, 64) == 0 and need(0, 4, 64) == 0 and need(-1, 4, 64) == 0 and need(1 << 62, 64, 4096) == 0 and need(9, 9, 5000) == 0
    many = need(50000, 2, 12)
    assert many >= 12 * 4 * 2 and 0 < need((1 << 31) // 64 - 1024, 64, 4096) <= 4096 * 4 * 1025
    assert dispatch(p, T=50000, E=12) == WORKSPACE and dispatch(p, T=50000, E=12, ws=p, wsb=many - 1) == WORKSPACE and dispatch(p, T=50000, E=12, ws=p + 4, wsb=many) == ALIGN
    assert dispatch(p, x=p + 8) == ALIGN and dispatch(p, rows=p + 8) == ALIGN and dispatch(p, out=1, rows=p + 4) == ALIGN


def combine(p, dt=0, R=8, N=64, ldy=64, T=4, k=2, sh=0, lds=64, y=None, pl=None, w=None, out=None):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_combine_experts(d(y), dt, R, N, ldy, d(pl), d(w), T, k, sh, lds, d(out), None)


def test_combine_refusals(p16):
    p = p16
    assert combine(p, dt=2) == DTYPE
    assert combine(p, R=-1) == SHAPE and combine(p, T=-1) == SHAPE and combine(p, N=60) == SHAPE and combine(p, ldy=56) == SHAPE and combine(p, ldy=68) == SHAPE
    assert combine(p, k=0) == SHAPE and combine(p, k=65) == SHAPE and combine(p, T=1 << 31) == SHAPE
    assert combine(p, sh=p, lds=56) == SHAPE and combine(p, sh=p, lds=68) == SHAPE
    assert combine(p, y=0) == NULL and combine(p, pl=0) == NULL and combine(p, w=0) == NULL and combine(p, out=0) == NULL
    assert combine(p, y=p + 8) == ALIGN and combine(p, out=p + 8) == ALIGN and combine(p, sh=p + 8) == ALIGN
    assert combine(p, T=0) == OK and combine(p, N=0, ldy=0) == OK


def grouped(p, lda=64, E=2, bias=0, bdt=0, dt=0, ldo=8, M=4, N=8, K=64, A=None, sa=None, B=None, sw=None, off=None, out=None):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_gemm_w8a8_grouped(d(A), lda, d(sa), d(B), d(sw), d(off), E, bias, bdt, d(out), dt, ldo, M, N, K, None)


def test_product_refusals(p16):
    p = p16
    assert grouped(p, dt=2) == DTYPE and grouped(p, bias=p, bdt=3) == DTYPE
    assert grouped(p, E=-1) == SHAPE and grouped(p, E=65537) == SHAPE and grouped(p, M=-1) == SHAPE and grouped(p, N=-1) == SHAPE and grouped(p, K=-16) == SHAPE
    assert grouped(p, K=72, lda=80) == SHAPE and grouped(p, lda=48) == SHAPE and grouped(p, lda=72) == SHAPE and grouped(p, ldo=7) == SHAPE
    assert grouped(p, K=1 << 17, lda=1 << 17) == SHAPE and grouped(p, lda=(1 << 23) + 16) == SHAPE and grouped(p, K=0) == SHAPE
    assert grouped(p, M=0x7fffff01) == SHAPE
    for name in ("A", "sa", "B", "sw", "off", "out"):
        assert grouped(p, **{name: 0}) == NULL
    assert grouped(p, A=p + 8) == ALIGN and grouped(p, B=p + 8) == ALIGN
    assert grouped(p, M=0) == OK and grouped(p, N=0, ldo=0) == OK and grouped(p, E=0) == OK
    L = _abi.lib()
    assert L.llmq_gemm_w8a8_grouped_force_plan(3) == SHAPE and L.llmq_gemm_w8a8_grouped_force_plan(13) == SHAPE
    assert L.llmq_gemm_w8a8_grouped_force_plan(-1) == OK


def silu(p, out=0, dt=0, M=4, N=32, ldx=64, x=None, y=None, s=None):
    d = lambda v: p if v is None else v  # noqa: E731
    return _abi.lib().llmq_silu_mul(out, d(x), dt, M, N, ldx, d(y), d(s), None)


def test_silu_refusals(p16):
    p = p16
    assert silu(p, out=4) == DTYPE and silu(p, out=-1) == DTYPE and silu(p, dt=2) == DTYPE
    assert silu(p, N=36, ldx=72) == SHAPE and silu(p, ldx=56) == SHAPE and silu(p, ldx=68) == SHAPE and silu(p, M=-1) == SHAPE
    assert silu(p, x=0) == NULL and silu(p, y=0) == NULL and silu(p, out=1, s=0) == NULL
    assert silu(p, x=p + 8) == ALIGN and silu(p, y=p + 8) == ALIGN and silu(p, out=1, y=p + 4) == ALIGN
    assert silu(p, M=0) == OK and silu(p, N=0, ldx=0) == OK


def test_ops_refuse_wrong_tensors():
    from llmqrt_amd import activation, experts
    from llmqrt_amd.sq_fp8_kernels import w8a8_int8_linear_per_channel_grouped
    x, ids = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32)
    calls = [lambda: experts.route_to_experts(x, 2), lambda: experts.route_to_experts(x, 2, scoring="tanh"), lambda: experts.route_to_experts(x, 2, group_score="sum"),
             lambda: experts.route_to_experts([1.0], 1), lambda: experts.dispatch_to_experts(x, ids, 4), lambda: experts.dispatch_to_experts(x, ids, 0),
             lambda: experts.dispatch_to_experts(x, ids, 4097), lambda: experts.dispatch_to_experts(x, ids, 4, -1),
             lambda: experts.dispatch_to_experts(x, ids[:3], 4), lambda: experts.dispatch_to_experts(x, ids.float(), 4),
             lambda: experts.dispatch_to_experts(x, ids[:, :0], 4), lambda: experts.dispatch_per_group_quantize(x[:, :60], ids, 4),
             lambda: experts.combine_from_experts(x, ids, ids.float()), lambda: activation.silu_mul(x), lambda: activation.silu_mul(x[:, :24]),
             lambda: w8a8_int8_linear_per_channel_grouped(x, x, None, x, x, ids)]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i}")
