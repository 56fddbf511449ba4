"""GPU: the operators around products by experts past 32-bit offsets and past what one launch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room(cuda):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of GPU memory")
    yield
    torch.cuda.empty_cache()


def as_bytes(t):
    return t.contiguous().view(torch.uint8)


def same(a, b):
    return bool(torch.equal(as_bytes(a), as_bytes(b)))


def halves(*size, dev, seed=0):
    """16-bit values of any size from the generator of the device."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(-999, 1000, size, generator=g, device=dev, dtype=torch.int16).to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["same", "int8", "group"])
@pytest.mark.parametrize("T,K,top", [(150001, 7168, 2), ((1 << 21) + 5, 8, 2), ((1 << 20) + 3, 24, 1)])
def test_dispatch(cuda, T, K, top, kind):
    from llmqrt_amd import experts
    from llmqrt_amd.quantize import per_group_quantize, quantize_activation_per_token_absmax_f32
    f = {"same": experts.dispatch_to_experts, "int8": experts.dispatch_quantize_activation_per_token_absmax, "group": experts.dispatch_per_group_quantize}[kind]
    E = 5
    x = halves(T, K, dev=cuda)
    ids = torch.randint(0, E, (T, top), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda, dtype=torch.int32)
    got = f(x, ids, E)
    flat = ids.reshape(-1).long()
    order = torch.sort(flat, stable=True)[1]
    places = torch.empty_like(order).scatter_(0, order, torch.arange(T * top, device=cuda)).view(T, top)
    assert torch.equal(got[-1].long(), places)
    assert torch.equal(got[-2].long(), torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=E).cumsum(0)]))
    step = (1 << 28) // K
    for r in range(0, T * top, step):
        part = x[order[r:r + step] // top]
        rows = (part,) if kind == "same" else quantize_activation_per_token_absmax_f32(part) if kind == "int8" else per_group_quantize(part)
        assert all(same(g[r:r + step], w) for g, w in zip(got, rows))


@pytest.mark.parametrize("T,N,R", [(330000, 7168, 330000), ((1 << 20) + 77, 16392, 5003)])
def test_combine(cuda, T, N, R):
    """Rows and outputs of more than 2^31 elements; and more chunks of an output than a launch takes."""
    from llmqrt_amd.experts import combine_from_experts
    y = halves(R, N, dev=cuda)
    at = torch.arange(T, device=cuda) % R
    out = combine_from_experts(y, at.to(torch.int32).view(T, 1), torch.ones(T, 1, device=cuda))
    step = (1 << 28) // N
    for t in range(0, T, step):
        assert same(out[t:t + step], y[at[t:t + step]])


@pytest.mark.parametrize("kind,M,N", [("same", (1 << 27) + 5, 8), ("group", (1 << 27) + 5, 8), ("int8", (1 << 21) + 3, 8), ("fp8", (1 << 21) + 3, 16), ("int8", 60000, 18944),
                                      ("group", 60000, 18944)])
def test_silu(cuda, kind, M, N):
    from llmqrt_amd import activation as A
    f = {"same": A.silu_mul, "int8": A.silu_mul_quantize_activation_per_token_absmax, "fp8": A.silu_mul_per_token_quantize, "group": A.silu_mul_per_group_quantize}[kind]
    x = halves(M, 2 * N, dev=cuda)
    x *= 2.0 ** -7
    got = f(x)
    got = (got,) if kind == "same" else got
    step = max((1 << 27) // N, 1)
    for m in [*range(0, M - 100, M // 7), M - 100]:
        want = f(x[m:m + 100].clone())
        assert all(same(g[m:m + 100], w) for g, w in zip(got, (want,) if kind == "same" else want))
    del got
    if kind == "same":  # all of them
        y = f(x)
        for m in range(0, M, step):
            assert same(y[m:m + step], f(x[m:m + step].clone()))


@pytest.mark.parametrize("bias", [False, True])
def test_route(cuda, bias):
    from llmqrt_amd.experts import route_to_experts
    T, E = (1 << 24) + 3, 4
    x = halves(T, E, dev=cuda)
    x *= 2.0 ** -6
    x += torch.tensor([0.0, 0.25, 0.5, 0.75], device=cuda, dtype=x.dtype)
    b = torch.zeros(E, device=cuda) if bias else None
    w, ids = route_to_experts(x, 1, scoring="sigmoid", bias=b, renormalize=True)
    # ties to the lowest expert
    best = x.amax(1, keepdim=True)
    if not bias:
        assert torch.equal(ids, (x == best).int().argmax(1, keepdim=True).int())
    else:  # sigmoids can be level in 64 bits where logits are not: nothing is larger by more than that
        chosen = torch.gather(x, 1, ids.long()).double()
        assert (torch.sigmoid(best.double()) - torch.sigmoid(chosen) <= 2.0 ** -52).all()
    assert (w == 1).all()


@pytest.mark.parametrize("cfg", [-1, *range(4, 13)])
@pytest.mark.parametrize("counts,N,K,lda", [([20000, 1, 0, 13001], 65560, 16, 16), ([2, 0, 3, 1] * 18, 65544, 512, 512), ([100, 70, 0, 130], 24, 48, 1 << 23)])
def test_product(cuda, counts, N, K, lda, cfg):
    """Outputs, weights and rows of activations past 2^31."""
    from llmqrt_amd import _abi
    from llmqrt_amd.sq_fp8_kernels import w8a8_int8_linear_per_channel_grouped
    E, M = len(counts), sum(counts)
    g = torch.Generator(device=cuda).manual_seed(2)
    w = torch.randint(-128, 128, (E, N, K), generator=g, device=cuda, dtype=torch.int8)
    q = torch.empty(M, lda, dtype=torch.int8, device=cuda)[:, :K]
    q.copy_(torch.randint(-128, 128, (M, K), generator=g, device=cuda, dtype=torch.int8))
    alpha, beta = torch.rand(M, 1, generator=g, device=cuda) + 0.5, torch.rand(E, N, generator=g, device=cuda) + 0.5
    offsets = torch.tensor([0, *counts], device=cuda).cumsum(0).to(torch.int32)
    _abi.check(_abi.lib().llmq_gemm_w8a8_grouped_force_plan(cfg), "force")
    try:
        out = w8a8_int8_linear_per_channel_grouped(q, w, None, alpha, beta, offsets, "bfloat16")
    finally:
        _abi.lib().llmq_gemm_w8a8_grouped_force_plan(-1)
    at = offsets.tolist()
    for e in range(E):
        for r in sorted({at[e], (at[e] + at[e + 1]) // 2, at[e + 1] - 1}) if at[e + 1] > at[e] else ():
            acc = (w[e].double() @ q[r].double()).float()  # whole numbers: exact
            assert same(out[r], ((acc * alpha[r]) * beta[e]).to(torch.bfloat16))
