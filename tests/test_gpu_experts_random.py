"""GPU: the operators around products by experts at sizes drawn at random, each in the variant that it chooses itself, on a stream that is not the default one;
and at the most experts."""
import random

import pytest
import torch

from test_gpu_experts import check_combine, check_dispatch, check_route, choose
from test_gpu_silu_mul import KINDS, check as check_silu
from test_gpu_w8a8_grouped import offsets_of, operands, product, reference, same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_a_stream(cuda):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        yield
    side.synchronize()


def log_uniform(r, lo, hi):
    return int(round(2 ** r.uniform(*[torch.tensor(float(v)).log2().item() for v in (lo, hi)])))


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("seed", range(60))
def test_route(cuda, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    groups = r.choice([1, 1, 2, 4, 8, 16, 20])
    E = groups * max(1, log_uniform(r, 4, 260) // groups)
    top_groups = r.randint(1, groups)
    top = r.randint(1, min(E // groups * top_groups, r.choice([4, 8, 16, 30])))
    T = log_uniform(r, 1, 250) if seed % 6 else 3300
    x = (torch.randn(T, E, generator=g) * r.choice([0.5, 2, 6])).to(r.choice(DTYPES))
    if seed % 3 == 0:
        x[torch.rand(T, E, generator=g) < 0.2] = float("-inf")
    bias = torch.randn(E, generator=g) * 0.3 if r.random() < 0.6 else None
    if bias is not None and seed % 2:
        bias = bias.bfloat16().float()
    wide = torch.zeros(T, E + 8, dtype=x.dtype, device=cuda)
    wide[:, 4:4 + E] = x.to(cuda)
    at = wide[:, 4:4 + E] if r.random() < 0.4 else x.to(cuda)
    check_route(at, top, r.choice(["softmax", "sigmoid"]), None if bias is None else bias.to(cuda), groups, top_groups, r.choice(["max", "top2"]), r.random() < 0.7,
                r.choice([1.0, 2.5]))


@pytest.mark.parametrize("seed", range(40))
def test_dispatch(cuda, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    top = r.choice([1, 2, 4, 6, 8, 11, 33])
    T, E = max(1, log_uniform(r, 1, 20000) // top), log_uniform(r, 1, 400)
    K = 8 * log_uniform(r, 1, 400 if T > 500 else 2600)
    x = torch.randn(T, K, generator=g).to(r.choice(DTYPES[:2])).to(cuda)
    ids = choose(T, E, top, g)
    ids[torch.rand(T, top, generator=g) < 0.1] = -1
    room = torch.empty(T * top + 3, dtype=torch.int32, device=cuda)
    odd = room[seed % 4:][:T * top].view(T, top)  # at any 4-byte address
    odd.copy_(ids)
    for kind in ("same", "int8", "group"):
        check_dispatch(kind, x, odd, E if seed % 3 else max(1, E // 2), 0 if seed % 3 else E // 3)


@pytest.mark.parametrize("seed", range(40))
def test_combine(cuda, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    T, top, R = log_uniform(r, 1, 6000), r.choice([1, 2, 3, 4, 8, 13, 40]), log_uniform(r, 1, 9000)
    N, dtype = 8 * log_uniform(r, 1, 900 if T < 600 else 60), r.choice(DTYPES[:2])
    y = torch.randn(R, N, generator=g).to(dtype).to(cuda)
    places = torch.randint(-1, R + 1, (T, top), generator=g, dtype=torch.int32).to(cuda)
    check_combine(y, places, torch.rand(T, top, generator=g).to(cuda), torch.randn(T, N, generator=g).to(dtype).to(cuda) if seed % 2 else None)


@pytest.mark.parametrize("seed", range(40))
def test_silu_mul(cuda, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    N = 8 * log_uniform(r, 1, 4500)
    M = log_uniform(r, 1, max(1, min(5000, 4000000 // N)))
    x = (torch.randn(M, 2 * N, generator=g) * 3).to(r.choice(DTYPES[:2])).to(cuda)
    for kind in KINDS:
        check_silu(kind, x)


@pytest.mark.parametrize("seed", range(80))
def test_product(cuda, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    E, K, N = log_uniform(r, 1, 130), 16 * log_uniform(r, 1, 260), log_uniform(r, 1, 3500)
    while E * N * K > 1 << 28:
        N = max(1, N // 2)
    M = log_uniform(r, 1, 6000)
    share = torch.rand(E, generator=g) ** r.choice([0.2, 1, 4])
    counts = torch.multinomial(share + 1e-6, M, replacement=True, generator=g).bincount(minlength=E).tolist()
    q, w, alpha, beta = operands(M, E, N, K, cuda, seed)
    dtype = r.choice(DTYPES[:2])
    bias = r.choice([None, torch.randn(E, N, generator=g).to(cuda), torch.randn(E, N, generator=g).to(dtype).to(cuda)])
    alpha *= 0.1
    off = offsets_of(counts, cuda)
    assert same(product(q, w, alpha, beta, bias, off, dtype), reference(q, w, alpha, beta, bias, off, dtype))


@pytest.mark.parametrize("M", [3, 700, 40000])
@pytest.mark.parametrize("cfg", [-1, 4, 6, 11, 12])
def test_many_experts(cuda, M, cfg):
    """More experts than the row-streaming kernel takes (it is not taken, asked for or not), and the most there are."""
    from llmqrt_amd import _abi
    g = torch.Generator().manual_seed(M)
    for E in (512, 513, 65536):
        counts = torch.randint(0, E, (M,), generator=g).bincount(minlength=E)
        N, K = 24, 32
        q, w, alpha, beta = operands(M, E, N, K, cuda)
        off = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32).to(cuda)
        owner = torch.repeat_interleave(torch.arange(E), counts).to(cuda)
        _abi.check(_abi.lib().llmq_gemm_w8a8_grouped_force_plan(cfg), "force")
        try:
            out = product(q, w, alpha, beta, None, off)
        finally:
            _abi.lib().llmq_gemm_w8a8_grouped_force_plan(-1)
        for m in range(0, M, 8000):
            e = owner[m:m + 8000]
            acc = (q[m:m + 8000, None].double() * w[e].double()).sum(-1).float()
            assert same(out[m:m + 8000], ((acc * alpha[m:m + 8000]) * beta[e]).to(torch.bfloat16))


@pytest.mark.parametrize("T,E,top", [(40, 8, 2), (3000, 16, 4), (9000, 64, 8)])
def test_captured_dispatch(cuda, T, E, top):
    """One launch, two and four: every replay sorts the ids that are there, beside eager calls."""
    from llmqrt_amd.experts import dispatch_to_experts
    g = torch.Generator().manual_seed(T)
    x, ids = torch.randn(T, 16, generator=g).bfloat16().to(cuda), choose(T, E, top, g).to(cuda)
    dispatch_to_experts(x, ids, E)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dispatch_to_experts(x, ids, E)
    for _ in range(4):
        ids.copy_(choose(T, E, top, g))
        want = dispatch_to_experts(x, ids, E)
        graph.replay()
        other = dispatch_to_experts(x, ids.flip(0), E)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want)) and int(other[1][-1]) == T * top


@pytest.mark.parametrize("T,top", [(5, 3), (16, 8), (3000, 4)])
def test_dispatch_to_the_most_experts(cuda, T, top):
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 72, generator=g).bfloat16().to(cuda)
    for kind in ("same", "int8", "group"):
        check_dispatch(kind, x, torch.randint(0, 4096, (T, top), generator=g, dtype=torch.int32).to(cuda), 4096)
