"""GPU: the operators around products by experts in a run, as a layer uses them: routing, dispatch, product, gated activation, product, combine.

Steps that plain indexing replaces (dispatch, combine) and the products one expert at a time have to give the same bits.  Against 64 bits (int8): codes of the first
quantizer and the first product are exact, so the layer's input to the activation is known to the bit; the second quantizer is off by half a step of its scale
and what the fp32 activation is off by, which the second product passes on as (s / 2 + slack) sum_k |W[n, k]|; y is rounded to its type, and the sum of a token's rows
once more."""
import threading

import pytest
import torch

from test_gpu_experts import route64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def same(a, b):
    return bool(torch.equal(a, b))


def layer(kind, dev, E=8, K=256, I=192, N=256, top=2, dtype=torch.bfloat16, seed=0, bias=False, **routing):
    from llmqrt_amd.linear import FP8BlockGroupedLinear, GatedExperts, SqW8A8GroupedLinear
    cls = SqW8A8GroupedLinear if kind == "int8" else FP8BlockGroupedLinear
    torch.manual_seed(seed)
    mods = [[torch.nn.Linear(a, b, bias=bias) for _ in range(E)] for a, b in ((K, 2 * I), (I, N))]
    first = routing.pop("first_expert", 0)
    score_bias = routing.pop("score_bias", None)
    m = GatedExperts(*(cls.from_linears([x.to(dev) for x in part], dtype) for part in mods), top, score_bias, first, **routing)
    return m.to(dev)


def inputs(T, K, E, dev, dtype=torch.bfloat16, seed=1):
    g = torch.Generator().manual_seed(seed + T)
    return torch.randn(T, K, generator=g).to(dtype).to(dev), (torch.randn(T, E, generator=g) * 1.5).to(dev)


def by_indexing(kind, m, x, logits, alone):
    """Rows sorted by torch, or (``alone``) every expert's product by itself; -> the weights and y in the order of the tokens' experts."""
    from llmqrt_amd.activation import silu_mul_per_group_quantize, silu_mul_quantize_activation_per_token_absmax
    from llmqrt_amd.experts import route_to_experts
    from llmqrt_amd.quantize import per_group_quantize, quantize_activation_per_token_absmax_f32
    E, top = m.gate_up.num_experts, m.top_k
    w, ids = route_to_experts(logits, top, bias=m.score_bias, **m.routing)
    q, s = quantize_activation_per_token_absmax_f32(x) if kind == "int8" else per_group_quantize(x)
    y = torch.zeros(ids.numel(), m.down.out_features, dtype=x.dtype, device=x.device)
    order = ids.view(-1).argsort(stable=True)
    counts = [int((ids == e).sum()) for e in range(E)]
    at = 0
    for e in range(E if alone else 1):
        mine = order[at:at + counts[e]] if alone else order
        at += counts[e]
        if len(mine):
            rows = [len(mine) if i == e else 0 for i in range(E)] if alone else counts
            off = torch.tensor([0] + rows).cumsum(0).to(torch.int32).to(x.device)
            t = mine // top
            h = m.gate_up.forward_quantized(q.view(torch.int8)[t].view(q.dtype), s[t], off)
            a = silu_mul_quantize_activation_per_token_absmax(h) if kind == "int8" else silu_mul_per_group_quantize(h)
            y[mine] = m.down.forward_quantized(*a, off)
    return w, y


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("T,E,K,I,N,top", [(1, 8, 256, 192, 256, 2), (7, 8, 256, 192, 256, 3), (33, 16, 896, 304, 896, 4), (600, 12, 512, 384, 520, 4), (1100, 64, 256, 128, 264, 8)])
def test_layer(cuda, T, E, K, I, N, top, kind):
    from llmqrt_amd.experts import combine_from_experts
    m = layer(kind, cuda, E, K, I, N, top)
    x, logits = inputs(T, K, E, cuda)
    out = m(x, logits)
    places = torch.arange(T * top, dtype=torch.int32, device=cuda).view(T, top)
    for alone in (False, True) if kind == "int8" else (False,):  # (fp8 sums over K are taken in an order that follows from the number of rows)
        w, y = by_indexing(kind, m, x, logits, alone)
        assert same(out, combine_from_experts(y, places, w))
        terms = y.double().view(T, top, N) * w.double()[..., None]
        want, mass = terms.sum(1), terms.abs().sum(1)
        assert ((out.double() - want).abs() <= torch.finfo(x.dtype).eps / 2 * want.abs() * 1.01 + U * (top + 2) * mass).all()


@pytest.mark.parametrize("T,bias", [(5, False), (300, True)])
def test_layer_against_64_bits(cuda, T, bias):
    E, K, I, N, top = 6, 320, 208, 264, 2
    m = layer("int8", cuda, E, K, I, N, top, bias=bias, scoring="sigmoid", score_bias=torch.randn(E, generator=torch.Generator().manual_seed(3)) * 0.1, scale=1.5)
    x, logits = inputs(T, K, E, cuda)
    out = m(x, logits)
    W, ids = route64(logits, top, "sigmoid", m.score_bias.cpu(), 1, 1, "max", True, 1.5)
    f = x.double()
    s = (f.abs().amax(1, keepdim=True).clamp_min(torch.tensor(1e-5).bfloat16().item()) / 127).bfloat16().double()
    codes = (f / s).bfloat16().double().round().clamp(-128, 127)
    want, bound = torch.zeros(T, N, dtype=torch.float64, device=cuda), torch.zeros(T, N, dtype=torch.float64, device=cuda)
    for j in range(top):
        for e in range(E):
            t = (ids[:, j] == e).nonzero().view(-1).to(cuda)
            if not len(t):
                continue
            h = ((codes[t] @ m.gate_up.qweight[e].double().t()).float() * s[t].float()) * m.gate_up.weight_scale[e]
            h = (h if not bias else h + m.gate_up.bias[e].float()).bfloat16().double()
            g, u = h[:, :I], h[:, I:]
            a = g * torch.sigmoid(g) * u
            off = U * (2 * g.abs() + 8) * a.abs()
            step = a.abs().amax(1, keepdim=True).clamp_min(1e-5) / 127
            wd = m.down.qweight[e].double() * m.down.weight_scale[e].double()[:, None]
            y = a @ wd.t() + (m.down.bias[e].double() if bias else 0)
            err = (step * 0.5001 + off.amax(1, keepdim=True) * 2) * wd.abs().sum(1) + torch.finfo(x.dtype).eps / 2 * y.abs() * 1.01
            weight = W[t.cpu(), j].to(cuda)[:, None]
            want[t] += weight * y
            bound[t] += weight * err * 1.01
    assert ((out.double() - want).abs() <= bound + torch.finfo(x.dtype).eps * want.abs() + 1e-6).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_padding_and_shared(cuda, kind):
    """Rows of masked logits get the shared row alone; others do not notice; any leading dimensions."""
    m = layer(kind, cuda, top=3)
    x, logits = inputs(24, 256, 8, cuda)
    want = m(x, logits)
    pad = logits.clone()
    pad[::5] = float("-inf")
    shared = torch.randn(24, 256, generator=torch.Generator().manual_seed(2)).bfloat16().to(cuda)
    out = m(x, pad, shared)
    assert same(out[::5], shared[::5])
    bare = m(x, pad)
    assert (bare[::5] == 0).all()
    keep = [t for t in range(24) if t % 5]
    if kind == "int8":
        assert same(bare[keep], want[keep])
    assert same(m(x.view(2, 3, 4, 256), pad.view(2, 3, 4, 8), shared.view(2, 3, 4, 256)).view(24, 256), out)
    assert m(x[:0], pad[:0]).shape == (0, 256)
    few = logits.clone()
    few[:, 2:] = float("-inf")  # fewer experts than asked for
    assert m(x, few).isfinite().all()


@pytest.mark.parametrize("T", [9, 1500])
def test_parts_of_the_experts(cuda, T):
    """Two halves of the experts, as two GPUs hold them: their outputs add up to the layer's, up to the roundings of three sums."""
    from llmqrt_amd.linear import GatedExperts, SqW8A8GroupedLinear
    m = layer("int8", cuda, top=3)
    x, logits = inputs(T, 256, 8, cuda)
    whole, parts = m(x, logits).double(), []
    for first in (0, 4):
        pair = []
        for lin in (m.gate_up, m.down):
            p = SqW8A8GroupedLinear(4, lin.in_features, lin.out_features, dev=cuda)
            p.qweight.copy_(lin.qweight[first:first + 4])
            p.weight_scale.copy_(lin.weight_scale[first:first + 4])
            pair.append(p)
        parts.append(GatedExperts(*pair, 3, first_expert=first)(x, logits).double())
    tol = torch.finfo(x.dtype).eps / 2 * 1.02 * (whole.abs() + parts[0].abs() + parts[1].abs()) + 1e-6
    assert ((parts[0] + parts[1] - whole).abs() <= tol).all() and parts[0].abs().max() > 0 and parts[1].abs().max() > 0


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("T", [4, 700])
def test_captured(cuda, kind, T):
    """Every replay follows the routing of its inputs, beside eager calls of the same layer."""
    m = layer(kind, cuda, top=4)
    x, logits = inputs(T, 256, 8, cuda)
    sx, sl = x.clone(), logits.clone()
    m(sx, sl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(sx, sl)
    for k in range(4):
        nx, nl = inputs(T, 256, 8, cuda, seed=10 + k)
        nl[:, k] += 6.0 * (k % 2)
        want = m(nx, nl)
        sx.copy_(nx)
        sl.copy_(nl)
        graph.replay()
        other = m(x, logits)
        torch.cuda.synchronize()
        assert same(out, want) and other.isfinite().all()


def test_streams_and_threads(cuda):
    """Four threads with a stream each, every one with its own layer and sizes: what each gets alone."""
    cases = [(kind, T, layer(kind, cuda, seed=T, top=2), *inputs(T, 256, 8, cuda)) for kind, T in (("int8", 3), ("fp8", 40), ("int8", 900), ("fp8", 1300))]
    want = [m(x, logits) for _, _, m, x, logits in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                got = cases[i][2](*cases[i][3:])
                torch.cuda.current_stream().synchronize()
                if not same(got, want[i]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


def test_grouped_module(cuda):
    """SqW8A8GroupedLinear: from activations, from codes, and one expert at a time with the module of one expert."""
    from llmqrt_amd.linear import SqW8A8BBF16OBF16PerChannel, SqW8A8GroupedLinear
    from llmqrt_amd.quantize import quantize_activation_per_token_absmax_f32
    torch.manual_seed(5)
    mods = [torch.nn.Linear(384, 136, bias=True).to(cuda) for _ in range(3)]
    singles = [SqW8A8BBF16OBF16PerChannel.from_linear(m, 8, 0, init_only=False, dtype=torch.float16) for m in mods]
    lin = SqW8A8GroupedLinear.from_linears(singles)
    x = torch.randn(50, 384, generator=torch.Generator().manual_seed(6)).half().to(cuda)
    off = torch.tensor([0, 20, 20, 50], dtype=torch.int32, device=cuda)
    y = lin(x, off)
    assert y.dtype == torch.float16 and same(y, torch.cat([singles[0](x[:20]), singles[2](x[20:])]))
    assert same(lin.forward_quantized(*quantize_activation_per_token_absmax_f32(x), off), y)
    out = torch.full((50, 136), 7.0, dtype=torch.float16, device=cuda)
    assert lin(x, torch.tensor([5, 20, 20, 40], dtype=torch.int32, device=cuda), out) is out
    assert same(out[5:20], y[5:20]) and (out[:5] == 7).all() and (out[40:] == 7).all()
    wide = torch.cat([x, x], 1)[:, :384]
    assert same(lin(wide, off), y) and lin(x[:0], off).shape == (0, 136)
