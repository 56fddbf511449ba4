"""GPU: routing, dispatch and combine against plain forms in 64 bits.

Whole numbers - experts, offsets, places - and rows have to be the same: ties go to the lowest expert, the order of rows is a stable sort's, and quantized rows are
the bits of the framework's quantizers.  Weights: |error| <= u (R + E + 12) w, u = 2^-24, R the largest difference of two logits: x - m loses u R, which exp
passes on; the sum of E terms loses at most u each, exp, the quotients and the factor a few more.  Sums of a combine: (eps(out) / 2) |y| for the last rounding
and u (top_k + 2) sum_j |w y| for the fp32 sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
INF = float("inf")


def same(a, b):
    return bool(torch.equal(a, b))


# ---- routing

def route64(logits, top, scoring, bias, groups, top_groups, score, renormalize, scale):
    """-> weights (64 bits), experts, by choosing one expert after the other."""
    x = logits.double().cpu()
    T, E = x.shape
    finite = x > -INF
    s = torch.zeros_like(x)
    for t in range(T):
        if finite[t].any():
            v = x[t][finite[t]]
            s[t][finite[t]] = torch.softmax(v, 0) if scoring == "softmax" else 1 / (1 + torch.exp(-v))
    # without a bias the order of the scores is the logits' (which stay apart where scores underflow)
    c = (x.clone() if bias is None and (groups == 1 or score == "max") else s + (0 if bias is None else bias.double().cpu())).masked_fill(~finite, -INF)
    if bias is not None:
        c[:, bias.cpu() == -INF] = -INF
    size = E // groups
    W, I = torch.zeros(T, top, dtype=torch.float64), torch.full((T, top), -1, dtype=torch.int32)
    for t in range(T):
        left = c[t].tolist()
        if groups > 1:
            best = []
            for g in range(groups):
                m = sorted((v for v in left[g * size:(g + 1) * size] if v > -INF), reverse=True)
                best.append(-INF if not m else m[0] if score == "max" else sum(m[:2]))
            kept = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
            left = [v if i // size in kept else -INF for i, v in enumerate(left)]
        order = sorted((i for i in range(E) if left[i] > -INF), key=lambda i: (-left[i], i))[:top]
        if not order:
            continue
        I[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
        v = x[t][order]
        if renormalize:  # ratios, taken relative to the largest so that none underflows
            log = v if scoring == "softmax" else -torch.nn.functional.softplus(-v)
            W[t, :len(order)] = torch.softmax(log, 0) * scale
        else:
            W[t, :len(order)] = s[t][order] * scale
    return W, I


def check_route(logits, top, scoring="softmax", bias=None, groups=1, top_groups=1, score="max", renormalize=True, scale=1.0):
    from llmqrt_amd.experts import route_to_experts
    w, ids = route_to_experts(logits, top, scoring, bias, groups, top_groups, score, renormalize, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.shape == ids.shape == (*logits.shape[:-1], top)
    rows = logits.reshape(-1, logits.shape[-1])
    W, I = route64(rows, top, scoring, bias, groups, top_groups, score, renormalize, scale)
    w, ids = w.reshape(-1, top).cpu().double(), ids.reshape(-1, top).cpu()
    assert same(ids, I)
    f = rows.float()[rows.float() > -INF]
    spread = (f.max() - f.min()).item() if f.numel() else 0.0
    assert ((w - W).abs() <= U * (2 * spread + rows.shape[1] + 12) * W + 1e-37).all()  # (the last: fp32's smallest normal numbers)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,top", [(1, 1, 1), (1, 8, 8), (3, 17, 5), (16, 64, 8), (33, 60, 4), (17, 65, 3), (40, 128, 6), (7, 129, 8), (100, 256, 8), (5, 257, 7),
                                     (9, 1000, 64), (3, 1024, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route(cuda, T, E, top, dtype, scoring):
    g = torch.Generator().manual_seed(T * 7 + E)
    x = (torch.randn(T, E, generator=g) * 2).to(dtype).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.2).to(cuda)
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        check_route(x, top, scoring, None, renormalize=renormalize, scale=scale)
        check_route(x, top, scoring, bias, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("T,E,groups,top_groups,top", [(5, 16, 4, 2, 3), (20, 64, 8, 3, 8), (9, 60, 6, 1, 4), (64, 256, 8, 4, 8), (7, 96, 32, 5, 6), (4, 640, 64, 64, 9),
                                                       (3, 1024, 2, 1, 8), (6, 63, 7, 2, 18)])
@pytest.mark.parametrize("score", ["max", "top2"])
def test_route_groups(cuda, T, E, groups, top_groups, top, score):
    g = torch.Generator().manual_seed(E + top)
    x = (torch.randn(T, E, generator=g) * 1.5).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.1).to(cuda)
    for scoring in ("softmax", "sigmoid"):
        check_route(x, top, scoring, None, groups, top_groups, score)
        check_route(x, top, scoring, bias, groups, top_groups, score, renormalize=False)
    x[:, ::3] = -INF
    x[0] = -INF
    check_route(x, top, "sigmoid", bias, groups, top_groups, score)
    check_route(x, top, "softmax", None, groups, top_groups, score)


def test_route_ties_and_zeros(cuda):
    """Equal scores go to the lowest expert, 0 and -0 are equal, and logits far apart keep their order where their scores are the same in any precision."""
    x = torch.zeros(4, 100, device=cuda)
    x[1, ::2] = -0.0
    x[2, 50:] = 1.0
    x[3] = 40 + torch.arange(100, device=cuda).flip(0) % 10  # sigmoid is 1 - 1e-18 and more
    for scoring in ("softmax", "sigmoid"):
        check_route(x, 12, scoring)
        check_route(x[:3], 12, scoring, torch.ones(100, device=cuda))
        check_route(x[:3], 12, scoring, None, 10, 4, "top2")
    half = torch.randint(-4, 4, (64, 256), generator=torch.Generator().manual_seed(1)).half().to(cuda)
    check_route(half, 8)
    check_route(half, 8, "sigmoid", torch.zeros(256, device=cuda), 8, 3, "top2")


@pytest.mark.parametrize("E,groups,top_groups,score", [(48, 1, 1, "max"), (128, 1, 1, "max"), (256, 1, 1, "max"), (64, 8, 3, "top2"), (256, 8, 4, "top2"), (160, 8, 3, "max")])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route_close_scores(cuda, E, groups, top_groups, score, scoring):
    """Scores with the bias in pairs, threes and fours that 32 bits do not tell apart: the order is that of 64 bits.  (The biases lift neighbours, in a shuffled order, to
    the same score up to their own rounding, 2^-25 at most; what 64 bits compute is off by 2^-52.)"""
    g = torch.Generator().manual_seed(E + groups)
    T = 400
    x = torch.randn(T, E, generator=g).bfloat16().float()
    x[1:] = x[0] + torch.randint(-1, 2, (T - 1, 1), generator=g).float() * 2.0 ** -20 * torch.randint(0, 2, (T - 1, E), generator=g)
    s = torch.sigmoid(x[0].double()) if scoring == "sigmoid" else torch.softmax(x[0].double(), 0)
    order = torch.randperm(E, generator=g)
    aim = torch.empty(E, dtype=torch.float64)
    at, value = 0, 1.5
    while at < E:
        n = int(torch.randint(1, 5, (1,), generator=g))
        aim[order[at:at + n]] = value
        at, value = at + n, value - 0.01
    bias = (aim - s).float()
    c = s[None] * 0 + (torch.sigmoid(x.double()) if scoring == "sigmoid" else torch.softmax(x.double(), 1)) + bias.double()
    gaps = c.sort(1, descending=True).values.diff(dim=1).abs()
    assert ((gaps > 0) & (gaps < 1e-7)).any(1).float().mean() > 0.9 and not ((gaps > 0) & (gaps < 1e-13)).any()
    check_route(x.to(cuda), 8, scoring, bias.to(cuda), groups, top_groups, score)
    check_route(x[:5].to(cuda), 8, scoring, bias.to(cuda), groups, top_groups, score)


@pytest.mark.parametrize("E,groups,top_groups,score", [(4, 1, 1, "max"), (64, 1, 1, "max"), (128, 1, 1, "max"), (256, 1, 1, "max"), (64, 4, 4, "top2"), (256, 8, 8, "max")])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [5, 3500])
def test_route_close_scores_at_the_last_choice(cuda, E, groups, top_groups, score, scoring, T):
    """The last choice lies among two, three or four scores that 32 bits do not tell apart, some of them not chosen."""
    g = torch.Generator().manual_seed(E + T)
    near = 8.0 if scoring == "sigmoid" else 0.0  # sigmoids near 1, or shares of a softmax near each other
    for top in (1, 2, 3):
        x = torch.randn(T, E, generator=g) - 12
        for t in range(T):
            at = torch.randperm(E, generator=g)[:4]
            few = 2 + t % 3 if E > 4 else 4
            x[t, at[:few]] = near + torch.randint(-6, 7, (few,), generator=g) * 2.0 ** -20
        check_route(x.to(cuda), min(top, E), scoring, torch.zeros(E, device=cuda), groups, top_groups, score)


def test_route_masks(cuda):
    """-inf is never chosen, the type's lowest value is a value; a row without experts goes nowhere."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        low = torch.finfo(dtype).min
        x = torch.randn(6, 40, generator=torch.Generator().manual_seed(2)).to(dtype)
        x[0] = -INF
        x[1, 3:] = -INF
        x[2, 1:] = low
        x[3] = low
        x[4, :39] = -INF
        for scoring in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                check_route(x.to(cuda), 5, scoring, renormalize=renormalize)
    bias = torch.zeros(40, device=cuda)
    bias[7:] = -INF
    check_route(torch.randn(5, 40, generator=torch.Generator().manual_seed(3)).to(cuda), 9, "sigmoid", bias)


def test_route_not_finite(cuda):
    """Experts in range and none twice, whatever the logits; other tokens do not notice."""
    from llmqrt_amd.experts import route_to_experts
    x = torch.randn(64, 48, generator=torch.Generator().manual_seed(4)).to(cuda)
    want = [route_to_experts(x, 6, *a) for a in (("softmax",), ("sigmoid", torch.zeros(48, device=cuda), 4, 2, "top2"))]
    bad = x.clone()
    bad[3, 5], bad[10, :], bad[20, 7] = float("nan"), float("nan"), INF
    keep = [t for t in range(64) if t not in (3, 10, 20)]
    for args, (w0, i0) in zip((("softmax",), ("sigmoid", torch.zeros(48, device=cuda), 4, 2, "top2")), want):
        w, ids = route_to_experts(bad, 6, *args)
        assert same(w[keep], w0[keep]) and same(ids[keep], i0[keep])
        assert ((ids >= 0) & (ids < 48)).all() and all(len(set(r.tolist())) == 6 for r in ids)
        assert w[10].isnan().all() and (args[0] == "sigmoid" or w[3].isnan().all())
        assert 7 in ids[20].tolist()


def test_route_tokens_of_nan(cuda):
    """A token with NaN alone, or NaN and masked experts, beside others: they get what they get without it, and it gets experts in range, none twice."""
    from llmqrt_amd.experts import route_to_experts
    g = torch.Generator().manual_seed(14)
    for T, E, groups in ((40, 64, 1), (40, 256, 8), (3100, 128, 4), (4200, 256, 1), (6000, 256, 8)):
        x = torch.randn(T, E, generator=g).to(cuda)
        bias = (torch.randn(E, generator=g) * 0.1).to(cuda)
        bad = x.clone()
        bad[3] = float("nan")
        bad[T - 1] = float("nan")
        bad[T // 2, 1:], bad[T // 2, 0] = -INF, float("nan")
        rest = [t for t in range(T) if t not in (3, T // 2, T - 1)]
        for scoring, b in (("softmax", None), ("sigmoid", bias), ("softmax", bias)):
            w, ids = route_to_experts(bad, 4, scoring, b, groups, groups, "max" if b is None else "top2")
            w0, ids0 = route_to_experts(x, 4, scoring, b, groups, groups, "max" if b is None else "top2")
            assert same(ids[rest], ids0[rest]) and same(w[rest], w0[rest])
            for t in (3, T // 2, T - 1):
                own = [i for i in ids[t].tolist() if i >= 0]
                assert all(i < E for i in own) and len(set(own)) == len(own) and ids[t].min() >= -1


def test_route_far_logits(cuda):
    """Renormalised weights are ratios, also of scores that underflow."""
    x = torch.full((3, 32), -200.0, device=cuda)
    x[0, 4], x[1, 5], x[2] = -150.0, 3.0, -90 - torch.arange(32, device=cuda).float() / 8
    check_route(x, 4, "sigmoid")
    check_route(x, 4, "softmax")
    bias = torch.zeros(32, device=cuda)
    bias[8:12] = 1e3
    check_route(x * 10, 4, "softmax", bias)


def test_route_layouts(cuda):
    from llmqrt_amd.experts import route_to_experts
    big = torch.randn(30, 200, generator=torch.Generator().manual_seed(5)).to(cuda)
    for view in (big[:, 3:67], big[::2, :64], big[:, ::2], big.t()[:60], big.view(5, 6, 200)[..., :96], big[4, :40], big[:1, 7:50].expand(6, 43), big.bfloat16()[:, 1:50]):
        w, ids = route_to_experts(view, 3)
        w2, ids2 = route_to_experts(view.contiguous(), 3)
        assert same(w, w2) and same(ids, ids2) and w.shape == (*view.shape[:-1], 3)
    w, ids = route_to_experts(big[:0], 3)
    assert w.shape == ids.shape == (0, 3)
    for bad in (lambda: route_to_experts(big, 0), lambda: route_to_experts(big, 65), lambda: route_to_experts(big, 2, num_groups=7),
                lambda: route_to_experts(big, 2, num_groups=4, top_groups=5), lambda: route_to_experts(big, 3, num_groups=100, top_groups=1),
                lambda: route_to_experts(big, 2, bias=torch.zeros(200)), lambda: route_to_experts(big, 2, bias=torch.zeros(199, device=cuda)),
                lambda: route_to_experts(big, 2, bias=torch.zeros(200, device=cuda).half()), lambda: route_to_experts(big.double(), 2),
                lambda: route_to_experts(big.repeat(1, 6), 2)):
        with pytest.raises(RuntimeError):
            bad()


# ---- dispatch

def sorted64(ids, experts, first):
    """offsets, places and the tokens of the rows."""
    flat = ids.reshape(-1).tolist()
    parts = [[] for _ in range(experts)]
    for i, e in enumerate(flat):
        if first <= e < first + experts:
            parts[e - first].append(i)
    order = [i for p in parts for i in p]
    places, offsets = [-1] * len(flat), [0]
    for r, i in enumerate(order):
        places[i] = r
    for p in parts:
        offsets.append(offsets[-1] + len(p))
    top = ids.shape[-1]
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(places, dtype=torch.int32).view(ids.shape), torch.tensor([i // top for i in order], dtype=torch.long)


def dispatched(kind, x, ids, E, first=0):
    from llmqrt_amd import experts
    f = {"same": experts.dispatch_to_experts, "int8": experts.dispatch_quantize_activation_per_token_absmax, "group": experts.dispatch_per_group_quantize}[kind]
    return f(x, ids, E, first)


def as_bytes(t):
    return t.contiguous().view(torch.uint8)


def check_dispatch(kind, x, ids, E, first=0):
    from llmqrt_amd.quantize import per_group_quantize, quantize_activation_per_token_absmax_f32
    got = dispatched(kind, x, ids, E, first)
    offsets, places, token = sorted64(ids.cpu(), E, first)
    dev = x.device
    assert same(got[-2].cpu(), offsets) and same(got[-1].cpu(), places)
    flat = x.reshape(-1, x.shape[-1]).contiguous()
    rows = (flat,) if kind == "same" else quantize_activation_per_token_absmax_f32(flat) if kind == "int8" else per_group_quantize(flat)
    n = int(offsets[-1])
    for g, r in zip(got, rows):
        assert g.shape == (ids.numel(), r.shape[1]) and g.dtype == r.dtype
        assert same(as_bytes(g[:n]), as_bytes(r[token.to(dev)]))


def choose(T, E, top, g):
    if top <= E:
        return (torch.randn(T, E, generator=g) + torch.randn(E, generator=g)).topk(top, dim=1).indices.to(torch.int32)
    return torch.randint(0, E, (T, top), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("kind", ["same", "int8", "group"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,E,top", [(1, 8, 1, 1), (1, 3584, 64, 8), (3, 136, 5, 2), (48, 3584, 64, 4), (17, 1000, 60, 7), (255, 896, 16, 8), (256, 896, 16, 8),
                                       (257, 896, 300, 8), (700, 264, 8, 3), (2049, 128, 128, 1), (130, 2056, 4, 40), (37, 18944, 9, 2), (33, 20488, 3, 64),
                                       (5000, 64, 256, 8), (40, 4104, 4096, 64), (6000, 64, 60, 8), (20001, 8, 200, 3), (41000, 16, 1, 1), (5100, 24, 257, 8), (700, 8, 4096, 5),
                                       (150000, 8, 33, 4)])
def test_dispatch(cuda, T, K, E, top, dtype, kind):
    g = torch.Generator().manual_seed(T + K + E)
    x = torch.randn(T, K, generator=g).to(dtype)
    x[0] = 0
    check_dispatch(kind, x.to(cuda), choose(T, E, top, g).to(cuda), E)


@pytest.mark.parametrize("kind", ["same", "int8", "group"])
@pytest.mark.parametrize("T,top", [(30, 4), (900, 6)])
def test_dispatch_of_a_part(cuda, T, top, kind):
    """Ids outside the part go nowhere: their copies have no place, and rows behind the last are left as they were."""
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 256, generator=g).bfloat16().to(cuda)
    ids = choose(T, 64, top, g)
    ids[1], ids[2, 0], ids[3, 1] = -1, 0x7fffffff, -0x80000000
    for first, n in ((0, 16), (16, 16), (48, 16), (60, 30), (64, 5), (5, 1), (0, 64), (0x7fff0000, 4)):
        check_dispatch(kind, x, ids.to(cuda), n, first)
        wide = ids.long()
        wide[4] += 1 << 32
        gone = ids.clone()
        gone[4] = -1
        a, b = dispatched(kind, x, wide.to(cuda), n, first), dispatched(kind, x, gone.to(cuda), n, first)
        end = int(a[-2][-1])
        assert same(a[-2], b[-2]) and same(a[-1], b[-1]) and all(same(as_bytes(p[:end]), as_bytes(q[:end])) for p, q in zip(a[:-2], b[:-2]))


def test_dispatch_skewed(cuda):
    """All to one expert, the same expert many times for one token, many experts without a token."""
    x = torch.randn(3000, 128, generator=torch.Generator().manual_seed(6)).half().to(cuda)
    for ids in (torch.full((3000, 2), 3), torch.arange(3000)[:, None] % 2 * 7, torch.zeros(3000, 5), torch.arange(6000).view(3000, 2) // 1000):
        check_dispatch("int8", x, ids.to(torch.int32).to(cuda), 8)
        check_dispatch("same", x[:50], ids[:50].to(torch.int32).to(cuda), 8)


@pytest.mark.parametrize("T", [6, 2000, 30000])
def test_dispatch_rows_left_alone(cuda, T):
    """The C entry writes the rows that have an expert and no other byte."""
    from llmqrt_amd import _abi
    L = _abi.lib()
    g = torch.Generator().manual_seed(T)
    K, E, top = 264, 12, 3
    x, ids = torch.randn(T, K, generator=g).bfloat16().to(cuda), choose(T, 24, top, g).to(cuda)
    n = T * top
    rows = torch.full((n + 2, K), 77, dtype=torch.int8, device=cuda)
    scale, places, offsets = torch.full((n + 2,), 7.0, device=cuda), torch.full((n + 2,), 7, dtype=torch.int32, device=cuda), torch.full((E + 3,), 7, dtype=torch.int32, device=cuda)
    need = L.llmq_dispatch_experts_workspace_bytes(T, top, E)
    assert (need > 0) == (T == 30000)
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device=cuda)
    _abi.check(L.llmq_dispatch_experts(1, x.data_ptr(), _abi.BF16, T, K, K, ids.data_ptr(), top, 0, E, rows[1].data_ptr(), scale[1:].data_ptr(), offsets[1:].data_ptr(),
                                       places[1:].data_ptr(), ws.data_ptr(), need, _abi.stream_of(x)), "dispatch")
    off, pl, _ = sorted64(ids.cpu(), E, 0)
    end = int(off[-1])
    assert same(offsets[1:E + 2].cpu(), off) and same(places[1:n + 1].view(T, top).cpu(), pl) and 0 < end < n
    assert (rows[0] == 77).all() and (rows[end + 1:] == 77).all() and scale[0] == 7 and (scale[end + 1:] == 7).all()
    assert (ws[need:] == 77).all() and offsets[0] == 7 and offsets[E + 2] == 7 and places[0] == 7 and places[n + 1] == 7


def test_dispatch_layouts(cuda):
    g = torch.Generator().manual_seed(8)
    big = torch.randn(40, 2048, generator=g).bfloat16().to(cuda)
    ids = torch.randint(0, 10, (40, 6), generator=g, dtype=torch.int32).to(cuda)
    for x, i in ((big[:, :1000], ids), (big[:, 3:1003], ids), (big[::2], ids[::2]), (big[:, ::2], ids[:, 1:4]), (big.view(8, 5, 2048), ids.view(8, 5, 6)), (big[5], ids[5]),
                 (big[:1].expand(40, 2048), ids), (big, ids.long()), (big, ids.t().contiguous().t())):
        for kind in ("same", "int8", "group"):
            check_dispatch(kind, x, i, 10)
    for kind in ("same", "int8", "group"):
        got = dispatched(kind, big[:0], ids[:0], 10)
        assert got[0].shape[0] == 0 and same(got[-2].cpu(), torch.zeros(11, dtype=torch.int32)) and got[-1].shape == (0, 6)


def test_dispatch_not_finite(cuda):
    """An infinity or a NaN stays in its token's rows (in its group for fp8), with the quantizers' own bits."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(20, 640, generator=g).bfloat16()
    x[3, 5], x[7, 300], x[9, 639] = float("nan"), INF, -INF
    ids = choose(20, 6, 2, g).to(cuda)
    for kind in ("same", "int8", "group"):
        check_dispatch(kind, x.to(cuda), ids, 6)


# ---- combine

def check_combine(y, places, weights, shared=None):
    from llmqrt_amd.experts import combine_from_experts
    got = combine_from_experts(y, places, weights, shared)
    p = places.reshape(-1, places.shape[-1]).long()
    has = (p >= 0) & (p < y.shape[0])
    pad = torch.cat([y.double(), torch.zeros(1, y.shape[1], dtype=torch.float64, device=y.device)])
    terms = torch.where(has, weights.reshape(p.shape).double(), 0.0)[..., None] * pad[torch.where(has, p, y.shape[0])]
    want, mass = terms.sum(1), terms.abs().sum(1)
    if shared is not None:
        s = shared.reshape(-1, y.shape[1]).double()
        want, mass = want + s, mass + s.abs()
    assert got.dtype == y.dtype and got.shape == (*places.shape[:-1], y.shape[1])
    bound = torch.finfo(y.dtype).eps / 2 * want.abs() * (1 + 1e-6) + U * (p.shape[1] + 2) * mass + 2.0 ** -25  # (the last: fp16 below its normal range)
    assert ((got.reshape(want.shape).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,N,top,R", [(1, 8, 1, 1), (1, 3584, 8, 8), (48, 3584, 4, 192), (33, 1000, 7, 300), (5, 264, 64, 40), (1001, 896, 2, 2002), (3000, 128, 5, 9), (17, 20488, 3, 60)])
def test_combine(cuda, T, N, top, R, dtype):
    g = torch.Generator().manual_seed(T + N)
    y = torch.randn(R, N, generator=g).to(dtype).to(cuda)
    places = torch.randint(-1, R, (T, top), generator=g, dtype=torch.int32).to(cuda)
    weights = torch.rand(T, top, generator=g).to(cuda)
    check_combine(y, places, weights)
    check_combine(y, places, weights, torch.randn(T, N, generator=g).to(dtype).to(cuda))


def test_combine_places_and_masks(cuda):
    """Places that are no row add nothing, whatever lies in their weight; weight 0 of an infinity is NaN, as the formula has it."""
    from llmqrt_amd.experts import combine_from_experts
    y = torch.randn(6, 64, generator=torch.Generator().manual_seed(10)).bfloat16().to(cuda)
    places = torch.tensor([[-1, -1, -1], [0, 6, 0x7fffffff], [5, -0x80000000, 2], [1, 1, 1], [3, -1, -1]], dtype=torch.int32, device=cuda)
    weights = torch.rand(5, 3, generator=torch.Generator().manual_seed(11)).to(cuda)
    weights[0], weights[1, 1], weights[2, 1] = float("nan"), INF, float("nan")
    y[3, 7], y[4] = INF, float("nan")
    weights[4, 0] = 0
    out = combine_from_experts(y, places, weights)
    assert (out[0] == 0).all() and out[:4].isfinite().all() and out[4, 7].isnan() and (out[4, :7] == 0).all()
    y[3, 7] = 1
    check_combine(y, places[:4], weights[:4].nan_to_num(0.0, 0.0))
    assert same(combine_from_experts(y[:0], places, weights), torch.zeros(5, 64, dtype=torch.bfloat16, device=cuda))


def test_combine_layouts(cuda):
    from llmqrt_amd.experts import combine_from_experts
    g = torch.Generator().manual_seed(12)
    big = torch.randn(40, 512, generator=g).half().to(cuda)
    places = torch.randint(-1, 20, (12, 4), generator=g, dtype=torch.int32).to(cuda)
    weights = torch.rand(12, 4, generator=g).to(cuda)
    for y in (big[:20, :256], big[::2, 8:264], big[:20, 3:259], big[:20, ::2], big[:1, :256].expand(20, 256)):
        want = combine_from_experts(y.contiguous(), places, weights, big[20:32, :256].contiguous())
        assert same(combine_from_experts(y, places, weights, big[20:32, :256]), want)
        assert same(combine_from_experts(y, places.view(3, 4, 4), weights.view(3, 4, 4), big[20:32, :256].reshape(3, 4, 256)), want.view(3, 4, 256))
        assert same(combine_from_experts(y, places.t().contiguous().t(), weights.double(), big[20:32, :256]), want)
    y = big[:20]
    check_combine(y, places, weights.half())
    check_combine(y, places[:, 1], weights[:, 1])
    assert combine_from_experts(y, places[:0], weights[:0]).shape == (0, 512)
    for bad in (lambda: combine_from_experts(y, places.long(), weights), lambda: combine_from_experts(y, places, weights[:, :3]),
                lambda: combine_from_experts(y, places, places), lambda: combine_from_experts(y.float(), places, weights),
                lambda: combine_from_experts(y[:, :500], places, weights), lambda: combine_from_experts(y, places, weights, big[:11]),
                lambda: combine_from_experts(y, places, weights, big[:12].bfloat16()), lambda: combine_from_experts(y, places[:, :0], weights[:, :0]),
                lambda: combine_from_experts(y, places, weights.cpu())):
        with pytest.raises(RuntimeError):
            bad()
