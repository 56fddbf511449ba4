"""GPU: what the products and operators by experts promise beyond their results on ordinary inputs."""
import pytest
import torch

from test_gpu_fp8_block import all_configs, exact_operands, grouped, grouped64
from test_gpu_w8a8_grouped import rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,M", [(4, 200), (70, 333)])
def test_block_scaled_offsets_that_descend(cuda, E, M):
    """Offsets below an earlier one count as that: every row has one expert at most, in every configuration, as in the W8A8 product by experts.  (Operands whose sums are
    exact: a row's bits are its expert's.)"""
    from llmqrt_amd import _abi
    a, w, sa, sw = exact_operands(M, 140, 272, 3, cuda, lead=(E,))
    g = torch.Generator().manual_seed(E)
    cases = [[0, M] * E, [M, 0] * E, [50, 20, 90, 80, 120] * E, [-9, -3, 5, 2 ** 31 - 1, -2 ** 31] * E, [7, 7, 150, 10] * E,
             torch.randint(-20, M + 20, (E + 1,), generator=g).tolist(), torch.randint(0, M + 1, (E + 1,), generator=g).sort().values.tolist()]
    for at in cases:
        at = at[:E + 1]
        off, ends = torch.tensor(at, dtype=torch.int32, device=cuda), rows_of(at, M)
        want = grouped64(a, w, sa, sw, ends, fill=7.0)[0].bfloat16()
        for cfg in [-1, *all_configs()]:
            room = torch.full((M + 2, 140), 7.0, dtype=torch.bfloat16, device=cuda)
            assert _abi.lib().llmq_gemm_fp8_block_force_plan(cfg, 0) == 0
            try:
                grouped(a, w, sa, sw, off, out=room[1:-1])
            finally:
                _abi.lib().llmq_gemm_fp8_block_force_plan(-1, 0)
            assert torch.equal(room[1:-1], want) and (room[0] == 7).all() and (room[-1] == 7).all(), (at[:6], cfg)


@pytest.mark.parametrize("kind", ["same", "int8", "fp8", "group"])
@pytest.mark.parametrize("N", [256, 18944, 33000])
def test_gates_whose_exponential_leaves_fp32(cuda, kind, N, monkeypatch):
    """exp(-g) is no fp32 number below -88, g sigmoid(g) u still one where u is large: the bound of ordinary gates, u_32 (2 |g| + 8) |y|, holds for far ones too,
    without a term in u of more than 3e-74 (exp(-174), behind which y is 0) and fp32's smallest normal number."""
    import test_gpu_silu_mul as ordinary

    def exact(x):
        g, u = x.double().chunk(2, dim=-1)
        y = g * torch.sigmoid(g) * u
        return y, ordinary.U * (2 * g.abs() + 8) * y.abs() + 3e-74 * u.abs() + 2.0 ** -126
    monkeypatch.setattr(ordinary, "exact", exact)
    x = torch.ones(9, 2 * N, dtype=torch.float64)
    x[:, :N] = torch.linspace(-200, -60, N, dtype=torch.float64)
    x[1, N:], x[2, N:], x[3, N:], x[4, N:] = 3e38, -1e30, 1e-30, 6e4
    x[5, :N], x[5, N:] = -89.0, 3e38
    x[6, : N - 1] = 2.0  # one far gate in a row of others
    x[7, :N], x[7, N:] = torch.linspace(-81, -79, N, dtype=torch.float64), 2e35
    x[8, :N], x[8, N:] = torch.linspace(-178, -170, N, dtype=torch.float64), 3e38
    x = x.to(torch.bfloat16)
    ordinary.check(kind, x.to(cuda))
    if kind == "same":
        y = ordinary.call(kind, x.to(cuda))
        assert ((y[5].double().cpu() / (x[5, :N].double() * torch.sigmoid(x[5, :N].double()) * x[5, N:].double()) - 1).abs() < 0.0041).all()
    ordinary.check(kind, x[[0, 4]].half().to(cuda))


@pytest.mark.parametrize("T,E,groups", [(3, 40, 1), (9, 64, 4), (70, 256, 8), (3000, 128, 1), (5, 300, 5), (4, 1024, 1)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_weights_of_a_softmax_without_value_are_nan(cuda, T, E, groups, bad):
    """A NaN or an infinity among the logits leaves the softmax of a token no value: its weights are NaN, with a bias and without, divided by their sum or not; its
    experts are in range and none twice, and other tokens do not notice."""
    from llmqrt_amd.experts import route_to_experts
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, E, generator=g).to(cuda)
    wrong = x.clone()
    wrong[1, E - 3] = bad  # (not among the lowest experts, which are chosen where all scores are NaN)
    rest = [t for t in range(T) if t != 1]
    for bias in (None, (torch.randn(E, generator=g) * 0.1).to(cuda)):
        for score in ("max", "top2"):
            for renormalize in (True, False):
                args = (4, "softmax", bias, groups, max(1, groups // 2), score, renormalize, 2.0)
                (w, ids), (w0, ids0) = route_to_experts(wrong, *args), route_to_experts(x, *args)
                assert w[1].isnan().all() and len(set(ids[1].tolist())) == 4 and ((ids[1] >= 0) & (ids[1] < E)).all()
                assert torch.equal(w[rest], w0[rest]) and torch.equal(ids[rest], ids0[rest])


def test_a_group_with_one_expert_left(cuda):
    """Where masks leave one expert of a group, the sum of its two largest scores is that one's alone, in the short form and in the long one."""
    from llmqrt_amd.experts import route_to_experts
    for T, E, groups in ((3, 16, 4), (40, 256, 8), (3000, 64, 2), (4, 600, 4)):
        n = E // groups
        x = torch.full((T, E), -8.0, device=cuda)
        x[:, :n] = -float("inf")
        x[:, 1] = 3.0  # sigmoid 0.953, alone
        x[:, n:n + 2] = torch.tensor([-0.4, -0.5], device=cuda)  # 0.401 + 0.378
        w, ids = route_to_experts(x, 1, "sigmoid", None, groups, 1, "top2")
        assert (ids == 1).all() and (w == 1).all()
        x[:, 2] = -3.0  # and 0.047: 1.0
        x[:, n:n + 2] = 0.05  # 0.5125 twice
        assert (route_to_experts(x, 1, "sigmoid", None, groups, 1, "top2")[1] == n).all()


def test_order_of_saturated_scores(cuda):
    """Logits decide without a bias; where scores are formed, in 64 bits, those that are level there are ties."""
    from llmqrt_amd.experts import route_to_experts
    x = torch.tensor([[40.0, 41.0, 42.0, 39.0]], device=cuda)
    assert route_to_experts(x, 4, "sigmoid")[1].tolist() == [[2, 1, 0, 3]]
    assert route_to_experts(x, 2, "sigmoid", None, 2, 2, "max")[1].tolist() == [[2, 1]]
    assert route_to_experts(x, 4, "sigmoid", None, 2, 2, "top2")[1].tolist() == [[0, 1, 2, 3]]
    assert route_to_experts(x, 4, "sigmoid", torch.zeros(4, device=cuda))[1].tolist() == [[0, 1, 2, 3]]
