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
