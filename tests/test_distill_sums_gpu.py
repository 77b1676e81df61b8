"""GPU: the sums over rows that onn_distill3d_fwd_bwd reports, at row counts where fp32 would not hold them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def capi(built):
    from opennn_b200 import capi as module
    module.lib()
    return module


@pytest.mark.parametrize("rows", [300_000, 4_194_304])
def test_distill_sums_over_many_rows(capi, rows):
    """The sums of the rows' losses are rounded once, however many rows there are and however alike they are."""
    V = 2
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    targets = torch.ones(rows, device="cuda")
    targets[::1001] = 0.0
    ids, values = torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), torch.zeros(rows, 1, device="cuda")
    for T, a, b in ((1.0, 0.5, 0.5), (2.0, 0.5, 0.5)):
        stats, losses, _ = capi.distill3d(x, targets, ids, values, temperature=T, soft_weight=a, hard_weight=b, want_gradient=False)
        want = losses.double().sum(1)
        # 64-bit sums of fp32 numbers: an error of rows * 2^-53 at most, then half a step of fp32
        assert ((stats[:2].double() - want).abs() <= (1 + 1e-6) * U * want).all(), (stats, want)
        assert stats[2] == (targets > 0).sum()


def test_distill_count_past_24_bits(capi):
    """#active is counted in whole numbers and rounded once: 2^25 + 6 rows make 2^25 + 8 in fp32."""
    rows, V = (1 << 25) + 64, 2
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    targets = torch.ones(rows, device="cuda")
    targets[(1 << 25) + 1:(1 << 25) + 32] = 0.0
    targets[(1 << 25) + 37:] = 0.0
    ids, values = torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), torch.zeros(rows, 1, device="cuda")
    active = int((targets > 0).sum())
    assert active == (1 << 25) + 6
    stats, _, _ = capi.distill3d(x, targets, ids, values, want_gradient=False)
    assert stats[2].item() == (1 << 25) + 8
