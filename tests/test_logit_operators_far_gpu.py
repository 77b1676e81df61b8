"""GPU: log probabilities of rows that hold finite masks (-1e9, -1e10 ...) or large logits at small temperatures, against
64 bits.

Tolerances count roundings, u = 2^-24, as in test_logit_operators_gpu.py (`chain(V)` for a sum over a row, `reach` for the
expected |z - z_max|).  In addition the sums of the forward pass may be relative to a number that misses the largest z by up to half a
step of it, `residual` <= 8 in base 2: the entropy is then a difference of two numbers of that size, one of which is a quotient of two
sums over the row.
"""

import math

import pytest
import torch

from tests.test_logit_operators_gpu import INF, TYPES, U, chain, check_close, generator, half_step, make_logits, reference_logprobs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi(built):
    from opennn_b200 import capi as module
    module.lib()
    return module


def residual(x, T):
    """Half a step of the largest logit in base 2, at most 8 (beyond that the pass starts from the difference)."""
    z = (x.double().amax(1) / T * math.log2(math.e)).abs().nan_to_num(0, 0, 0)
    return torch.where(z < 2 ** 28, z * U, 0.0)


def entropy_tolerance(x, T, H, reach):
    rel = chain(x.shape[1]) + 4 * U * reach
    return (rel + 8 * U) * (2 + 2 * reach + H.abs().nan_to_num(0.0)) + 2 * residual(x, T) * (rel + U)


def check_far(capi, x, tokens, top, T):
    got = capi.token_logprobs(x, tokens, top=top, temperature=T)
    given, H, lse, ids, values, reach = reference_logprobs(x, tokens, top, T)
    rel = chain(x.shape[1]) + 4 * U * reach + 2 * U * residual(x, T)
    check_close(got[0], given, rel + 6 * U * (given.abs().nan_to_num(0, 0, 0) + reach + 1), "logprob")
    check_close(got[1], H, entropy_tolerance(x, T, H, reach), "entropy")
    z_max = (x.double().amax(1) / T).nan_to_num(0, 0, 0).abs()
    check_close(got[2], lse, rel + 4 * U * (lse.abs().nan_to_num(0, 0, 0) + z_max + 1), "lse")
    if top:
        assert torch.equal(got[3], ids), "top ids"
        check_close(got[4], values, rel[:, None] + 6 * U * (values.abs().nan_to_num(0, 0, 0) + 1 + reach[:, None]), "top values")


def masked_rows(V, dtype, mask, seed=0, copies=1):
    """Ordinary rows of which a part is `mask`: all, either half, all but a last or first stretch, the first stretch, a vector in the
    middle, the first or the last element alone, every other one."""
    i = torch.arange(V, device="cuda")
    where = torch.stack([i >= 0, i < V // 2, i >= V // 2, i < V - 64, i >= 64, i < min(64, V // 2), (i >= V // 3) & (i < V // 3 + 8),
                         i == 0, i == V - 1, i % 2 == 0, i < V - 1]).repeat(copies, 1)
    x = make_logits(where.shape[0], V, dtype, pitch=V + 3, offset=1, seed=seed)
    x[where] = mask
    return x


# fp16 ends at 65504
MASKS = [(dtype, mask) for dtype in TYPES for mask in ((-1e4, -6e4) if dtype == "f16" else (-1e4, -1e7, -1e9, -1e10, -3e10, -1e12, -1e20))]


@pytest.mark.parametrize("T", [1.0, 0.5, 0.3, 0.1, 2.0, 1e-3])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_token_logprobs_finite_masks(capi, dtype, mask, T):
    for V in (41, 1000, 9001, 131072):
        x = masked_rows(V, dtype, mask, seed=V)
        for place in (0, V - 1, V // 2):                  # the last one is masked in some rows, 0 is padding
            tokens = torch.full((x.shape[0],), float(place), device="cuda")
            check_far(capi, x, tokens, 0 if place == V - 1 else 5, T)
        check_far(capi, x, tokens, 64, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_logprobs_finite_masks_of_many_rows(capi, dtype):
    """Rows enough that single warps walk over them."""
    for V, mask, T in ((301, -1e10, 1.0), (2047, -1e9, 0.3), (20011, -1e12, 1.0)):
        x = masked_rows(V, dtype, mask, copies=110)
        tokens = torch.full((x.shape[0],), float(V // 2), device="cuda")
        tokens[::5] = 0.0
        for top in (0, 9, 40):
            check_far(capi, x, tokens, top, T)


@pytest.mark.parametrize("T", [1e-6, 1e-5, 1e-3])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_large_logits_at_small_temperatures(capi, dtype, T):
    for V, spread in ((40, 3.0), (1500, 60.0), (40000, 12000.0)):
        x = make_logits(9, V, dtype, seed=V, spread=spread)
        x[1] = 60000.0
        x[2] = -60000.0
        x[3, V // 2] = 60000.0
        x[4] = torch.where(torch.arange(V, device="cuda") % 3 == 1, 200.0, x[4].float()).to(x.dtype)
        x[5] = 180.0
        tokens = torch.full((9,), float(V // 2), device="cuda")
        tokens[8] = float(V - 1)
        for top in (0, 3):
            check_far(capi, x, tokens, top, T)
