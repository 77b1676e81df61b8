"""GPU: log probabilities, and their gradient, of rows that hold finite masks (-1e9, -1e10 ...) or large logits at small temperatures, against
64 bits.

Tolerances count roundings, u = 2^-24, as in test_logit_operators_gpu.py (`chain(V)` for a sum over a row, `reach` for the
expected |z - z_max|).  In addition the sums of the forward pass may be relative to a number that misses the largest z by up to half a
step of it, `residual` <= 64 in base 2: the entropy is then a difference of two numbers of that size, one of which is a quotient of two
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
    """Half a step of the largest z in base 2 (beyond 2^31 the pass starts from the difference)."""
    z = (x.double().amax(1) / T * math.log2(math.e)).abs().nan_to_num(0, 0, 0)
    return torch.where(z < 2 ** 31, z * U, 0.0)


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
MASKS = [(dtype, mask) for dtype in TYPES for mask in ((-1e4, -6e4) if dtype == "f16" else (-1e4, -1e7, -1e9, -1.4e9, -1.6e9, -1e10, -3e10, -1e12, -1e20))]


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


# ---------------------------------------------------------------------------------------------------------------------

def check_far_bwd(capi, x, tokens, T, with_entropy, seed=3):
    """The gradient against the definition, with p from the logits themselves.  Rows of |lse| < 2^14 take p from lse, whose rounding
    is in it; beyond that only the roundings of the difference from the largest logit are."""
    rows, V = x.shape
    _, H, lse, _, _ = capi.token_logprobs(x, tokens, temperature=T)
    gen = generator(seed)
    # of the temperature's size, so that gradients divided by it fit fp16
    g = torch.randn(rows, generator=gen, device="cuda") * min(T, 1.0)
    h = torch.randn(rows, generator=gen, device="cuda") * min(T, 1.0) if with_entropy else None
    _, true_H, true_lse, _, _, reach = reference_logprobs(x, tokens, 0, T)
    z = x.double() / T
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    active = tokens > 0
    hot = torch.zeros_like(z).scatter_(1, tokens.long()[:, None], 1.0)
    gd, reach = g.double()[:, None], reach[:, None]
    dx = gd * (hot - p)
    lp = torch.where(p > 0, logp, 0.0)
    d = torch.where(p > 0, z - z.amax(1, keepdim=True), 0.0).abs()
    near = (true_lse.abs() < 2 ** 14)[:, None]
    rel = chain(V) + (4 * d + 4 * reach + 8) * U + torch.where(near, 4 * U * (true_lse.abs()[:, None] + z.abs().amin(1, keepdim=True) + d), 0.0)
    tol = gd.abs() * p * rel + 4 * U * dx.abs()
    lost = gd.abs() + 1
    if h is not None:
        hd, Hd = h.double()[:, None], true_H[:, None]
        inner = lp + Hd
        dx = dx - hd * p * inner
        off = entropy_tolerance(x, T, true_H, reach[:, 0])[:, None]
        tol = tol + hd.abs() * p * (inner.abs() * rel + rel + off + 6 * U * (lp.abs() + Hd.abs() + 1))
        lost = lost + hd.abs() * inner.abs()
    eps, tiny = half_step(x.dtype)
    dx, tol = torch.where(active[:, None], dx / T, 0.0), torch.where(active[:, None], tol / T, 0.0)
    # 2^d below 2^-126 is flushed to zero: with it goes p (|g| + |h| |log p + H|) / T, where p < 2^-126 and |log p + H| is about 90
    tol = tol * (1 + eps) + eps * dx.abs() + tiny + 2.0 ** -126 * lost / T
    got = capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T)
    check_close(got, dx, tol, "dlogits")
    # rows of another alignment, and in the logits' place, with their surroundings as they were
    room = torch.full((rows * (V + 5) + 3,), 7.0, dtype=x.dtype, device="cuda")
    out = room[3:].view(rows, V + 5)[:, :V]
    capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T, out=out)
    check_close(out, dx, tol, "dlogits, own pitch")
    assert (room[:3] == 7).all() and (room[3:].view(rows, V + 5)[:, V:] == 7).all()
    capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T, out=x)
    check_close(x, dx, tol, "in place")


@pytest.mark.parametrize("with_entropy", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.3, 0.1, 2.0])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_token_logprobs_bwd_finite_masks(capi, dtype, mask, T, with_entropy):
    for V in (41, 1000, 9001, 50021):
        x = masked_rows(V, dtype, mask, seed=V)
        tokens = torch.full((x.shape[0],), float(V // 2), device="cuda")
        tokens[1] = 0.0
        check_far_bwd(capi, x, tokens, T, with_entropy)


@pytest.mark.parametrize("with_entropy", [False, True])
@pytest.mark.parametrize("T", [1e-6, 1e-5, 1e-3])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_bwd_large_logits_at_small_temperatures(capi, dtype, T, with_entropy):
    for V, spread in ((40, 3.0), (1500, 60.0), (40000, 12000.0)):
        x = make_logits(9, V, dtype, seed=V, spread=spread)
        x[1] = 60000.0
        x[2] = -60000.0
        x[3, V // 2] = 60000.0
        x[4] = torch.where(torch.arange(V, device="cuda") % 3 == 1, 200.0, x[4].float()).to(x.dtype)
        x[5] = 180.0
        tokens = torch.full((9,), float(V // 2), device="cuda")
        tokens[7], tokens[8] = 0.0, float(V - 1)
        check_far_bwd(capi, x, tokens, T, with_entropy)


def test_token_logprobs_bwd_log_sum_past_fp32(capi):
    """z of the largest logit beyond fp32: lse is infinite, the gradient is not."""
    V, T = 300, 0.5
    for value in (3e38, -3e38, -INF):
        x = torch.full((2, V), value, device="cuda")
        x[1, 7] = 2.9e38 if value > 0 else -INF
        tokens = torch.full((2,), 5.0, device="cuda")
        g, h = torch.tensor([0.5, -1.5], device="cuda"), torch.tensor([0.25, 1.0], device="cuda")
        _, H, lse, _, _ = capi.token_logprobs(x, tokens, temperature=T)
        assert torch.isinf(lse).all()
        dx = capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T).double()
        live = x == value if value > -INF else torch.zeros_like(x, dtype=torch.bool)
        p = live.double() / live.sum(1, keepdim=True).clamp(min=1)
        hot = torch.zeros_like(p).scatter_(1, tokens.long()[:, None], 1.0)
        want = g.double()[:, None] * (hot - p) / T                # equal logits: log p + H = 0
        # H and log p, each of size log V, cancel but for their roundings
        tol = (g.abs().double()[:, None] * p * (chain(V) + 8 * U) + h.abs().double()[:, None] * p * 4 * (chain(V) + 8 * U) * (1 + math.log(V))) / T + 4 * U * want.abs()
        check_close(dx, want, tol, "dlogits")


@pytest.mark.parametrize("T", [0.25, 1.0, 2.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_bwd_rows_without_a_finite_logit(capi, dtype, T):
    """p = 0 throughout: the gradient is the token's alone.  Powers of two: no rounding at all."""
    for V in (33, 40000):
        x = torch.full((3, V), -INF, dtype=TYPES[dtype], device="cuda")
        tokens = torch.tensor([1.0, 0.0, V - 1.0], device="cuda")
        g, h = torch.tensor([0.5, 0.25, -2.0], device="cuda"), torch.ones(3, device="cuda")
        _, H, lse, _, _ = capi.token_logprobs(x, tokens, temperature=T)
        assert lse[0] == -INF and lse[2] == -INF
        want = torch.zeros(3, V, dtype=x.dtype, device="cuda")
        want[0, 1], want[2, V - 1] = 0.5 / T, -2.0 / T
        for entropy in (None, h):
            assert torch.equal(capi.token_logprobs_bwd(x, tokens, lse, H, g, entropy, temperature=T), want)
        capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T, out=x)
        assert torch.equal(x, want)
