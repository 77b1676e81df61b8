"""GPU: log probabilities of given tokens, distillation from a teacher's top logits and the embedding gradient by sorted
tokens against plain implementations in 64 bits.

Tolerances come from counting roundings, with u = 2^-24 for fp32:
  * 2^d by the hardware: relative 2^-22 = 4u; d = c (x - m): two roundings and the constant, 3u |d|;
  * a sum of V positive terms, at most V / 256 + 64 of them one after the other in a thread and the rest in a tree:
    relative (V / 256 + 64) u  -- called `chain` below, with the 4u above inside the 64;
  * results in 16 bits: half a step, finfo(t).eps / 2 relative, and half the smallest subnormal.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


@pytest.fixture(scope="module")
def capi(built):
    from opennn_b200 import capi as module
    module.lib()
    return module


def chain(V):
    return (V / 256 + 64) * U


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(dtype):
    if dtype is torch.float32:
        return 0.0, 0.0
    info = torch.finfo(dtype)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def make_logits(rows, V, dtype, pitch=None, offset=0, seed=0, spread=3.0):
    """[rows, V] with a row pitch, starting `offset` elements into its buffer.  Everything around the logits is NaN."""
    pitch = V if pitch is None else pitch
    buffer = torch.full((offset + rows * pitch + 64,), math.nan, dtype=TYPES[dtype], device="cuda")
    x = buffer[offset:offset + rows * pitch].view(rows, pitch)[:, :V]
    x.copy_(torch.randn(rows, V, generator=generator(seed), device="cuda") * spread)
    return x


def make_tokens(rows, V, seed=1, padding=True):
    t = torch.randint(1, V, (rows,), generator=generator(seed), device="cuda").float()
    if padding and rows > 2:
        t[1] = 0.0
        t[rows // 2] = V          # outside: padding too
    return t


def active_rows(tokens, V):
    t = tokens.long()
    return (t > 0) & (t < V)


def reference_logprobs(x, tokens, top, T):
    """As documented, in 64 bits.  Also returns m, E|d| for the tolerances."""
    rows, V = x.shape
    z = x.double() / T
    lse = torch.logsumexp(z, 1)
    none = (x == -INF).all(1)
    # relative to the largest logit: at the type's lowest value lse itself cannot tell log V from nothing, even in 64 bits
    logp = torch.where(none[:, None], torch.full_like(z, -INF), torch.log_softmax(z, 1))
    p = logp.exp()
    H = -torch.where(p > 0, p * logp, 0.0).sum(1) + 0.0 * p.sum(1)
    lse = torch.where(none, torch.full_like(lse, -INF), lse)
    broken = torch.isnan(x).any(1) | (x == INF).any(1)
    for v in (lse, H):
        v[broken] = math.nan
    logp[broken] = math.nan
    active = torch.ones(rows, dtype=torch.bool, device="cuda") if tokens is None else active_rows(tokens, V)
    t = torch.where(active, tokens.long(), 0) if tokens is not None else torch.zeros(rows, dtype=torch.long, device="cuda")
    given = logp.gather(1, t[:, None])[:, 0]
    zero = torch.zeros_like(lse)
    ids = torch.full((rows, top), -1, dtype=torch.int32, device="cuda")
    values = torch.full((rows, top), -INF, dtype=torch.float64, device="cuda")
    if top:
        k = min(top, V)
        clean = torch.where(torch.isnan(x), torch.full_like(x, -INF), x).double()
        order = torch.sort(clean, dim=1, descending=True, stable=True).indices[:, :k]
        there = (clean.gather(1, order) > -INF) & active[:, None]
        ids[:, :k] = torch.where(there, order, -1).int()
        values[:, :k] = torch.where(there, logp.gather(1, order), -INF)
    reach = torch.where(p > 0, p * (z - z.amax(1, keepdim=True)).abs(), 0.0).sum(1).nan_to_num(0.0)
    return (torch.where(active, given, zero), torch.where(active, H, zero), torch.where(active, lse, zero), ids, values, reach)


def check_close(got, want, tol, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    special = ~torch.isfinite(want)
    assert torch.equal(got[special].nan_to_num(7.0), want[special].nan_to_num(7.0)), what + ": infinities differ"
    tol = torch.as_tensor(tol, device="cuda", dtype=torch.float64).expand_as(want)
    off = (got - want).abs()[~special] - tol[~special]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: over the tolerance by {off.max().item():.3e}"


def check_logprobs(capi, x, tokens, top, T):
    V = x.shape[1]
    got = capi.token_logprobs(x, tokens, top=top, temperature=T)
    given, H, lse, ids, values, reach = reference_logprobs(x, tokens, top, T)
    rel = chain(V) + 4 * U * reach                      # of the sum
    if tokens is not None:
        check_close(got[0], given, rel + 6 * U * (given.abs().nan_to_num(0, 0, 0) + reach + 1), "logprob")
    else:
        assert got[0] is None
    check_close(got[1], H, (rel + 8 * U) * (2 + 2 * reach + H.abs().nan_to_num(0.0)), "entropy")
    # lse also rounds z of the largest logit: the temperature's reciprocal and the sum
    z_max = (x.double().amax(1) / T).nan_to_num(0, 0, 0).abs()
    check_close(got[2], lse, rel + 4 * U * (lse.abs().nan_to_num(0, 0, 0) + z_max + 1), "lse")
    if top:
        assert torch.equal(got[3], ids), "top ids"
        check_close(got[4], values, rel[:, None] + 6 * U * (values.abs().nan_to_num(0, 0, 0) + 1 + reach[:, None]), "top values")
    return got


SHAPES = [(1, 2), (3, 3), (5, 7), (4, 31), (7, 255), (3, 1000), (9, 1023), (5, 1024), (2, 4097), (33, 8000), (3, 32000), (2, 50021), (1, 131072),
          (700, 515), (1, 300001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
def test_token_logprobs(capi, rows, V, dtype):
    x = make_logits(rows, V, dtype, seed=V)
    tokens = make_tokens(rows, V)
    for top, T in ((0, 1.0), (1, 0.7), (5, 1.0), (20, 2.0), (64, 1.0), (128, 1.0)):
        check_logprobs(capi, x, tokens, top, T)
    check_logprobs(capi, x, None, 9, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(5000, 301), (4000, 2047), (620, 9001), (640, 1500), (400, 60000)])
def test_token_logprobs_many_rows(capi, rows, V, dtype):
    """Rows enough to fill the GPU: one CTA or warp each, several rows one after the other in the same warp."""
    x = make_logits(rows, V, dtype, pitch=V + 2, seed=V)
    x[::7] = (x[::7] * 2).round() / 2                     # ties
    x[3::11] = 1.5                                        # all equal
    x[5::13, V // 3:] = -INF
    tokens = make_tokens(rows, V)
    tokens[rows // 3: rows // 3 + 50] = 0.0
    for top in (0, 7, 64, 128):
        check_logprobs(capi, x, tokens, top, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch,offset", [(0, 1), (1, 0), (5, 3), (64, 7), (3, 2)])
@pytest.mark.parametrize("V", [6, 77, 4100, 20011])
def test_token_logprobs_strides(capi, V, pitch, offset, dtype):
    x = make_logits(6, V, dtype, pitch=V + pitch, offset=offset, seed=3)
    check_logprobs(capi, x, make_tokens(6, V), 8, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 1500, 9001, 40000])
def test_token_logprobs_orders_and_masks(capi, V, dtype):
    """Rows on which a search for the largest goes wrong most easily."""
    lowest = torch.finfo(TYPES[dtype]).min
    rows = 16
    x = make_logits(rows, V, dtype, seed=11)
    i = torch.arange(V, device="cuda")
    x[0] = 0.0                                            # all equal
    x[2] = lowest                                         # all at the type's lowest value
    x[3] = -INF                                           # nothing left
    x[4] = (i.float() / V * 20 - 10).to(x.dtype)          # rising
    x[5] = (10 - i.float() / V * 20).to(x.dtype)          # falling
    x[6] = torch.where(i % 7 == 3, x[6], torch.full_like(x[6], -INF))
    x[7] = torch.where(i == V - 1, x[7], torch.full_like(x[7], -INF))      # one token left
    x[8] = torch.where(i < V // 2, x[8], torch.full_like(x[8], lowest))
    x[9] = torch.where(i % 1024 < 4, torch.full_like(x[9], 9.0), x[9])     # ties in places a stride apart
    x[10] = (x[10] * 2).round() / 2                       # ties everywhere
    x[11, V // 3] = math.nan
    x[12, V // 2] = INF
    x[13] = torch.where(i % 2 == 0, 0.0, -0.0).to(x.dtype)                 # equal zeros
    x[14] = torch.where(i >= V - 40, torch.full_like(x[14], 12.0), torch.full_like(x[14], -12.0))
    x[15, 0] = torch.finfo(TYPES[dtype]).max if dtype == "f32" else 60000.0
    tokens = torch.full((rows,), float(V - 1), device="cuda")
    tokens[1] = 0.0
    tokens[5] = 1.0
    for top in (1, 20, 128):
        check_logprobs(capi, x, tokens, top, 1.0)


def test_token_logprobs_many_ties_past_any_list(capi):
    """More equal logits than a candidate list could hold, in the middle of the vocabulary; the order is that of the index."""
    x = torch.full((3, 60000), -5.0, device="cuda")
    x[0, 20000:50000] = 3.0
    x[1, 59000:] = 3.0
    x[2, ::3] = 3.0
    check_logprobs(capi, x, None, 128, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_runs_of_nan(capi, dtype):
    """Stretches of NaN: the values are NaN, the ids those of the other logits in order."""
    x = make_logits(4, 30000, dtype, seed=8)
    x[0, 64:128] = math.nan
    x[1, :29000] = math.nan
    x[2] = math.nan
    x[3, ::2] = math.nan
    for top in (1, 3, 50, 128):
        check_logprobs(capi, x, None, top, 1.0)


def test_token_logprobs_each_output_alone(capi):
    x, tokens = make_logits(5, 999, "f32"), make_tokens(5, 999)
    full = capi.token_logprobs(x, tokens, top=7)
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    for keep in range(4):
        out = [torch.full_like(t, 77) for t in full]
        use = [out[0] if keep == 0 else None, out[1] if keep == 1 else None, out[2] if keep == 2 else None]
        top = 7 if keep == 3 else 0
        capi.check(capi.lib().onn_token_logprobs(x.data_ptr(), 0, 999, tokens.data_ptr(), P(use[0]), P(use[1]), P(use[2]),
                                                 P(out[3]) if top else None, P(out[4]) if top else None, top, 5, 999, 1.0,
                                                 torch.cuda.current_stream().cuda_stream))
        for k, t in enumerate(out):
            written = k == keep or (keep == 3 and k >= 3)
            # entropy is summed by another kernel variant or not at all: the others' bits do not depend on it beyond rounding
            torch.testing.assert_close(t, full[k] if written else torch.full_like(t, 77), rtol=0 if t.dtype == torch.int32 else 2e-6, atol=0 if t.dtype == torch.int32 else 2e-6)


def test_token_logprobs_rows_past_32_bits(capi):
    """More than 2^31 logits, of which the padding leaves only the last rows: nothing else is read."""
    rows, V = 17000, 131072
    x = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, V, generator=generator(5), device="cuda")
    tokens = torch.zeros(rows, device="cuda")
    tokens[-3:] = torch.tensor([5.0, 131071.0, 70000.0], device="cuda")
    got = capi.token_logprobs(x, tokens, top=4)
    want = reference_logprobs(x[-3:], tokens[-3:], 4, 1.0)
    check_close(got[0][-3:], want[0], 1e-4, "logprob")
    assert torch.equal(got[3][-3:], want[3]) and (got[3][:-3] == -1).all() and (got[0][:-3] == 0).all()
    g = torch.ones(rows, device="cuda")
    capi.token_logprobs_bwd(x, tokens, got[2], got[1], g, out=x)
    assert (x[:-3] == 0).all()
    p = torch.exp(got[0][-3:].double())
    there = x[-3:].gather(1, tokens[-3:].long()[:, None])[:, 0].double()
    check_close(there, 1 - p, 2.0 ** -8, "gradient at the token")


# ---------------------------------------------------------------------------------------------------------------------

def reference_bwd(x, tokens, lse, H, g, h, T):
    """(gradient, tolerance) in 64 bits."""
    rows, V = x.shape
    active = active_rows(tokens, V)[:, None]
    t = torch.where(active[:, 0], tokens.long(), 0)[:, None]
    z = x.double() / T
    lse = lse.double()[:, None]
    logp = torch.where(lse == -INF, torch.full_like(z, -INF), z - lse)
    p = logp.exp()
    g = g.double()[:, None]
    hot = torch.zeros_like(z).scatter_(1, t, 1.0)
    dx = g * (hot - p)
    # log p: the temperature's reciprocal and one fused rounding; times log2 e; 2^d
    zf, lf = torch.where(p > 0, z, 0.0).abs(), torch.where(p > 0, logp, 0.0).abs()
    rel = (3 * zf + 4 * lf + 8) * U
    tol = g.abs() * p * rel + 4 * U * dx.abs()
    if h is not None:
        h, H = h.double()[:, None], H.double()[:, None]
        inner = torch.where(p > 0, logp, 0.0) + H
        dx = dx - h * p * inner
        tol = tol + h.abs() * p * (inner.abs() * rel + 6 * U * (zf + lf + H.abs()))
    eps, tiny = half_step(x.dtype)
    dx, tol = torch.where(active, dx / T, 0.0), torch.where(active, tol / T, 0.0)
    # 2^d below 2^-126 is flushed to zero
    return dx, tol * (1 + eps) + eps * dx.abs() + tiny + 2.0 ** -126 * (g.abs() + 1) / T


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 2), (5, 7), (4, 31), (3, 1000), (9, 1023), (33, 8000), (2, 50021), (1, 131072), (700, 515)])
def test_token_logprobs_bwd(capi, rows, V, dtype):
    for T, with_entropy, extra, offset in ((1.0, False, 0, 0), (0.7, True, 3, 1), (2.0, True, 0, 0)):
        x = make_logits(rows, V, dtype, pitch=V + extra, offset=offset, seed=V)
        if V > 1000:
            x[:, 5:300] = -INF
        tokens = make_tokens(rows, V)
        tokens = torch.where((tokens >= 5) & (tokens < 300), torch.ones_like(tokens), tokens) if V > 1000 else tokens
        _, H, lse, _, _ = capi.token_logprobs(x, tokens, temperature=T)
        gen = generator(9)
        g = torch.randn(rows, generator=gen, device="cuda")
        h = torch.randn(rows, generator=gen, device="cuda") if with_entropy else None
        want, tol = reference_bwd(x, tokens, lse, H, g, h, T)
        check_close(capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T), want, tol, "dlogits")
        # rows of another alignment than the logits', and what lies between them
        buffer = torch.full((rows * (V + 5) + 3,), 7.0, dtype=x.dtype, device="cuda")
        out = buffer[3:].view(rows, V + 5)[:, :V]
        check_close(capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T, out=out), want, tol, "dlogits, own pitch")
        assert (buffer[:3] == 7).all() and (buffer[3:].view(rows, V + 5)[:, V:] == 7).all()
        first = out.clone()
        around = x.as_strided((rows, V + extra), (V + extra, 1))[:, V:].clone()
        capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T, out=x)
        assert torch.equal(x, first), "in place"
        if extra:
            assert torch.isnan(around).all() and torch.isnan(x.as_strided((rows, V + extra), (V + extra, 1))[:, V:]).all()


def test_token_logprobs_bwd_against_differences(capi):
    rows, V, T = 6, 301, 1.3
    x, tokens = make_logits(rows, V, "f32"), make_tokens(rows, V)
    _, H, lse, _, _ = capi.token_logprobs(x, tokens, temperature=T)
    gen = generator(2)
    g, h = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    dx = capi.token_logprobs_bwd(x, tokens, lse, H, g, h, temperature=T).double()

    def loss(y):
        given, entropy, *_ = reference_logprobs(y, tokens, 0, T)
        return (given * g.double() + entropy * h.double()).sum()

    for seed in range(4):
        v = torch.randn(rows, V, generator=generator(20 + seed), device="cuda", dtype=torch.float64)
        e = 1e-4
        difference = (loss(x.double() + e * v) - loss(x.double() - e * v)) / (2 * e)
        # central differences leave e^2 / 6 of the third derivative, here below 50; the fp32 gradient its own roundings
        assert abs((dx * v).sum() - difference) <= 50 * e * e * rows + 200 * U * (dx * v).abs().sum()


# ---------------------------------------------------------------------------------------------------------------------

def make_teacher(rows, V, top, seed=4):
    gen = generator(seed)
    ids = torch.rand(rows, V, generator=gen, device="cuda").topk(min(top, V), dim=1).indices
    if top > V:
        ids = torch.cat([ids, torch.full((rows, top - V), -1, device="cuda")], 1)
    values = torch.randn(rows, top, generator=gen, device="cuda") * 2 - 3
    return ids.int(), values


def reference_distill(x, targets, ids, values, T, a, b):
    """(stats, losses, gradient, loss tolerance, gradient tolerance) in 64 bits."""
    rows, V = x.shape
    active = active_rows(targets, V)
    t = torch.where(active, targets.long(), 0)[:, None]
    count = active.sum().double()
    valid = (ids >= 0) & (ids < V)
    at = torch.where(valid, ids, 0).long()
    u = torch.where(valid, values.double() / T, -INF)
    taught = (u > -INF).any(1, keepdim=True) | torch.isnan(u).any(1, keepdim=True)
    q = torch.where(taught, torch.softmax(u, 1), 0.0)
    log_q = torch.log_softmax(u, 1)
    xd = x.double()
    none = (x == -INF).all(1, keepdim=True)
    logp = torch.where(none, torch.full_like(xd, -INF), torch.log_softmax(xd / T, 1))
    logp1 = torch.where(none, torch.full_like(xd, -INF), torch.log_softmax(xd, 1))
    p, p1 = logp.exp(), logp1.exp()
    terms = torch.where(q != 0, q * (log_q - logp.gather(1, at)), 0.0)
    soft = T * T * terms.sum(1)
    q_dense = torch.zeros_like(xd).scatter_add_(1, at, torch.where(valid, q, 0.0))
    dx = a * T * (p * taught.double() - q_dense) if a else torch.zeros_like(xd)
    hard = torch.zeros_like(soft)
    eps32 = torch.finfo(torch.float32).eps
    if b:
        hard = -torch.log(p1.gather(1, t)[:, 0] + eps32)
        dx = dx + b * (p1 - torch.zeros_like(xd).scatter_(1, t, 1.0))
    dx = torch.where(active[:, None], dx / max(count.item(), 1.0), 0.0)
    losses = torch.where(active, torch.stack([soft, hard]), 0.0)
    stats = torch.cat([losses.sum(1), count[None]])

    # roundings: q by exponent differences and one sum over the list; p by the chain and its exponent
    span = torch.where(valid & (u > -INF), (u - u.amax(1, keepdim=True)).abs(), 0.0).nan_to_num(0.0)
    rel_q = (4 * span.amax(1, keepdim=True) + ids.shape[1] + 16) * U
    reach = torch.where(p > 0, p * (xd / T - (xd / T).amax(1, keepdim=True)).abs(), 0.0).sum(1, keepdim=True).nan_to_num(0.0)
    reach1 = torch.where(p1 > 0, p1 * (xd - xd.amax(1, keepdim=True)).abs(), 0.0).sum(1, keepdim=True).nan_to_num(0.0)
    d = torch.where(p > 0, (xd - xd.amax(1, keepdim=True)).abs() / T, 0.0).nan_to_num(0.0)
    d1 = torch.where(p1 > 0, (xd - xd.amax(1, keepdim=True)).abs(), 0.0).nan_to_num(0.0)
    rel_p, rel_p1 = chain(V) + (4 * d + 4 * reach) * U, chain(V) + (4 * d1 + 4 * reach1) * U
    lq, lp = log_q.abs().nan_to_num(0, 0, 0), torch.where(q != 0, logp.gather(1, at), 0.0).abs().nan_to_num(0, 0, 0)
    soft_tol = T * T * ((q.nan_to_num(0.0) * (rel_q * (lq + lp + 2) + 8 * U * (lq + lp + 1) + chain(V) + 4 * U * reach)).sum(1)
                        + 8 * U * q.nan_to_num(0.0).sum(1))
    hard_tol = (rel_p1.gather(1, t)[:, 0] + 4 * U) * 2 + 4 * U * hard.abs().nan_to_num(0, 0, 0)
    scale = 1 / max(count.item(), 1.0)
    tol = scale * (abs(a) * T * (p * (rel_p + 8 * U) + q_dense.nan_to_num(0.0) * (rel_q + 8 * U)) + abs(b) * (p1 * (rel_p1 + 8 * U) + 8 * U * p1))
    if b:
        tol = tol + scale * abs(b) * 8 * U * torch.zeros_like(xd).scatter_(1, t, 1.0)
    eps, tiny = half_step(x.dtype)
    tol = tol * (1 + eps) + eps * dx.abs() + tiny + 2.0 ** -126 * scale * (abs(a) * T + abs(b) + 1)
    return stats, losses, dx, torch.stack([soft_tol, hard_tol]), tol


def check_distill(capi, x, targets, ids, values, T, a, b, out=None):
    want_stats, want_losses, want_dx, loss_tol, tol = reference_distill(x, targets, ids, values, T, a, b)
    stats, losses, dx = capi.distill3d(x, targets, ids, values, temperature=T, soft_weight=a, hard_weight=b, out=out)
    check_close(losses, want_losses, loss_tol, "losses")
    rows = x.shape[0]
    check_close(stats, want_stats, torch.cat([loss_tol.nan_to_num(0.0).sum(1) + (rows / 1024 + 24) * U * want_losses.abs().sum(1).nan_to_num(0, 0, 0),
                                              torch.zeros(1, device="cuda", dtype=torch.float64)]), "stats")
    check_close(dx, want_dx, tol, "gradient")
    return stats, losses, dx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 2), (5, 7), (4, 31), (3, 1000), (9, 1023), (5, 1025), (3, 4097), (2, 8193), (33, 8000), (5, 16384), (4, 16391),
                                    (3, 32000), (2, 50021), (3, 65537), (2, 131072), (1, 262147), (700, 515), (1, 530000)])
def test_distill(capi, rows, V, dtype):
    for top, T, a, b in ((1, 1.0, 1.0, 0.0), (8, 2.0, 0.5, 0.5), (64, 1.0, 0.3, 0.7), (128, 3.0, 1.0, 0.0), (5, 1.0, 0.0, 1.0), (16, 0.7, 0.5, 0.5)):
        if V > 100000 and top == 64:
            continue
        scale = 64.0 if dtype == "f16" else 1.0
        x = make_logits(rows, V, dtype, seed=V + top)
        ids, values = make_teacher(rows, V, top)
        check_distill(capi, x, make_tokens(rows, V), ids, values, T, a * scale, b * scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(3000, 300), (700, 5003), (320, 20000), (320, 36001), (160, 90000)])
def test_distill_many_rows(capi, rows, V, dtype):
    """Rows enough to fill the GPU, at the lengths where the number of threads changes."""
    x = make_logits(rows, V, dtype, seed=V)
    x[3::11] = 1.5
    x[5::13, V // 3:] = -INF
    targets = make_tokens(rows, V)
    targets[rows // 3: rows // 3 + 50] = 0.0
    scale = 1024.0 if dtype == "f16" else 1.0
    for top, T, a, b in ((12, 2.0, 0.5, 0.5), (128, 1.0, 0.5, 0.5), (30, 1.5, 0.7, 0.3)):
        ids, values = make_teacher(rows, V, top)
        # a teacher of tokens that the student keeps, or the loss is infinite
        ids = torch.where(ids >= V // 3, ids % (V // 3), ids)
        check_distill(capi, x, targets, ids, values, T, a * scale, b * scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra,offset", [(0, 1), (3, 0), (5, 2)])
@pytest.mark.parametrize("V", [9, 1001, 20011, 40005])
def test_distill_strides(capi, V, extra, offset, dtype):
    rows = 5
    targets = make_tokens(rows, V)
    ids, values = make_teacher(rows, V, 6)
    for in_place in (False, True):
        x = make_logits(rows, V, dtype, pitch=V + extra, offset=offset, seed=V)
        if in_place:
            keep = x.clone()
            stats, losses, dx = capi.distill3d(keep, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
            out = (torch.empty(3, device="cuda"), torch.empty(2, rows, device="cuda"), x)
            capi.distill3d(x, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5, out=out)
            # another alignment cuts the row elsewhere, which changes the order of the sums, not more
            eps = torch.finfo(x.dtype).eps if x.dtype is not torch.float32 else 2 * chain(V) + 64 * U
            torch.testing.assert_close(x, dx, rtol=eps, atol=torch.finfo(x.dtype).smallest_normal)
            if extra:
                assert torch.isnan(x.as_strided((rows, V + extra), (V + extra, 1))[:, V:]).all()
        else:
            buffer = torch.full((rows * (V + 7) + 1,), 7.0, dtype=x.dtype, device="cuda")
            out = (torch.empty(3, device="cuda"), torch.empty(2, rows, device="cuda"), buffer[1:].view(rows, V + 7)[:, :V])
            check_distill(capi, x, targets, ids, values, 2.0, 0.5, 0.5, out=out)
            assert buffer[0] == 7 and (buffer[1:].view(rows, V + 7)[:, V:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 9000, 40000])
def test_distill_lists_and_masks(capi, V, dtype):
    rows, top = 14, 9
    x = make_logits(rows, V, dtype, seed=6)
    targets = make_tokens(rows, V, padding=False)
    ids, values = make_teacher(rows, V, top)
    ids[1, 3], ids[1, 7] = ids[1, 0], ids[1, 0]                    # one token in three places
    ids[2, :] = -1                                                 # no teacher
    ids[3, ::2] = -1
    ids[4, 0], ids[4, 1] = V, 2 ** 31 - 1                          # outside
    values[5, 2:] = -INF                                           # listed with probability 0
    values[6, :] = -INF                                            # nothing but
    targets[7] = 0.0                                               # padding
    x[8] = -INF                                                    # a student with nothing left
    x[9, ids[9, 0].long()] = -INF                                  # a teacher's token masked
    targets[10] = ids[10, 4].float().clamp(min=1)                  # the target in the list
    ids[10, 4] = targets[10].int()
    x[11, targets[11].long()] = -INF                               # the target masked
    x[12] = torch.finfo(x.dtype).min                               # all at the type's lowest value
    ids[13, 0], values[13, 0] = ids[13, 1], 40.0                   # the likeliest token stands twice
    for T, a, b in ((1.0, 1.0, 0.0), (2.0, 0.5, 0.5), (1.0, 0.25, 0.75), (1.5, 0.5, 0.5)):
        check_distill(capi, x, targets, ids, values, T, a, b)
    # NaN and +inf stay in their rows
    x[0, V // 2], x[1, 1], values[3, 1] = math.nan, INF, math.nan
    stats, losses, dx = capi.distill3d(x, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    assert torch.isnan(losses[:, :2]).all() and torch.isnan(losses[0, 3]) and torch.isfinite(losses[1, 3])
    assert torch.isnan(dx[0]).all() and torch.isnan(dx[1]).all() and torch.isfinite(dx[4:8]).all() and torch.isfinite(dx[2]).all()


def test_distill_losses_alone_and_count_of_all_ranks(capi):
    rows, V, top = 40, 3000, 8
    x, targets = make_logits(rows, V, "f32"), make_tokens(rows, V)
    ids, values = make_teacher(rows, V, top)
    stats, losses, dx = capi.distill3d(x, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    alone = capi.distill3d(x, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5, want_gradient=False)
    assert alone[2] is None and torch.equal(alone[0], stats) and torch.equal(alone[1], losses)
    count = torch.tensor([2.0 * stats[2].item()], device="cuda")       # as if another rank had as many
    half = capi.distill3d(x, targets, ids, values, temperature=2.0, soft_weight=0.5, hard_weight=0.5, active_count=count)[2]
    torch.testing.assert_close(half, dx / 2, rtol=4 * U, atol=1e-30)
    # nothing but padding: zeros, and no division by zero
    stats, losses, dx = capi.distill3d(x, torch.zeros(rows, device="cuda"), ids, values)
    assert (stats == 0).all() and (losses == 0).all() and (dx == 0).all()


def test_distill_hard_part_is_the_cross_entropy(capi):
    """With the hard-label part alone the gradient is onn_ce3d_fwd_bwd's."""
    rows, V = 64, 8000
    x, targets = make_logits(rows, V, "f32"), make_tokens(rows, V)
    ids, values = make_teacher(rows, V, 4)
    stats, losses, dx = capi.distill3d(x, targets, ids, values, soft_weight=0.0, hard_weight=1.0)
    error, _, gradient, _ = capi.ce3d(x.clone(), targets)
    assert abs(stats[1].item() / stats[2].item() - error) <= 1e-5 * error
    p = torch.softmax(x.double(), 1)
    # both stay within their roundings of (p - onehot) / #active
    tol = 2 * (chain(V) + 100 * U) * (p + 1e-30) / stats[2].item() + 16 * U * gradient.abs()
    check_close(dx, gradient, tol, "gradient")


def test_distill_against_differences(capi):
    rows, V, top, T, a, b = 6, 301, 7, 1.7, 0.6, 0.4
    x, targets = make_logits(rows, V, "f32"), make_tokens(rows, V)
    ids, values = make_teacher(rows, V, top)
    dx = capi.distill3d(x, targets, ids, values, temperature=T, soft_weight=a, hard_weight=b)[2].double()

    def loss(y):
        stats = reference_distill(y, targets, ids, values, T, a, b)[0]
        return (a * stats[0] + b * stats[1]) / stats[2]

    for seed in range(4):
        v = torch.randn(rows, V, generator=generator(20 + seed), device="cuda", dtype=torch.float64)
        e = 1e-4
        difference = (loss(x.double() + e * v) - loss(x.double() - e * v)) / (2 * e)
        # FLT_EPSILON inside the hard-label logarithm is not in the gradient (as in the loss beside it): p / (p + eps) - 1
        share = (2.0 ** -23 / torch.softmax(x.double(), 1).gather(1, targets.long().clamp(0, V - 1)[:, None])).amax() * v.abs().amax() * 2
        assert abs((dx * v).sum() - difference) <= 50 * e * e + 200 * U * (dx * v).abs().sum() + b * share


# ---------------------------------------------------------------------------------------------------------------------

def reference_embedding(ids, dY, dY2, V, scale, before):
    E = dY.shape[-1]
    t = ids.double().trunc().long().reshape(-1)
    live = (t > 0) & (t < V)
    g = dY.double().reshape(-1, E)[live]
    magnitude = g.abs()
    if dY2 is not None:
        other = dY2.double().reshape(-1, E)[live]
        g, magnitude = g + other, magnitude + other.abs()
    s = math.sqrt(E) if scale else 1.0
    zero = torch.zeros(V, E, dtype=torch.float64, device="cuda")
    dW = zero.index_add(0, t[live], g) * s
    size = zero.index_add(0, t[live], magnitude) * s
    terms = torch.bincount(t[live], minlength=V).double()[:, None]
    if before is not None:
        dW, size = dW + before.double(), size + before.double().abs()
    return dW, (terms + 6) * U * size + 1e-45             # each term and each partial sum is rounded once


def check_embedding(capi, ids, dY, V, scale=True, dY2=None, before=None):
    want, tol = reference_embedding(ids, dY, dY2, V, scale, before)
    E = dY.shape[-1]
    guard = torch.full((V * E + 64,), 3.0, device="cuda")
    dW = guard[:V * E].view(V, E)
    if before is not None:
        dW.copy_(before)
    got = capi.embedding_bwd_sorted(ids, dY, V, scale=scale, dY2=dY2, dW=dW, accumulate=before is not None)
    check_close(got, want, tol, "dW")
    assert (guard[V * E:] == 3).all()
    if before is not None:
        t = ids.long().reshape(-1)
        absent = torch.ones(V, dtype=torch.bool, device="cuda")
        absent[t[(t > 0) & (t < V)]] = False
        assert torch.equal(dW[absent], before[absent])
    first = got.clone()
    if before is not None:
        dW.copy_(before)
    again = capi.embedding_bwd_sorted(ids, dY, V, scale=scale, dY2=dY2, dW=dW, accumulate=before is not None)
    assert torch.equal(first, again), "the same inputs give the same bits"


def make_ids(B, S, V, kind, seed=0):
    gen = generator(seed)
    if kind == "uniform":
        ids = torch.randint(0, V, (B, S), generator=gen, device="cuda")
    elif kind == "zipf":
        ids = torch.exp(torch.rand(B, S, generator=gen, device="cuda") * math.log(V)).long().clamp(0, V - 1)
    elif kind == "one":
        ids = torch.full((B, S), V - 1, device="cuda")
    elif kind == "none":
        ids = torch.zeros(B, S, device="cuda")
    elif kind == "two":
        ids = torch.where(torch.rand(B, S, generator=gen, device="cuda") < 0.5, 1, V - 1)
    elif kind == "rising":
        ids = torch.arange(B * S, device="cuda").view(B, S) % V
    elif kind == "falling":
        ids = (B * S - torch.arange(B * S, device="cuda")).view(B, S) % V
    else:                                     # outside on both sides, and fractions that truncate
        ids = torch.randint(-3, V + 3, (B, S), generator=gen, device="cuda") + 0.5
        ids = torch.where(ids < 0, ids - 1, ids)
    return ids.float()


@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "none", "two", "rising", "falling", "outside"])
@pytest.mark.parametrize("B,S,E,V", [(1, 1, 1, 2), (2, 3, 5, 11), (4, 33, 64, 1000), (3, 700, 36, 70), (8, 129, 130, 301), (2, 2048, 1024, 5000)])
def test_embedding_bwd_sorted(capi, B, S, E, V, kind):
    gen = generator(B * S)
    ids = make_ids(B, S, V, kind)
    dY, dY2 = (torch.randn(B, S, E, generator=gen, device="cuda") for _ in range(2))
    before = torch.randn(V, E, generator=gen, device="cuda")
    check_embedding(capi, ids, dY, V)
    check_embedding(capi, ids, dY, V, scale=False, dY2=dY2, before=before)


@pytest.mark.parametrize("tokens,E,V,kind", [(5000, 8, 200000, "uniform"), (40000, 20, 3000, "zipf"), (140000, 12, 70000, "zipf"), (300000, 4, 400000, "uniform"),
                                             (300001, 3, 1000, "zipf"), (131072, 4, 2, "two"), (20000, 2052, 40000, "zipf"), (66000, 4, 65536, "rising")])
def test_embedding_bwd_sorted_sizes(capi, tokens, E, V, kind):
    ids = make_ids(1, tokens, V, kind)
    dY = torch.randn(1, tokens, E, generator=generator(1), device="cuda")
    check_embedding(capi, ids, dY, V, dY2=torch.randn(1, tokens, E, generator=generator(2), device="cuda"))
    check_embedding(capi, ids, dY, V, before=torch.randn(V, E, generator=generator(3), device="cuda"))


def test_embedding_bwd_sorted_agrees_with_embedding_bwd(capi):
    B, S, E, V = 8, 128, 256, 900
    ids, dY = make_ids(B, S, V, "zipf"), torch.randn(B, S, E, generator=generator(1), device="cuda")
    _, tol = reference_embedding(ids, dY, None, V, True, None)
    check_close(capi.embedding_bwd_sorted(ids, dY, V), capi.embedding_bwd(ids, dY, V), 2 * tol, "dW")


def test_embedding_bwd_sorted_large_addresses(capi):
    """dY and dW of more than 2^32 bytes each; few positions are not padding."""
    S, E, V = 530000, 2052, 600000
    ids = torch.zeros(1, S, device="cuda")
    at = torch.tensor([0, 7, 300000, S - 2, S - 1], device="cuda")
    ids[0, at] = torch.tensor([V - 1.0, 5.0, V - 1.0, 590000.0, V - 1.0], device="cuda")
    dY = torch.empty(1, S, E, device="cuda")
    dY[0, at] = torch.randn(5, E, generator=generator(1), device="cuda")
    dW = torch.empty(V, E, device="cuda")
    capi.embedding_bwd_sorted(ids, dY, V, dW=dW)
    s = math.sqrt(E)
    torch.testing.assert_close(dW[V - 1], (dY[0, 0] + dY[0, 300000] + dY[0, S - 1]) * s, rtol=1e-5, atol=1e-4)
    torch.testing.assert_close(dW[590000], dY[0, S - 2] * s, rtol=1e-6, atol=0)
    torch.testing.assert_close(dW[5], dY[0, 7] * s, rtol=1e-6, atol=0)
    assert dW.count_nonzero(1).count_nonzero() == 3


# ---------------------------------------------------------------------------------------------------------------------

def run_chain(capi, embedding, projection, teacher_projection, ids, targets, T=2.0, top=6):
    """A tied pair of token networks (lookup, projection to logits) as a training program would step it: the teacher's list, the
    student's distillation loss, and the gradients of the student's projection and table."""
    B, S = ids.shape
    V, E = embedding.shape
    hidden = capi.embedding_fwd(ids, embedding, torch.zeros(S, E, device="cuda"), scale=True, add_pe=False)
    teacher_logits = capi.dense_fwd(hidden, teacher_projection, torch.zeros(V, device="cuda"), "Linear")
    _, _, _, top_ids, top_logprobs = capi.token_logprobs(teacher_logits.view(B * S, V), top=top)
    logits = capi.dense_fwd(hidden, projection, torch.zeros(V, device="cuda"), "Linear")
    stats, losses, gradient = capi.distill3d(logits, targets, top_ids, top_logprobs, temperature=T, soft_weight=0.5, hard_weight=0.5)
    dX, dW, _ = capi.dense_bwd(hidden, projection, logits, gradient, "Linear")
    table = capi.embedding_bwd_sorted(ids, dX, V)
    score = capi.token_logprobs(logits, targets)[0]
    return stats, dW, table, score, top_ids


def chain_inputs(seed=0, B=4, S=16, E=64, V=512):
    gen = generator(seed)
    embedding = torch.randn(V, E, generator=gen, device="cuda") / math.sqrt(E)
    projection, teacher = (torch.randn(E, V, generator=gen, device="cuda") / math.sqrt(E) for _ in range(2))
    ids = torch.randint(1, V, (B, S), generator=gen, device="cuda").float()
    targets = torch.randint(1, V, (B, S), generator=gen, device="cuda").float()
    ids[1, 9:], targets[1, 9:] = 0.0, 0.0
    return embedding, projection, teacher, ids, targets


def test_the_operators_together(capi):
    embedding, projection, teacher, ids, targets = chain_inputs()
    V, E = embedding.shape
    T, top = 2.0, 6
    stats, dW, table, score, top_ids = run_chain(capi, embedding, projection, teacher, ids, targets)

    W, P = embedding.double().requires_grad_(), projection.double().requires_grad_()
    hidden = W[ids.long()] * math.sqrt(E)
    logits = (hidden @ P).view(-1, V)
    active = targets.view(-1) > 0
    with torch.no_grad():
        # the list itself is checked elsewhere; two teachers' logits within tf32 rounding of one another may change places
        teacher_logp = torch.log_softmax((hidden @ teacher.double()).view(-1, V), 1)
        q = torch.softmax(teacher_logp.gather(1, top_ids.long()) / T, 1)
    logp = torch.log_softmax(logits / T, 1).gather(1, top_ids.long())
    soft = (T * T * (q * (q.log() - logp)).sum(1))[active].sum()
    given = torch.log_softmax(logits, 1).gather(1, targets.view(-1, 1).long())[:, 0]
    hard = -given[active].sum()
    ((0.5 * soft + 0.5 * hard) / active.sum()).backward()
    from tests.util import TOL, assert_close
    host = lambda t: t.detach().cpu().numpy()  # noqa: E731
    assert_close(host(stats), host(torch.stack([soft, hard, active.sum().double()])), TOL, "stats")
    assert_close(host(score), host(torch.where(active, given, 0.0)), TOL, "score")
    assert_close(host(dW), host(P.grad), TOL, "projection gradient")
    expected = W.grad.clone()
    expected[0] = 0.0                                     # padding trains nothing
    assert_close(host(table), host(expected), TOL, "table gradient")


def test_on_another_stream_and_in_graphs(capi):
    """The same values on a stream of its own, and from a captured graph whose inputs change between replays; a second graph
    and an eager call in between do not disturb the first."""
    a, b = chain_inputs(0), chain_inputs(1)
    want = [[t.clone() for t in run_chain(capi, *inputs)] for inputs in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_chain(capi, *a)
    side.synchronize()
    # the projections accumulate with atomics where a reduction is split: compare to rounding
    for x, y in zip(got, want[0]):
        torch.testing.assert_close(x, y, rtol=1e-4, atol=1e-6)

    held = [t.clone() for t in a]
    graphs, results = [], []
    for inputs in (held, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run_chain(capi, *inputs))
        graphs.append(graph)
    for turn in (0, 1, 0):
        for t, new in zip(held, (a, b)[turn]):
            t.copy_(new)
        graphs[0].replay()
        graphs[1].replay()
        run_chain(capi, *a)
        torch.cuda.synchronize()
        for x, y in zip(results[0], want[turn]):
            torch.testing.assert_close(x, y, rtol=1e-4, atol=1e-6)
        for x, y in zip(results[1], want[1]):
            torch.testing.assert_close(x, y, rtol=1e-4, atol=1e-6)


def test_two_streams_at_once(capi):
    """Calls of one operator in flight on two streams share nothing."""
    V, rows = 20011, 64
    x = [make_logits(rows, V, "f32", seed=s) for s in (1, 2)]
    t = make_tokens(rows, V)
    ids, values = make_teacher(rows, V, 16)
    tokens = [make_ids(1, 9000, 400, "zipf", seed=s) for s in (1, 2)]
    dY = torch.randn(1, 9000, 64, generator=generator(3), device="cuda")

    def step(k):
        return (*capi.token_logprobs(x[k], t, top=20), *capi.distill3d(x[k], t, ids, values, temperature=2.0), capi.embedding_bwd_sorted(tokens[k], dY, 400))

    want = [step(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(k))
    torch.cuda.synchronize()
    for k in range(2):
        for result in got[k]:
            for p, q in zip(result, want[k]):
                assert torch.equal(p, q)


@pytest.mark.parametrize("kind", ["transformer", "decoder"])
def test_trainer_scores_tokens(capi, kind):
    """The trainer's scores are the logarithms of the probabilities that its inference pass leaves in the output layer."""
    from opennn_b200 import trainer
    S_in, S_dec, V, B = 24, 16, 320, 4
    decoder_only = kind == "decoder"
    t = trainer.Trainer(trainer.DECODER_ONLY if decoder_only else trainer.TRANSFORMER, S_dec if decoder_only else S_in, S_dec, V, V, 128, 2, 256, 1, B)
    try:
        import numpy as np
        rng = np.random.default_rng(3)
        t.set_parameters((rng.standard_normal(t.parameters_number) * 0.08).astype(np.float32))
        gen = generator(4)
        dec, tgt = (torch.randint(1, V, (B, S_dec), generator=gen, device="cuda").float() for _ in range(2))
        enc = None if decoder_only else torch.randint(1, V, (B, S_in), generator=gen, device="cuda").float()
        tgt[1, 9:] = 0.0
        given, entropy, ids, values = t.token_logprobs(dec, enc, tgt, top=5)
        t.forward(dec, enc, is_training=False)
        p = torch.from_numpy(t.layer_output(t.layers_number - 1)).cuda().view(B, S_dec, V).double()
        active = tgt > 0
        logp = p.log()
        want = torch.where(active, logp.gather(2, tgt.long()[..., None])[..., 0], 0.0)
        # the probabilities are rounded to fp32, after an exponential and a division of their own
        torch.testing.assert_close(given.double(), want, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(entropy.double(), torch.where(active, -(p * logp).sum(2), 0.0), rtol=1e-5, atol=1e-5)
        assert torch.equal((ids == -1).all(2), ~active)
        torch.testing.assert_close(values[active].double(), p.topk(5, dim=2).values.log()[active], rtol=1e-5, atol=1e-5)
        _, all_entropy, _, _ = t.token_logprobs(dec, enc)
        assert (all_entropy > 0).all()
        with pytest.raises(capi.OnnError):
            t.token_logprobs(dec, enc, tgt, top=500)
        with pytest.raises(capi.OnnError):
            t.token_logprobs(dec[:2], enc, tgt)
    finally:
        t.close()


def test_wrapper_refusals(capi):
    x = torch.zeros(4, 10, device="cuda")
    t = torch.ones(4, device="cuda")
    for call in (lambda: capi.token_logprobs(x, t[:3]), lambda: capi.token_logprobs(x, t.long()), lambda: capi.token_logprobs(x.t(), t),
                 lambda: capi.token_logprobs(x, t, top=200), lambda: capi.token_logprobs(x, t, temperature=0.0),
                 lambda: capi.token_logprobs(x.view(2, 2, 10).transpose(0, 1), t), lambda: capi.token_logprobs_bwd(x, t, t, t, t, out=x.half()),
                 lambda: capi.distill3d(x, t, torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, device="cuda")),
                 lambda: capi.embedding_bwd_sorted(t, torch.zeros(2, 3, 8, device="cuda"), 10)):
        with pytest.raises(capi.OnnError):
            call()


def test_trainer_refuses_ids_that_are_not_floats(capi):
    from opennn_b200 import trainer
    t = trainer.Trainer(trainer.DECODER_ONLY, 16, 16, 320, 320, 128, 2, 256, 1, 4)
    try:
        ids = torch.ones(4, 16, device="cuda")
        for call in (lambda: t.token_logprobs(ids, None, ids.long()), lambda: t.token_logprobs(ids.int(), None, ids),
                     lambda: t.token_logprobs(ids, None, torch.ones(16, 4, device="cuda").t()), lambda: t.token_logprobs(ids.cpu(), None, ids)):
            with pytest.raises(capi.OnnError):
                call()
        t.token_logprobs(ids, None, ids)
        torch.cuda.synchronize()
    finally:
        t.close()


@pytest.mark.parametrize("E", [3, 5, 14, 17, 62, 66, 130, 793])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_embedding_bwd_sorted_writes_every_absent_row(capi, E, offset):
    """Rows of any length and alignment that do not occur: all of their elements, and nothing around the table."""
    V, n = 4000, 2100
    gen = generator(E)
    room = torch.full((V * E + 8,), 7.0, device="cuda")
    dW = room[offset:offset + V * E].view(V, E)
    ids = torch.randint(1, 60, (1, n), generator=gen, device="cuda").float() * 50
    dY = torch.randn(1, n, E, generator=gen, device="cuda")
    capi.embedding_bwd_sorted(ids, dY, V, dW=dW)
    want = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1).long(), dY[0].double()) * math.sqrt(E)
    absent = torch.ones(V, dtype=torch.bool, device="cuda")
    absent[ids.view(-1).long()] = False
    assert (dW[absent] == 0).all()
    size = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1).long(), dY[0].double().abs()) * math.sqrt(E)
    count = torch.bincount(ids.view(-1).long(), minlength=V)[:, None]
    # at most count + 2 roundings, each of at most half a step of a partial sum that the sum of the sizes bounds
    assert ((dW.double() - want).abs() <= (count + 2) * 2.0 ** -24 * size).all()
    assert (room[:offset] == 7).all() and (room[offset + V * E:] == 7).all()


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("two", [False, True])
def test_embedding_bwd_sorted_small_tables_of_repeated_ids(capi, two, accumulate):
    """The kernel for few positions with runs of equal ids, both inputs and earlier values."""
    V, n, E = 90, 2048, 70
    gen = generator(11)
    ids = torch.where(torch.rand(1, n, generator=gen, device="cuda") < 0.5, torch.tensor(5.0, device="cuda"),
                      torch.randint(0, V, (1, n), generator=gen, device="cuda").float())
    dY, dY2 = (torch.randn(1, n, E, generator=gen, device="cuda") for _ in range(2))
    before = torch.randn(V, E, generator=gen, device="cuda")
    dW = before.clone()
    capi.embedding_bwd_sorted(ids, dY, V, dY2=dY2 if two else None, dW=dW, accumulate=accumulate)
    g = dY[0].double() + (dY2[0].double() if two else 0.0)
    want = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1).long(), g)
    size = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, ids.view(-1).long(), g.abs()) * math.sqrt(E)
    want, count = want * math.sqrt(E), torch.bincount(ids.view(-1).long(), minlength=V)[:, None]
    want[0] = 0
    size[0] = 0
    if accumulate:
        want, size = want + before.double(), size + before.double().abs()
    # at most count + 4 roundings, each of at most half a step of a partial sum that the sum of the sizes bounds
    assert ((dW.double() - want).abs() <= (count + 4) * 2.0 ** -24 * size + 1e-30).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 650])
@pytest.mark.parametrize("V", [100, 130, 257, 300, 520, 700, 1000, 1030, 1300, 1600, 2050, 2600])
def test_token_logprobs_long_lists_of_short_rows(capi, rows, V, dtype):
    """Lists as long as a row has vectors or longer: the warps of a row have different numbers of vectors, some none."""
    x = make_logits(rows, V, dtype, pitch=V + 3, offset=1, seed=V)
    x[::5] = (x[::5] * 2).round() / 2
    x[2::9, : V - V // 16] = -INF
    tokens = make_tokens(rows, V)
    for top in (3, 20, 24, 25, 33, 64, 65, 100, 128):
        check_logprobs(capi, x, tokens, top, 1.0)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("E", [100004, 100001])
def test_embedding_bwd_sorted_very_wide_rows(capi, E, accumulate):
    """More column blocks than the kernel that joins runs has CTAs; one long run, several short ones."""
    V, n = 40, 200
    gen = generator(E)
    ids = torch.randint(1, V, (1, n), generator=gen, device="cuda").float()
    ids[0, 20:150] = 7.0
    ids[0, 150:175] = 9.0
    dY = torch.randn(1, n, E, generator=gen, device="cuda")
    before = torch.randn(V, E, generator=gen, device="cuda")
    dW = before.clone()
    capi.embedding_bwd_sorted(ids, dY, V, dW=dW, accumulate=accumulate)
    index = ids.view(-1).long()
    want = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, index, dY[0].double()) * math.sqrt(E)
    size = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, index, dY[0].double().abs()) * math.sqrt(E)
    if accumulate:
        want, size = want + before.double(), size + before.double().abs()
    count = torch.bincount(index, minlength=V)[:, None]
    # at most count + 3 roundings (with the scale's own and the earlier value's), each of at most half a step of a partial sum
    assert ((dW.double() - want).abs() <= (count + 3) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("two", [False, True])
def test_embedding_bwd_sorted_same_bits_at_any_alignment(capi, two):
    B, S, E, V = 8, 600, 132, 900
    gen = generator(5)
    ids = torch.exp(torch.rand(B, S, generator=gen, device="cuda") * math.log(V)).floor().clamp(1, V - 1)
    dY, dY2 = (torch.randn(B, S, E, generator=gen, device="cuda") for _ in range(2))
    aligned = capi.embedding_bwd_sorted(ids, dY, V, dY2=dY2 if two else None)
    room = torch.empty(dY.numel() + 1, device="cuda")
    moved = room[1:].view(B, S, E)
    moved.copy_(dY)
    assert torch.equal(capi.embedding_bwd_sorted(ids, moved, V, dY2=dY2 if two else None), aligned)
