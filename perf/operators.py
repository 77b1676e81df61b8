"""The operators at the vocabulary end of a token network, as cases that can be timed and compared.

score      log probability of a given token in each row of logits, entropy, log-sum-exp and the top alternatives
score_bwd  the gradient of log probability and entropy with respect to the logits
distill    distillation from a teacher's top logits mixed with the hard-label cross entropy: loss and gradient
embed      gradient of the embedding table, summed by token in order of position

`own` chooses between the plain form (elementary torch operations) and the library's entry points.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
LOSS_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 4096.0}      # gradients held in fp16 would otherwise fall below its range
EPSILON = 1.1920928955078125e-07        # FLT_EPSILON, the constant inside the hard-label term


def _score(name, rows, V, dtype, top, **more):
    return {"name": name, "op": "score", "rows": rows, "V": V, "dtype": dtype, "top": top, "temperature": 1.0, "pitch": V,
            "padding": False, "tokens": True, "banned": False, **more}


def _score_bwd(name, rows, V, dtype, **more):
    return {"name": name, "op": "score_bwd", "rows": rows, "V": V, "dtype": dtype, "temperature": 1.0, "padding": False,
            "entropy": True, **more}


def _distill(name, rows, V, dtype, top, **more):
    return {"name": name, "op": "distill", "rows": rows, "V": V, "dtype": dtype, "top": top, "temperature": 2.0, "soft": 0.5,
            "hard": 0.5, "padding": True, **more}


def _embed(name, B, S, E, V, **more):
    return {"name": name, "op": "embed", "B": B, "S": S, "E": E, "V": V, "ids": "uniform", "two": False, "padding": True,
            "accumulate": False, **more}


def listed():
    return [
        # one decoding position of eight sequences: log probability of the chosen token and five alternatives
        _score("score decode 8x32000", 8, 32000, "f32", 5),
        # one sequence, a long vocabulary in 16 bits, some tokens banned by -inf
        _score("score one row 131072 bf16", 1, 131072, "bf16", 20, banned=True),
        # evaluation of a micro-batch of 64 sequences of 256 with padding: no alternatives wanted
        _score("score evaluate 16384x32000", 16384, 32000, "f32", 0, padding=True),
        # a teacher writes down its 64 best tokens for each position; vocabulary of odd size in a padded buffer
        _score("score teacher 8192x50021 bf16", 8192, 50021, "bf16", 64, tokens=False, pitch=50048),
        # policy-gradient step over 32 sequences of 256 with an entropy bonus
        _score_bwd("score_bwd 8192x32000", 8192, 32000, "f32", padding=True),
        # the same in 16 bits over rows that start at odd places, likelihood only
        _score_bwd("score_bwd 2048x100003 f16", 2048, 100003, "f16", entropy=False),
        # the tiny network's micro-batch
        _distill("distill 1024x1000", 1024, 1000, "f32", 8),
        # the large network's micro-batch: 64 sequences of 256
        _distill("distill 16384x32000", 16384, 32000, "f32", 32),
        # long vocabulary in 16 bits, soft targets alone at temperature one
        _distill("distill 4096x131072 bf16", 4096, 131072, "bf16", 64, temperature=1.0, soft=1.0, hard=0.0, padding=False),
        # embedding gradient of the tiny network
        _embed("embed 32x32 E64 V1000", 32, 32, 64, 1000),
        # embedding gradient of the large network's micro-batch
        _embed("embed 64x256 E1024 V32000", 64, 256, 1024, 32000),
        # a long batch of natural text: a few tokens make up much of it; two consumers of the embedding's output
        _embed("embed 128x1024 E1024 V50021", 128, 1024, 1024, 50021, ids="zipf", two=True, padding=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["score", "score_bwd", "distill", "embed"])
    if op == "embed":
        B, E, V = _spread(rng, 1, 256), 4 * _spread(rng, 8, 256) + rng.choice([0, 0, 0, 1, 2]), _spread(rng, 500, 130000)
        S = _spread(rng, 1, max(1, min(1024, 130000 // B)))
        return {"op": op, "B": B, "S": S, "E": E, "V": V, "ids": rng.choice(["uniform", "zipf"]), "two": rng.random() < 0.3,
                "padding": rng.random() < 0.7, "accumulate": rng.random() < 0.3}
    V = _spread(rng, 500, 200000)
    rows = _spread(rng, 1, max(1, min(16384, 500_000_000 // V)))
    case = {"op": op, "rows": rows, "V": V, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]), "padding": rng.random() < 0.5}
    if op == "score":
        tokens = rng.random() < 0.8
        case |= {"top": rng.choice([0, 1, 5, 20, 64, 128]), "pitch": V + rng.choice([0, 0, 5, 64]),
                 "tokens": tokens, "padding": tokens and case["padding"], "banned": rng.random() < 0.3}
    elif op == "score_bwd":
        case |= {"entropy": rng.random() < 0.5}
    else:
        hard, loss_scale = rng.choice([0.0, 0.5, 0.9]), LOSS_SCALE[case["dtype"]]
        case |= {"top": rng.choice([1, 8, 20, 32, 64, 128]), "soft": (1.0 - hard) * loss_scale, "hard": hard * loss_scale}
    return case


def _tokens(case, rows, V, g):
    """Token ids as the network holds them, floats with 0 for padding; the rows of a padded batch end after 1/4 .. 4/4 of 256 places."""
    t = torch.randint(1, V, (rows,), generator=g, device="cuda").float()
    if case["padding"]:
        place = torch.arange(rows, device="cuda")
        length = torch.randint(64, 257, (rows // 256 + 1,), generator=g, device="cuda")
        t = torch.where(place % 256 < length[place // 256], t, torch.zeros_like(t))
    return t


def _logits(case, rows, V, pitch, tokens, g):
    """Logits of a trained network: a bell of width two, a few likely tokens in each row, the given token often among them."""
    buffer = torch.empty(rows, pitch, dtype=DTYPES[case["dtype"]], device="cuda")
    step = max(1, (1 << 27) // pitch)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = torch.randn(n, pitch, generator=g, device="cuda") * 2.0
        likely = torch.randint(0, V, (n, 16), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand(n, 16, generator=g, device="cuda") * 9.0)
        own_token = tokens[r:r + n].long()[:, None]
        x.scatter_add_(1, own_token, torch.rand(n, 1, generator=g, device="cuda") * 12.0)
        if case.get("banned"):
            x[:, torch.randint(0, V, (V // 50 + 1,), generator=g, device="cuda")] = -math.inf
            x.scatter_(1, own_token, torch.randn(n, 1, generator=g, device="cuda") + 8.0)
        buffer[r:r + n] = x
    return buffer[:, :V]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "embed":
        B, S, E, V = case["B"], case["S"], case["E"], case["V"]
        if case["ids"] == "zipf":      # frequency of the v-th token ~ 1 / v
            u = torch.rand(B, S, generator=g, device="cuda", dtype=torch.float64)
            ids = torch.exp(u * math.log(V)).floor().clamp(1, V - 1)
            ids = torch.randperm(V - 1, generator=g, device="cuda")[ids.long() - 1] + 1
        else:
            ids = torch.randint(1, V, (B, S), generator=g, device="cuda")
        if case["padding"]:
            length = torch.randint((S + 3) // 4, S + 1, (B, 1), generator=g, device="cuda")
            ids = torch.where(torch.arange(S, device="cuda")[None] < length, ids, torch.zeros_like(ids))
        state["ids"] = ids.float()
        state["dY"] = torch.randn(B, S, E, generator=g, device="cuda") * 1e-3
        state["dY2"] = torch.randn(B, S, E, generator=g, device="cuda") * 1e-3 if case["two"] else None
        state["before"] = torch.randn(V, E, generator=g, device="cuda") * 1e-3 if case["accumulate"] else None
        state["dW"] = torch.empty(V, E, device="cuda")         # the table's part of the gradient arena
        return state

    rows, V = case["rows"], case["V"]
    tokens = _tokens(case, rows, V, g)
    state["tokens"] = tokens
    state["x"] = _logits(case, rows, V, case.get("pitch", V), tokens, g)
    if case["op"] == "score":
        if not case["tokens"]:
            state["tokens"] = None
        k = case["top"]
        state["out"] = (None if state["tokens"] is None else torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
                        torch.empty(rows, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda") if k else None,
                        torch.empty(rows, k, device="cuda") if k else None)
    elif case["op"] == "score_bwd":
        # what the forward pass kept
        lse, entropy = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        step = max(1, (1 << 26) // V)
        for r in range(0, rows, step):
            z = state["x"][r:r + step].double() / case["temperature"]
            l = torch.logsumexp(z, 1)
            lse[r:r + step] = l
            entropy[r:r + step] = l - (torch.exp(z - l[:, None]) * z).sum(1)
        state["lse"], state["entropy"] = lse, entropy
        each = LOSS_SCALE[case["dtype"]] / rows
        state["g"] = torch.randn(rows, generator=g, device="cuda") * each      # advantage over the number of tokens
        state["h"] = torch.full((rows,), -0.01 * each, device="cuda") if case["entropy"] else None
        state["out"] = torch.empty_like(state["x"])
    else:
        k = min(case["top"], V)
        # the teacher's list: distinct ids, values that fall off, some places unused in the padded batches
        first = torch.randint(0, V, (rows, 1), generator=g, device="cuda")
        ids = (first + torch.arange(k, device="cuda") * max(1, V // max(k, 1))) % V
        values = torch.randn(rows, k, generator=g, device="cuda").sort(1, descending=True).values * 3.0 - 4.0
        if case["padding"]:
            ids = torch.where(torch.rand(rows, k, generator=g, device="cuda") < 0.05, torch.full_like(ids, -1), ids)
        state["teacher_ids"], state["teacher"] = ids.int(), values
        state["out"] = (torch.empty(3, device="cuda"), torch.empty(2, rows, device="cuda"), torch.empty_like(state["x"]))
    return state


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------

def _active(tokens, rows, V):
    if tokens is None:
        return torch.ones(rows, dtype=torch.bool, device="cuda"), torch.zeros(rows, dtype=torch.long, device="cuda")
    t = tokens.long()
    active = (t > 0) & (t < V)
    return active, torch.where(active, t, torch.zeros_like(t))


def _plain_score(s):
    case, x = s["case"], s["x"].float()
    rows, V = x.shape
    active, t = _active(s["tokens"], rows, V)
    z = x / case["temperature"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1)
    lse = m[:, 0] + torch.log(total)
    d = torch.where(e > 0, z - m, 0.0)
    entropy = torch.log(total) - (e * d).sum(1) / total
    logprob = z.gather(1, t[:, None])[:, 0] - lse
    out = {"entropy": torch.where(active, entropy, 0.0), "lse": torch.where(active, lse, 0.0)}
    if s["tokens"] is not None:
        out["logprobs"] = torch.where(active, logprob, 0.0)
    k = min(case["top"], V)
    if k:
        # value first, then the lower index, in one whole number: equal logits stand in order of index
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = order * (1 << 32) + ((1 << 31) - torch.arange(V, device="cuda"))
        ids = torch.topk(key, k, dim=1).indices
        values = x.gather(1, ids)
        there = (values > -math.inf) & active[:, None]
        listed_ids = torch.full((rows, case["top"]), -1, dtype=torch.int32, device="cuda")
        listed_values = torch.full((rows, case["top"]), -math.inf, device="cuda")
        listed_ids[:, :k] = torch.where(there, ids, -1).int()
        listed_values[:, :k] = torch.where(there, z.gather(1, ids) - lse[:, None], -math.inf)
        out["top_ids"], out["top_logprobs"] = listed_ids, listed_values
    return out


def _plain_score_bwd(s):
    case, x = s["case"], s["x"].float()
    rows, V = x.shape
    active, t = _active(s["tokens"], rows, V)
    T = case["temperature"]
    logp = x / T - s["lse"][:, None]
    p = torch.exp(logp)
    dx = -s["g"][:, None] * p
    dx.scatter_add_(1, t[:, None], s["g"][:, None])
    if s["h"] is not None:
        dx = dx - s["h"][:, None] * p * (torch.where(p > 0, logp, 0.0) + s["entropy"][:, None])
    return {"dlogits": torch.where(active[:, None], dx / T, 0.0).to(s["x"].dtype)}


def _plain_distill(s):
    case, x = s["case"], s["x"].float()
    rows, V = x.shape
    T, a, b = case["temperature"], case["soft"], case["hard"]
    active, t = _active(s["tokens"], rows, V)
    count = active.sum().float()
    ids = s["teacher_ids"].long()
    there = (ids >= 0) & (ids < V)
    u = torch.where(there, s["teacher"] / T, -math.inf)
    top = u.amax(1, keepdim=True)
    e = torch.where(there, torch.exp(u - top), 0.0)
    q = torch.where(there.any(1, keepdim=True), e / e.sum(1, keepdim=True), 0.0)
    index = torch.where(there, ids, 0)

    m = x.amax(1, keepdim=True)
    z = (x - m) / T
    ez = torch.exp(z)
    total = ez.sum(1, keepdim=True)
    logp = z.gather(1, index) - torch.log(total)
    soft = T * T * torch.where(q > 0, q * (torch.log(q) - logp), 0.0).sum(1)
    has = there.any(1, keepdim=True).float()
    dx = (ez / total * has).scatter_add_(1, index, -q) * (a * T)
    hard = torch.zeros(rows, device="cuda")
    if b:
        e1 = torch.exp(x - m)
        p1 = e1 / e1.sum(1, keepdim=True)
        hard = -torch.log(p1.gather(1, t[:, None])[:, 0] + EPSILON)
        dx = dx + b * p1
        dx.scatter_add_(1, t[:, None], torch.full((rows, 1), -b, device="cuda"))
    losses = torch.where(active, torch.stack([soft, hard]), 0.0)
    dx = torch.where(active[:, None], dx / count, 0.0)
    # the sums over rows are long: 64 bits
    sums = losses.double().sum(1).float()
    return {"stats": torch.cat([sums, count[None]]), "losses": losses, "dlogits": dx.to(s["x"].dtype)}


def _plain_embed(s):
    case = s["case"]
    E, V = case["E"], case["V"]
    t = s["ids"].long().reshape(-1)
    active = (t > 0) & (t < V)
    dY = s["dY"] if s["dY2"] is None else s["dY"] + s["dY2"]
    dY = torch.where(active[:, None], dY.reshape(-1, E) * math.sqrt(E), 0.0)
    # a frequent token's sum has many terms, and its order would change from pass to pass: 64 bits
    dW = torch.zeros(V, E, dtype=torch.float64, device="cuda").index_add_(0, torch.where(active, t, 0), dY.double())
    if s["before"] is not None:
        dW = dW + s["before"]
    return {"dW": dW.float()}


# ---------------------------------------------------------------------------------------------------------------------
# the library's entry points
# ---------------------------------------------------------------------------------------------------------------------

def _own_run(s):
    from opennn_b200 import capi
    case = s["case"]
    if case["op"] == "score":
        logprobs, entropy, lse, top_ids, top_logprobs = capi.token_logprobs(
            s["x"], s["tokens"], top=case["top"], temperature=case["temperature"], out=s["out"])
        out = {"entropy": entropy, "lse": lse}
        if logprobs is not None:
            out["logprobs"] = logprobs
        if top_ids is not None:
            out["top_ids"], out["top_logprobs"] = top_ids, top_logprobs
        return out
    if case["op"] == "score_bwd":
        return {"dlogits": capi.token_logprobs_bwd(s["x"], s["tokens"], s["lse"], s["entropy"], s["g"], s["h"],
                                                   temperature=case["temperature"], out=s["out"])}
    if case["op"] == "distill":
        stats, losses, gradient = capi.distill3d(s["x"], s["tokens"], s["teacher_ids"], s["teacher"],
                                                 temperature=case["temperature"], soft_weight=case["soft"],
                                                 hard_weight=case["hard"], out=s["out"])
        return {"stats": stats, "losses": losses, "dlogits": gradient}
    if s["before"] is not None:
        s["dW"].copy_(s["before"])
    return {"dW": capi.embedding_bwd_sorted(s["ids"], s["dY"], case["V"], dY2=s["dY2"], dW=s["dW"], accumulate=case["accumulate"])}


def run(state):
    if own:
        return _own_run(state)
    plain = {"score": _plain_score, "score_bwd": _plain_score_bwd, "distill": _plain_distill, "embed": _plain_embed}
    return plain[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "embed":
        tokens, E, V = case["B"] * case["S"], case["E"], case["V"]
        live = tokens * (0.625 if case["padding"] else 1.0)
        # distinct tokens: expected for uniform ids; with frequencies ~ 1 / v, those with an expected count, summed smoothly
        if case["ids"] == "uniform":
            distinct = V * (1.0 - math.exp(-live / V))
        else:
            c = live / math.log(V)
            distinct = sum((1.0 - math.exp(-c / v)) * w for v, w in ((1.5 ** i, 1.5 ** i * 0.5) for i in range(int(math.log(V, 1.5)))))
        table = 2 * distinct if case["accumulate"] else V
        return {"bytes": 4.0 * tokens + 4.0 * live * E * (2 if case["two"] else 1) + 4.0 * table * E, "flops": live * E * (3.0 if case["two"] else 2.0)}
    rows, V, size = case["rows"], case["V"], BYTES[case["dtype"]]
    # a padded row is neither read nor computed: sequences fill 160 of 256 places on average; fewer rows are the start of one
    live = rows * (160 / 256 if rows >= 256 else min(1.0, (min(rows, 64) + max(0, rows - 64) * (1 - (rows - 64) / 386)) / rows)) if case["padding"] else rows
    if case["op"] == "score":
        return {"bytes": live * V * size + rows * (16.0 + 8 * case["top"]), "flops": 6.0 * live * V}
    if case["op"] == "score_bwd":
        return {"bytes": live * V * size + rows * (V * size + 20.0), "flops": (8.0 if case["entropy"] else 4.0) * live * V}
    return {"bytes": live * V * size + rows * (V * size + 12.0 + 8 * case["top"]), "flops": (12.0 if case["hard"] else 7.0) * live * V}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def _exact_rows(s, r, n):
    """The outputs of rows r .. r + n of a case over logits, from the definition."""
    case = s["case"]
    x = s["x"][r:r + n].double()
    V, T, n = x.shape[1], case["temperature"], x.shape[0]
    if s["tokens"] is None:
        live, t = x.new_ones(n), torch.zeros(n, dtype=torch.long, device="cuda")
    else:
        given = s["tokens"][r:r + n].double().trunc().long()
        live = ((given >= 1) & (given <= V - 1)).double()
        t = (given * live.long())
    logp = torch.log_softmax(x / T, 1)
    p = logp.exp()
    pick = torch.nn.functional.one_hot(t, V) if case["op"] != "score" else None
    if case["op"] == "score":
        lse = torch.logsumexp(x / T, 1)
        plogp = torch.special.entr(p)
        out = {"entropy": plogp.sum(1) * live, "lse": lse * live}
        if s["tokens"] is not None:
            out["logprobs"] = logp[torch.arange(n, device="cuda"), t] * live
        if case["top"]:
            k = min(case["top"], V)
            best = torch.full((n, case["top"]), -math.inf, dtype=torch.float64, device="cuda")
            best[:, :k] = torch.topk(logp, k, dim=1).values
            best[live == 0] = -math.inf
            out["top_logprobs"] = best
        return out
    if case["op"] == "score_bwd":
        kept = torch.exp(x / T - s["lse"][r:r + n].double()[:, None])     # lse and entropy are inputs of this pass
        g = s["g"][r:r + n].double()[:, None]
        dx = g * (pick - kept)
        if s["h"] is not None:
            dx = dx - s["h"][r:r + n].double()[:, None] * (torch.xlogy(kept, kept) + kept * s["entropy"][r:r + n].double()[:, None])
        return {"dlogits": dx / T * live[:, None]}
    ids, u = s["teacher_ids"][r:r + n].long(), s["teacher"][r:r + n].double() / T
    u = u.masked_fill((ids < 0) | (ids >= V), -math.inf)
    q = torch.softmax(u, 1).nan_to_num(0.0)                               # a row without a teacher has none
    at = ids.clamp(0, V - 1)
    dense_q = torch.zeros_like(x)
    dense_q.scatter_add_(1, at, q)
    some = (q.sum(1, keepdim=True) > 0.5).double()
    soft = (torch.xlogy(q, q).sum(1) - torch.where(q > 0, q * logp.gather(1, at), 0.0).sum(1)) * T * T * live
    dx = case["soft"] * T * (p * some - dense_q)
    hard = torch.zeros_like(soft)
    if case["hard"]:
        p1 = torch.softmax(x, 1)
        hard = -torch.log((p1 * pick).sum(1) + EPSILON) * live
        dx = dx + case["hard"] * (p1 - pick)
    return {"soft": soft, "hard": hard, "dlogits": dx * live[:, None]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        E, V = case["E"], case["V"]
        ids = s["ids"].reshape(-1).double()
        total = s["dY"].double().reshape(-1, E)
        if s["dY2"] is not None:
            total = total + s["dY2"].double().reshape(-1, E)
        chosen = ((ids >= 1) & (ids < V)).nonzero()[:, 0]
        # the product of the one-hot matrix of the tokens with their gradients
        onehot = torch.sparse_coo_tensor(torch.stack([ids[chosen].long(), torch.arange(len(chosen), device="cuda")]),
                                         torch.full((len(chosen),), float(E), dtype=torch.float64, device="cuda").sqrt(), (V, len(chosen)))
        dW = torch.sparse.mm(onehot, total[chosen]) if len(chosen) else torch.zeros(V, E, dtype=torch.float64, device="cuda")
        if s["before"] is not None:
            dW = dW + s["before"].double()
        return {"dW": dW}

    rows, V = case["rows"], case["V"]
    step = max(1, (1 << 26) // V)
    parts = []
    for r in range(0, rows, step):
        parts.append(_exact_rows(s, r, step))
    out = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    parts.clear()
    if case["op"] == "distill":
        t = s["tokens"].trunc()
        count = float(((t >= 1) & (t <= V - 1)).sum())
        out["dlogits"] /= count
        out["losses"] = torch.stack([out.pop("soft"), out.pop("hard")])
        out["stats"] = torch.cat([out["losses"].sum(1), out["losses"].new_tensor([count])])
    elif case["op"] == "score" and case["top"]:
        out["top_ids"] = None
    return out
