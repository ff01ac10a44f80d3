"""Cases of the operators either side of the scorers: feature projection, dropout, and the losses over scores.

    features -> linear -> dropout -> rows -> scorer -> preference_loss
    scores over candidates -> log_prob -> policy_loss

`run` computes an operator in its plain form (elementary torch operations, 32 bits) or, where `own` is true, through the
entry points of cuke_b200.features and cuke_b200.losses.  `exact` computes the same outputs in 64 bits from the
definitions.  Sizes follow the framework's configurations: 15,000 / 40,000 / 100,000 / 4,000,000 entities, 1350 relations,
rows of 128 to 1024 numbers, batches of 1024 to 65,536 triples.
"""
import math

import torch

own = False


def listed():
    return [
        # embedding dropout of a small batch's rows: forward and gradient, launch-bound
        {"name": "dropout_small", "op": "dropout", "rows": 256, "dim": 128, "dtype": "f32", "p": 0.1, "residual": False},
        # every row slot of a 65,536-triple batch with shared negatives (three slots a triple), rows of 400 numbers
        {"name": "dropout_batch", "op": "dropout", "rows": 196608, "dim": 400, "dtype": "f32", "p": 0.2, "residual": False},
        # 1000 pairs of a preferred and a rejected triple against a frozen scorer: the smallest useful loss call
        {"name": "preference_pairs", "op": "preference", "rows": 1000, "n": 1, "ref": True, "mask": False, "kind": "logistic"},
        # 65,536 triples x 1024 shared negatives, known-true triples masked out, reference scores beside the trained ones
        {"name": "preference_chunks", "op": "preference", "rows": 65536, "n": 1024, "ref": True, "mask": True, "kind": "logistic"},
        # next-hop choice of a path-walking policy: up to 64 outgoing edges per node, ragged
        {"name": "policy_hops", "op": "policy", "rows": 1024, "n": 64, "dtype": "f32", "ragged": True, "kl": 0.05},
        # a policy over all entities of a 15,000-entity graph
        {"name": "policy_all_15k", "op": "policy", "rows": 4096, "n": 15000, "dtype": "f32", "ragged": False, "kl": 0.02},
        # the same over 100,000 entities, scores stored in 16 bits
        {"name": "policy_all_100k", "op": "policy", "rows": 1024, "n": 100000, "dtype": "bf16", "ragged": False, "kl": 0.02},
        # four link-prediction queries ranked against every entity of a 4,000,000-entity table
        {"name": "logprob_queries", "op": "logprob", "rows": 4, "n": 4000000, "dtype": "f32", "ragged": False, "backward": False},
        # relation prediction for a batch: 1350 classes, 16-bit scores whose rows are not a multiple of 16 bytes, with gradient
        {"name": "logprob_relations", "op": "logprob", "rows": 8192, "n": 1350, "dtype": "bf16", "ragged": False, "backward": True},
        # one new entity projected from its features while serving
        {"name": "linear_one", "op": "linear", "m": 1, "k": 1024, "n": 512, "act": "gelu", "residual": False, "backward": False},
        # one training batch of entity features into rows of 400 numbers
        {"name": "linear_batch", "op": "linear", "m": 8191, "k": 1024, "n": 400, "act": "silu", "residual": False, "backward": True},
        # a residual block of the feature encoder over a 65,536-entity batch
        {"name": "linear_block", "op": "linear", "m": 65536, "k": 1024, "n": 1024, "act": "gelu", "residual": True, "backward": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout", "preference", "policy", "logprob", "linear"])
    if op == "dropout":
        rows = _log(rng, 1, 200000)
        return {"op": op, "rows": rows, "dim": _log(rng, 1, min(4096, max(1, 78000000 // rows))), "dtype": rng.choice(["f32", "bf16"]),
                "p": rng.choice([0.05, 0.1, 0.2, 0.5]), "residual": rng.random() < 0.5}
    if op == "preference":
        rows = _log(rng, 1, 65536)
        return {"op": op, "rows": rows, "n": _log(rng, 1, min(8192, max(1, 67000000 // rows))), "ref": rng.random() < 0.6,
                "mask": rng.random() < 0.5, "kind": rng.choice(["logistic", "logistic", "square"])}
    if op == "policy":
        rows = _log(rng, 1, 16384)
        return {"op": op, "rows": rows, "n": _log(rng, 2, min(200000, max(2, 100000000 // rows))), "dtype": rng.choice(["f32", "bf16"]),
                "ragged": rng.random() < 0.5, "kl": rng.choice([0.0, 0.02, 0.1])}
    if op == "logprob":
        rows = _log(rng, 1, 16384)
        return {"op": op, "rows": rows, "n": _log(rng, 2, min(4000000, max(2, 60000000 // rows))), "dtype": rng.choice(["f32", "bf16"]),
                "ragged": rng.random() < 0.5, "backward": rng.random() < 0.6}
    m = _log(rng, 1, 65536)
    return {"op": op, "m": m, "k": 8 * _log(rng, 4, 256), "n": 8 * _log(rng, 4, 128), "act": rng.choice(["none", "relu", "silu", "gelu"]),
            "residual": rng.random() < 0.5, "backward": m > 16 and rng.random() < 0.7}


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}
    op = case["op"]
    if op == "dropout":
        shape = (case["rows"], case["dim"])
        st["x"] = (randn(*shape) / math.sqrt(case["dim"])).to(_dtype(case))
        st["dy"] = (randn(*shape) * 1e-2).to(_dtype(case))
        st["res"] = randn(*shape).to(_dtype(case)) if case["residual"] else None
        st["seed"], st["stream"], st["step"] = 20240501 + seed, 3, seed % 1000
    elif op == "preference":
        b, n = case["rows"], case["n"]
        # log-sigmoid scale scores of a trained scorer and of the frozen one it started from
        st["pos"], st["neg"] = randn(b) * 2 + 1, randn(b, n) * 2 - 1
        st["rpos"] = st["pos"] + 0.3 * randn(b) - 0.2 if case["ref"] else None
        st["rneg"] = st["neg"] + 0.3 * randn(b, n) + 0.1 if case["ref"] else None
        st["mask"] = rand(b, n) > 0.05 if case["mask"] else None
        if case["mask"]:
            st["mask"][::17] = rand(b, 1)[::17] > 0.5       # rows that keep everything or nothing
        st["weight"] = rand(b) + 0.5 if case["mask"] else None
        st["margin"], st["smooth"] = (0.5, 0.0) if case["kind"] == "square" else (0.1, 0.05)
        st["beta"] = 0.5
    elif op in ("policy", "logprob"):
        r, n = case["rows"], case["n"]
        st["scores"] = (randn(r, n) * 3).to(_dtype(case))
        cand = torch.full((r,), n, dtype=torch.int64, device="cuda")
        if case["ragged"]:
            cand = 1 + (rand(r) * n).long().clamp_(max=n - 1)
            cand[5::31] = 0                                   # nodes without an outgoing edge
            st["scores"][3::31, 0] = float("-inf")            # an edge that the walk may not take
        st["cand"] = cand.to(torch.int32) if case["ragged"] else None
        action = (rand(r) * cand).long().clamp_(min=0)
        action = torch.minimum(action, (cand - 1).clamp_(min=0))
        taken = st["scores"].gather(1, action[:, None])
        action = torch.where((cand > 1) & torch.isinf(taken[:, 0]), torch.ones_like(action), action)
        cand = torch.where(torch.isinf(st["scores"].gather(1, action[:, None])[:, 0]), torch.zeros_like(cand), cand)
        st["action"] = torch.where(cand > 0, action, torch.full_like(action, -1))   # -1: nothing was chosen
        if case["ragged"]:
            st["cand"] = cand.to(torch.int32)
        st["temp"] = 1.25
        if op == "policy":
            logp = _logp64(st["scores"], st["action"], cand, st["temp"])[0]
            # the policy that sampled is a few updates old; a ratio on a clip border itself has no defined gradient
            delta = 0.15 * randn(r).double()
            for edge in (math.log(0.8), math.log(1.28)):
                near = (delta - edge).abs() < 1e-3
                delta = torch.where(near, delta + 4e-3, delta)
            st["old"] = (logp - delta).float()
            st["ref"] = (logp + 0.2 * randn(r).double()).float() if case["kl"] else None
            st["adv"] = randn(r)
            st["weight"] = (rand(r) > 0.1).float()            # 0: a step past the end of its walk
        else:
            st["dlogp"] = randn(r) / r
    else:
        m, k, n = case["m"], case["k"], case["n"]
        bf = torch.bfloat16
        st["x"], st["w"] = randn(m, k).to(bf), (randn(k, n) / math.sqrt(k)).to(bf)
        st["b"] = (0.1 * randn(n)).to(bf)
        st["res"] = randn(m, n).to(bf) if case["residual"] else None
        st["dy"] = randn(m, n).to(bf) if case["backward"] else None
    return st


def _logp64(scores, action, cand, temp):
    """(log-probability of the action, 0 where there is none; row maximum; sum) in 64 bits, a block of rows at a time."""
    logp, step = [], max(1, 50000000 // scores.shape[1])
    for i in range(0, scores.shape[0], step):
        s = scores[i:i + step].double() / temp
        s.masked_fill_(torch.arange(s.shape[1], device=s.device)[None, :] >= cand[i:i + step, None], float("-inf"))
        a = action[i:i + step]
        v = s.gather(1, a.clamp(min=0)[:, None])[:, 0] - torch.logsumexp(s, 1)
        logp.append(torch.where(a >= 0, v, torch.zeros_like(v)))
    return torch.cat(logp), None


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _philox(n, seed, stream, step, device):
    """Words of the elements 0..n-1: word i % 4 of Philox4x32-10 at counter (i/4, stream, 2^31 | step), key = seed."""
    low = 0xFFFFFFFF
    q = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = q & low, q >> 32
    c2, c3 = torch.full_like(q, stream), torch.full_like(q, 0x80000000 | (step & 0x7FFFFFFF))
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _plain_dropout(x, p, keep, res):
    y = torch.where(keep, x.float() * (1.0 / (1.0 - p)), 0.0)
    return (y if res is None else y + res.float()).to(x.dtype)


def _plain_preference(st):
    c = st["case"]
    h = st["pos"][:, None] - st["neg"]
    if st["rpos"] is not None:
        h = h - (st["rpos"][:, None] - st["rneg"])
    z = st["beta"] * h - st["margin"]
    if c["kind"] == "square":
        loss, dz = z * z, 2 * z
    else:
        e = st["smooth"]
        soft = torch.log1p(torch.exp(-z.abs()))
        loss = (1 - e) * (soft + (-z).clamp(min=0)) + e * (soft + z.clamp(min=0))
        dz = 1 / (1 + torch.exp(-z)) - (1 - e)
    w = torch.full_like(st["pos"], 1.0 / c["n"])
    if st["mask"] is not None:
        loss, dz = torch.where(st["mask"], loss, 0.0), torch.where(st["mask"], dz, 0.0)
        w = 1.0 / st["mask"].sum(1).clamp(min=1)
    if st["weight"] is not None:
        w = w * st["weight"]
    total = (w.double() * loss.sum(1, dtype=torch.float64)).sum().float().reshape(1)
    d = dz * (st["beta"] * w)[:, None]
    return total, d.sum(1), -d


def _plain_softmax(st):
    """(log-probability of the action in 64 bits, probabilities) with the row statistics in 32 bits."""
    s = st["scores"].float()
    if st["cand"] is not None:
        s = torch.where(torch.arange(s.shape[1], device=s.device)[None, :] < st["cand"][:, None], s, float("-inf"))
    top = s.max(1, keepdim=True).values
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp((s - top) * (1.0 / st["temp"]))
    total = e.sum(1, keepdim=True)
    a = st["action"].clamp(min=0)[:, None]
    logp = (s.gather(1, a).double() - top.double()) / st["temp"] - torch.log(total.double())
    logp = torch.where(st["action"] >= 0, logp[:, 0], 0.0)
    return logp, e / torch.where(total > 0, total, 1.0)


def _plain_gradient(st, prob, g):
    """g / T (1[j = action] - prob), rows without an action zero, in the type of the scores."""
    g = torch.where(st["action"] >= 0, g / st["temp"], 0.0).float()
    d = prob * -g[:, None]
    d = d.scatter_add(1, st["action"].clamp(min=0)[:, None], g[:, None])
    return d.to(st["scores"].dtype)


def _plain_policy(st):
    c = st["case"]
    logp, prob = _plain_softmax(st)
    live = (st["action"] >= 0).double() * st["weight"].double()
    ratio, adv = torch.exp(logp - st["old"].double()), st["adv"].double()
    loss = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.28) * adv)
    held = ((adv > 0) & (ratio > 1.28)) | ((adv < 0) & (ratio < 0.8))
    g = torch.where(held, 0.0, -ratio * adv)
    kl = torch.zeros_like(logp)
    if st["ref"] is not None:
        d = st["ref"].double() - logp
        kl = torch.where(st["action"] >= 0, torch.exp(d) - d - 1, 0.0)
        loss, g = loss + c["kl"] * kl, g + c["kl"] * (1 - torch.exp(d))
    total = ((loss * live).sum() / c["rows"]).float().reshape(1)
    return total, logp.float(), kl.float(), _plain_gradient(st, prob, g * live / c["rows"])


def _act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    s = 1 / (1 + torch.exp(-2 * u))
    return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def _plain_linear(st):
    c, bf = st["case"], torch.bfloat16
    x, w = st["x"].float(), st["w"].float()
    y, slope = _act(x @ w + st["b"].float(), c["act"])
    out = {"out": (y if st["res"] is None else y + st["res"].float()).to(bf)}
    if c["backward"]:
        dz = st["dy"].float() * slope
        out["dx"], out["dw"], out["db"] = (dz @ w.T).to(bf), (x.T @ dz).to(bf), dz.sum(0).to(bf)
    return out


def run(st):
    c = st["case"]
    op = c["op"]
    if own:
        from cuke_b200 import features, losses
    if op == "dropout":
        if own:
            how = {"stream_id": st["stream"], "step": st["step"]}
            return {"y": features.dropout(st["x"], c["p"], st["seed"], residual=st["res"], **how),
                    "dx": features.dropout(st["dy"], c["p"], st["seed"], **how)}
        keep = _philox(st["x"].numel(), st["seed"], st["stream"], st["step"], "cuda") >= math.floor(c["p"] * 2.0 ** 32)
        keep = keep.view(st["x"].shape)
        return {"y": _plain_dropout(st["x"], c["p"], keep, st["res"]), "dx": _plain_dropout(st["dy"], c["p"], keep, None)}
    if op == "preference":
        if own:
            r = losses.preference_loss(st["pos"], st["neg"], st["rpos"], st["rneg"], mask=st["mask"], weight=st["weight"],
                                       kind=c["kind"], beta=st["beta"], margin=st["margin"], smoothing=st["smooth"])
        else:
            r = _plain_preference(st)
        return {"loss": r[0], "dpos": r[1], "dneg": r[2]}
    if op == "policy":
        if own:
            r = losses.policy_loss(st["scores"], st["action"], st["old"], st["adv"], ref_logp=st["ref"], n_cand=st["cand"],
                                   weight=st["weight"], temperature=st["temp"], clip_low=0.2, clip_high=0.28, kl_coef=c["kl"])
        else:
            r = _plain_policy(st)
        return {"loss": r[0], "logp": r[1], "kl": r[2], "dscores": r[3]}
    if op == "logprob":
        if own:
            logp, stats = losses.log_prob(st["scores"], st["action"], n_cand=st["cand"], temperature=st["temp"])
            if c["backward"]:
                return {"logp": logp, "dscores": losses.log_prob_backward(st["scores"], st["action"], stats, st["dlogp"],
                                                                          n_cand=st["cand"], temperature=st["temp"])}
            return {"logp": logp}
        logp, prob = _plain_softmax(st)
        if c["backward"]:
            return {"logp": logp.float(), "dscores": _plain_gradient(st, prob, st["dlogp"].double())}
        return {"logp": logp.float()}
    if own:
        if not c["backward"]:
            return {"out": features.linear(st["x"], st["w"], st["b"], act=c["act"], residual=st["res"])}
        out, preact = features.linear(st["x"], st["w"], st["b"], act=c["act"], residual=st["res"], save_preact=True)
        dx, dw, db = features.linear_backward(st["dy"], st["x"], st["w"], preact, act=c["act"])
        return {"out": out, "dx": dx, "dw": dw, "db": db}
    return _plain_linear(st)


def work(case):
    op = case["op"]
    size = 2 if case.get("dtype") == "bf16" else 4
    if op == "dropout":
        n = case["rows"] * case["dim"]
        return {"bytes": n * size * (5 if case["residual"] else 4), "flops": 2 * n}
    if op == "preference":
        b, n = case["rows"], case["n"]
        return {"bytes": b * n * (4 + 4 + 4 * case["ref"] + case["mask"]) + b * 4 * (2 + case["ref"] + case["mask"]) + 4, "flops": 20 * b * n}
    if op in ("policy", "logprob"):
        r, n = case["rows"], case["n"]
        back = op == "policy" or case["backward"]
        small = r * (8 + 4 * (7 if op == "policy" else 2)) + 4 * r * case["ragged"]
        live = 0.52 if case["ragged"] else 1.0              # the candidates that exist, on average
        return {"bytes": int(r * n * size * (live + back)) + small, "flops": 6 * r * n}
    m, k, n = case["m"], case["k"], case["n"]
    b = 2 * (m * k + k * n + n + m * n * (2 if case["residual"] else 1))
    if case["backward"]:
        b += 2 * (m * n + m * k + k * n + n)
    return {"bytes": b, "flops": 2 * m * n * k * (3 if case["backward"] else 1)}


# ---- 64 bits ------------------------------------------------------------------------------------------------------------
def _words64(index, seed, stream, step):
    """The same generator one element at a time, with the 32 x 32 bit products cut into 16-bit halves."""
    def wide(a, b):
        al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
        mid = ah * bl + ((al * bl) >> 16)
        mid2 = al * bh + (mid & 0xFFFF)
        return ah * bh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((al * bl) & 0xFFFF)
    quad = index // 4
    x = [quad % 2 ** 32, quad // 2 ** 32, torch.full_like(quad, stream), torch.full_like(quad, 2 ** 31 + step % 2 ** 31)]
    key = [seed % 2 ** 32, (seed // 2 ** 32) % 2 ** 32]
    for r in range(10):
        h0, l0 = wide(x[0], 0xD2511F53)
        h1, l1 = wide(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ ((key[0] + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x[3] ^ ((key[1] + r * 0xBB67AE85) % 2 ** 32), l0]
    return torch.stack(x).gather(0, (index % 4)[None])[0]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "dropout":
        x, dy = st["x"].double().reshape(-1), st["dy"].double().reshape(-1)
        y, dx = torch.empty_like(x), torch.empty_like(dy)
        for i in range(0, x.numel(), 1 << 24):
            at = torch.arange(i, min(i + (1 << 24), x.numel()), device="cuda")
            keep = (_words64(at, st["seed"], st["stream"], st["step"]) >= int(case["p"] * 2 ** 32)).double() / (1 - case["p"])
            y[at], dx[at] = x[at] * keep, dy[at] * keep
        y = y.view(st["x"].shape)
        return {"y": y if st["res"] is None else y + st["res"].double(), "dx": dx.view(st["x"].shape)}
    if op == "preference":
        pos, neg = st["pos"].double(), st["neg"].double()
        margin = pos.unsqueeze(1) - neg
        if case["ref"]:
            margin -= st["rpos"].double().unsqueeze(1)
            margin += st["rneg"].double()
        z = margin.mul_(st["beta"]).sub_(st["margin"])
        e, kind = st["smooth"], case["kind"]
        valid = torch.ones_like(z) if st["mask"] is None else st["mask"].double()
        scale = 1 / valid.sum(1).clamp(min=1)
        if st["weight"] is not None:
            scale = scale * st["weight"].double()
        scale = scale.unsqueeze(1) * valid
        zero = torch.zeros_like(z)
        each = z.square() if kind == "square" else (1 - e) * torch.logaddexp(zero, -z) + e * torch.logaddexp(zero, z)
        slope = 2 * z if kind == "square" else e * torch.sigmoid(z) - (1 - e) * torch.sigmoid(-z)
        d = slope * scale * st["beta"]
        return {"loss": (each * scale).sum().reshape(1), "dpos": d.sum(1), "dneg": -d}
    if op in ("policy", "logprob"):
        r, n = case["rows"], case["n"]
        have = st["action"] >= 0
        cand = st["cand"].long() if st["cand"] is not None else torch.full((r,), n, device="cuda")
        logp, _ = _logp64(st["scores"], st["action"], cand, st["temp"])
        if op == "logprob":
            if not case["backward"]:
                return {"logp": logp}
            g, answer = st["dlogp"].double(), {"logp": logp}
        else:
            up, down = st["adv"].double() > 0, st["adv"].double() < 0
            ratio = torch.exp(logp - st["old"].double())
            live = st["weight"].double() * have / r
            inside = ~((up & (ratio > 1.28)) | (down & (ratio < 0.8)))
            bounded = torch.where(inside, ratio, torch.where(up, torch.full_like(ratio, 1.28), torch.full_like(ratio, 0.8)))
            each, g, kl = -bounded * st["adv"].double(), -ratio * st["adv"].double() * inside, torch.zeros_like(logp)
            if case["kl"]:
                gap = logp - st["ref"].double()
                kl = (torch.expm1(-gap) + gap) * have
                each, g = each + case["kl"] * kl, g - case["kl"] * torch.expm1(-gap)
            answer = {"loss": (each * live).sum().reshape(1), "logp": logp, "kl": kl}
            g = g * live
        g = torch.where(have, g, torch.zeros_like(g)) / st["temp"]
        grad, step = torch.empty(r, n, dtype=torch.float64, device="cuda"), max(1, 50000000 // n)
        for i in range(0, r, step):
            s = st["scores"][i:i + step].double() / st["temp"]
            s[torch.arange(n, device="cuda").unsqueeze(0) >= cand[i:i + step].unsqueeze(1)] = float("-inf")
            rows = torch.nan_to_num(torch.softmax(s, 1)) * -g[i:i + step].unsqueeze(1)
            grad[i:i + step] = rows
        grad[torch.arange(r, device="cuda"), st["action"].clamp(min=0)] += g
        answer["dscores"] = grad
        return answer
    x, w = st["x"].double(), st["w"].double()
    z = torch.addmm(st["b"].double(), x, w).requires_grad_(case["backward"])
    if case["act"] == "relu":
        y = torch.relu(z)
    elif case["act"] == "silu":
        y = z * torch.sigmoid(z)
    elif case["act"] == "gelu":
        y = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    else:
        y = z * 1.0
    out = y if st["res"] is None else y + st["res"].double()
    if not case["backward"]:
        return {"out": out.detach()}
    dz, = torch.autograd.grad(y, z, st["dy"].double())
    return {"out": out.detach(), "dx": torch.mm(dz, w.t()), "dw": torch.mm(x.t(), dz), "db": dz.sum(0)}
