"""The operators as they are used together: entity rows computed from features, scored, trained on preferences or as a
policy, and the gradients taken back to the weights; against the same chain in 64 bits without a rounding."""
import numpy as np
import pytest
import torch

from cuke_b200 import features, losses, scoring
from tests.test_dropout import keep64
from tests.test_linear import act64

gpu = pytest.mark.gpu
F32, BF, HALF = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11      # half a step of fp32, bf16 and fp16, relative


def chain(x, w, b, rel, h, r, t, neg, chunk, p, seed, step, beta):
    """One step without an update: (loss, dw, db, every stage that a reader of the chain may want to look at)."""
    out, slope = features.linear(x, w, b, act="gelu", save_preact=True)
    ent = features.dropout(out, p, seed, 3, step)
    sc = scoring.Scorer("DistMult", ent, rel, neg_mode="chunk_shared", chunk=chunk)
    pos, negs, _ = sc.forward(h, r, t, neg)
    loss, dpos, dneg = losses.preference_loss(pos, negs, beta=beta, reduction="mean")
    g = sc.backward(h, r, t, neg, pos, negs, dpos, dneg)
    ids = scoring.inspect(scoring.entity_id_list(h, t, neg), ent.shape[0])
    rows = scoring.segment_reduce(g.ent_slots, ids, n_out=min(ids.n, ent.shape[0]))
    dent = torch.zeros(ent.shape, dtype=torch.float32, device=ent.device)
    scoring.scatter_rows(rows, ids.uniq, dent, n_dev=ids.n_unique)
    dout = features.dropout(dent.to(torch.bfloat16), p, seed, 3, step)
    _, dw, db = features.linear_backward(dout, x, w, slope, act="gelu", need_dx=False)
    return loss, dw, db, dent


def gelu_slope(z):
    with torch.enable_grad():
        q = z.clone().requires_grad_()
        return torch.autograd.grad(act64(q, "gelu").sum(), q)[0]


def chain64(x, w, b, rel, h, r, t, neg, chunk, keep, p, beta):
    """Values, gradients and first-order bounds.  A bound's terms are the roundings named beside them; each is carried on
    through the absolute values of what it meets.  Second-order terms are a few 2^-8 of the first: the 1.1."""
    x, w, b, rel = (q.double() for q in (x, w, b, rel))
    w.requires_grad_(), b.requires_grad_()
    z = x @ w + b
    y = act64(z, "gelu")
    scale = keep / (1 - p)
    ent = y * scale
    ent.retain_grad()
    tails = ent[neg].repeat_interleave(chunk, 0)                                     # (B, n, d)
    pos = (ent[h] * rel[r] * ent[t]).sum(1)
    negs = ((ent[h] * rel[r])[:, None] * tails).sum(2)
    n = neg.shape[1]
    zz = beta * (pos[:, None] - negs)
    loss = torch.nn.functional.softplus(-zz).mean()
    loss.backward()
    with torch.no_grad():
        a = lambda q: q.detach().abs()  # noqa: E731
        k, d, rows = x.shape[1], w.shape[1], h.numel()
        e, R = a(ent), a(rel)[r]
        zerr = (k + 4) * F32 * (a(x) @ a(w) + a(b))
        ee = scale * (1.13 * zerr + 2.0 ** -20 * (1 + a(z)) + BF * a(y)) + BF * e    # the product's rounding, dropout's
        H, T, N, eh, et, en = e[h], e[t], a(tails), ee[h], ee[t], ee[neg].repeat_interleave(chunk, 0)
        perr = (R * (H * et + eh * T) + (d + 4) * F32 * R * H * T).sum(1)
        nerr = ((R * H)[:, None] * en + (R * eh)[:, None] * N + (d + 4) * F32 * (R * H)[:, None] * N).sum(2)
        s = torch.sigmoid(-zz)                                                      # the loss's derivative, slope at most 1/4
        gn = beta * s / (rows * n)
        gnerr = beta / (rows * n) * (beta * (perr[:, None] + nerr) / 4 + 16 * F32 + 6 * F32 * s)
        gp, gperr = gn.sum(1), gnerr.sum(1)
        lerr = (beta * s * (perr[:, None] + nerr)).mean() + 32 * F32 * loss.detach()
        col = lambda q: q[:, None]  # noqa: E731
        acc = (n + 8) * F32
        sh = R * (col(gp) * et + col(gperr) * T + torch.einsum("bn,bnd->bd", gn, en) + torch.einsum("bn,bnd->bd", gnerr, N) +
                  acc * (col(gp) * T + torch.einsum("bn,bnd->bd", gn, N)))
        st = R * (col(gp) * eh + col(gperr) * H + acc * col(gp) * H)
        by = lambda q: q.view(-1, chunk, *q.shape[1:])  # noqa: E731
        sn = torch.einsum("cin,cid->cnd", by(gn), by(R * eh)) + torch.einsum("cin,cid->cnd", by(gnerr), by(R * H)) + \
            (chunk + 8) * F32 * torch.einsum("cin,cid->cnd", by(gn), by(R * H))
        size = torch.zeros_like(e)                                                  # what the segmented sum adds up, in size
        derr = torch.zeros_like(e)
        for ids, mag, err in ((h, R * (col(gp) * T + torch.einsum("bn,bnd->bd", gn, N)), sh), (t, R * col(gp) * H, st),
                              (neg.reshape(-1), torch.einsum("cin,cid->cnd", by(gn), by(R * H)).reshape(-1, d), sn.reshape(-1, d))):
            size.index_add_(0, ids, mag)
            derr.index_add_(0, ids, err)
        derr = derr + (2 * rows + neg.numel()) * F32 * size
        de = a(ent.grad)
        doerr = scale * (derr + BF * de) + BF * scale * de                          # to bf16, then dropout's rounding
        slope = gelu_slope(z.detach())
        do = scale * de
        serr = 1.2 * zerr + 2.0 ** -20 * (1 + a(z)) + HALF * a(slope) + 2.0 ** -25
        dz = do * a(slope)
        dzerr = doerr * a(slope) + do * serr + BF * dz
        rows_x = x.shape[0]
        dwerr = a(x).T @ dzerr + (rows_x + 4) * F32 * (a(x).T @ dz) + BF * a(w.grad)
        dberr = (doerr * a(slope) + do * serr).sum(0) + (rows_x + 4) * F32 * dz.sum(0) + BF * a(b.grad)
    return loss.detach(), w.grad, b.grad, ent.grad, (1.1 * lerr, 1.1 * dwerr, 1.1 * dberr, 1.1 * derr)


def case(n_ent, k, d, n_rel, batch, chunk, n, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n_ent)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ri = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")  # noqa: E731
    return dict(x=rn(n_ent, k).bfloat16(), w=(rn(k, d) / k ** 0.5).bfloat16(), b=(rn(d) / 4).bfloat16(), rel=rn(n_rel, d) / d ** 0.5,
                h=ri(n_ent, batch), r=ri(n_rel, batch), t=ri(n_ent, batch), neg=ri(n_ent, batch // chunk, n), chunk=chunk)


@gpu
@pytest.mark.parametrize("n_ent,k,d,n_rel,batch,chunk,n,p", [(40, 24, 16, 3, 32, 8, 5, 0.25), (600, 136, 200, 11, 512, 128, 96, 0.1), (5, 8, 8, 1, 1, 1, 1, 0.0)])
def test_preferences_over_computed_entities(n_ent, k, d, n_rel, batch, chunk, n, p):
    c = case(n_ent, k, d, n_rel, batch, chunk, n)
    # bf16 tables take bf16 relation rows: the chain below and the 64-bit one start from the same values
    c["rel"] = c["rel"].bfloat16()
    got = chain(**c, p=p, seed=77, step=5, beta=1.5)
    keep = torch.from_numpy(keep64(n_ent * d, p, 77, 3, 5).astype(np.float64)).view(n_ent, d).cuda()
    *want, bounds = chain64(**c, keep=keep, p=p, beta=1.5)
    for name, a, b, tol in zip(("loss", "dw", "db", "dent"), got, want, bounds):
        assert ((a.double() - b).abs() <= tol + 1e-12).all(), name
    again = chain(**c, p=p, seed=77, step=5, beta=1.5)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert scoring.device_flags() == 0


@gpu
def test_captured_step_draws_new_masks():
    """The whole step in a graph, the step number a tensor that is advanced between replays: each replay is the eager call
    of its step number."""
    c = case(300, 64, 72, 5, 64, 16, 12)
    c["rel"] = c["rel"].bfloat16()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                                   # grows the scorer's scratch before the capture
        chain(**c, p=0.3, seed=1, step=step, beta=1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = chain(**c, p=0.3, seed=1, step=step, beta=1.0)
    seen = []
    for i in (4, 0, 9):
        step.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        eager = chain(**c, p=0.3, seed=1, step=i, beta=1.0)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        seen.append(out[1].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@gpu
def test_policy_over_scored_candidates():
    """Candidate tails scored for (head, relation), a policy step on them, the gradient back to the table; fp32 throughout.
    At ratio 1 and without a KL term the step's gradient is that of -A log_prob / rows."""
    n_ent, d, n_rel, rows, n = 500, 64, 7, 48, 130
    c = case(n_ent, 8, d, n_rel, rows, 1, n)
    g = torch.Generator(device="cuda").manual_seed(2)
    ent = torch.randn(n_ent, d, generator=g, device="cuda")
    n_cand = torch.randint(1, n + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    n_cand[3] = 0
    action = (torch.rand(rows, generator=g, device="cuda") * n_cand).long().clamp(max=n - 1)
    action[3], action[4] = -1, -1
    adv = torch.randn(rows, generator=g, device="cuda")
    sc = scoring.Scorer("DistMult", ent, c["rel"], neg_mode="per_triple")
    pos, negs, _ = sc.forward(c["h"], c["r"], c["t"], c["neg"])
    old, stats = losses.log_prob(negs, action, n_cand, temperature=0.7)
    loss, logp, kl, dneg = losses.policy_loss(negs, action, old, adv, ref_logp=old, n_cand=n_cand, temperature=0.7, kl_coef=0.0)
    # the call's own log-probability is held in more bits than the fp32 `old` it gave out before: they differ by x, at most
    # half a step of fp32 of |old|; the ratio is 1 + x to first order, and kl = e^x - x - 1 <= x^2 for |x| <= 1
    x = F32 * old.abs().double()
    assert torch.equal(logp, old) and (kl >= 0).all() and (kl <= x * x).all()
    direct = losses.log_prob_backward(negs, action, stats, -adv / rows, n_cand, temperature=0.7)
    assert ((dneg - direct).abs() <= (8 * F32 + 2 * x[:, None]) * direct.abs() + 1e-12).all()
    zero = torch.zeros_like(pos)
    slots = sc.backward(c["h"], c["r"], c["t"], c["neg"], pos, negs, zero, dneg).ent_slots
    e = ent.double().requires_grad_()
    s = (e[c["h"]] * c["rel"].double()[c["r"]])[:, None] * e[c["neg"]]
    z = s.sum(2) / 0.7
    out = torch.arange(n, device="cuda") >= n_cand[:, None]
    lp = torch.log_softmax(z.masked_fill(out, -1e300), 1).gather(1, action.clamp(min=0)[:, None])[:, 0]
    live = action >= 0
    want = -(torch.where(live, lp * adv.double(), torch.zeros_like(lp))).sum() / rows
    want.backward()
    got = torch.zeros_like(e).index_add_(0, scoring.entity_id_list(c["h"], c["t"], c["neg"]), slots.double())
    with torch.no_grad():
        zerr = (d + 6) * F32 * s.abs().sum(2) / 0.7                                # the score's additions, the division
        pr = torch.softmax(z.masked_fill(out, -1e300), 1) * ~out
        top = zerr.masked_fill(out, 0).amax(1, keepdim=True)
        cw = (adv.abs() * live)[:, None].double() / rows / 0.7
        # p is off by twice the largest error of a logit plus its own evaluation; the chosen one's 1 - p the same
        gerr = cw * (pr * (2 * top + 2 * x[:, None] + 64 * F32) + torch.nn.functional.one_hot(action.clamp(min=0), n) * (2 * x[:, None] + 32 * F32))
        gabs = cw * (pr + torch.nn.functional.one_hot(action.clamp(min=0), n))
        H, R, N = e.abs()[c["h"]], c["rel"].double().abs()[c["r"]], e.abs()[c["neg"]]
        tol = torch.zeros_like(e)
        k = gerr + (n + d + 8) * F32 * gabs
        tol.index_add_(0, c["h"], R * torch.einsum("bn,bnd->bd", k, N))
        tol.index_add_(0, c["neg"].reshape(-1), (k[:, :, None] * (H * R)[:, None]).reshape(-1, d))
    assert ((got - e.grad).abs() <= tol + 1e-12).all()
    assert (dneg[3] == 0).all() and (dneg[4] == 0).all() and (dneg[out] == 0).all()
    # at ratio 1 the loss is -sum(A) / rows over the rows with an action
    assert abs(loss.item() + (adv.double() * live).sum().item() / rows) <= ((rows * F32 + 2 * x) * adv.abs()).sum().item() / rows
