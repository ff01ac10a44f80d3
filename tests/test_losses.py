"""Preference loss, candidate log-probabilities and policy loss (cuke_b200.losses) against their definitions in 64 bits."""
import os

import numpy as np
import pytest
import torch

from cuke_b200 import _lib, losses

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
NULL, SOME, ODD = None, 4096, 4098          # stand-ins for device addresses: a refused call never follows them
EPS = 2.0 ** -24                            # half a step of fp32, relative
gpu = pytest.mark.gpu


# ---- refusals (no GPU) --------------------------------------------------------------------------------------------------
def pref(pos=SOME, rpos=NULL, neg=SOME, ldn=8, rneg=NULL, ldr=0, mask=NULL, ldm=0, weight=NULL, rows=4, n=8, kind=0, beta=1.0, margin=0.0,
         smoothing=0.0, loss=SOME, dpos=SOME, dneg=SOME, ldd=8, ws=SOME, wsb=1 << 20):
    return _lib.lib().kge_preference_loss(pos, rpos, neg, ldn, rneg, ldr, mask, ldm, weight, rows, n, kind, beta, margin, smoothing, 1.0, loss,
                                          dpos, dneg, ldd, ws, wsb, None)


@needs_lib
@pytest.mark.parametrize("kw,code", [
    (dict(kind=2), -3), (dict(kind=1, smoothing=0.1), -3), (dict(smoothing=1.5), -6), (dict(smoothing=float("nan")), -6), (dict(rows=-1), -4),
    (dict(n=-1), -4), (dict(n=(1 << 30) + 1, ldn=1 << 31, ldd=1 << 31), -6), (dict(ldn=7), -4), (dict(ldd=7), -4), (dict(mask=SOME, ldm=7), -4),
    (dict(rpos=SOME, rneg=SOME, ldr=7), -4), (dict(pos=NULL), -1), (dict(neg=NULL), -1), (dict(dpos=NULL), -1), (dict(dneg=NULL), -1),
    (dict(loss=NULL), -1), (dict(rpos=SOME), -1), (dict(rneg=SOME, ldr=8), -1), (dict(pos=ODD), -2), (dict(neg=ODD), -2), (dict(dneg=ODD), -2),
    (dict(loss=ODD), -2), (dict(wsb=0), -5), (dict(ws=NULL), -1), (dict(ws=4104), -2)])
def test_preference_refusals(kw, code):
    assert pref(**kw) == code
    assert _lib.lib().kge_last_error().startswith(b"kge_preference_loss: ")


def cand(fn, scores=SOME, dtype=0, ld=8, rows=4, n=8, n_cand=NULL, action=SOME, bits=64, temp=1.0, old=SOME, ref=NULL, adv=SOME, weight=NULL,
         lo=0.2, hi=0.2, kl_coef=0.0, loss=SOME, logp=SOME, kl=SOME, stats=SOME, d=SOME, ldd=8, ws=SOME, wsb=1 << 26):
    L = _lib.lib()
    head = (scores, dtype, ld, rows, n, n_cand, action, bits, temp)
    if fn == "kge_log_prob":
        return L.kge_log_prob(*head, logp, stats, ws, wsb, None)
    if fn == "kge_log_prob_backward":
        return L.kge_log_prob_backward(*head, stats, adv, d, ldd, None)
    return L.kge_policy_loss(*head, old, ref, adv, weight, lo, hi, kl_coef, 1.0, loss, logp, kl, d, ldd, ws, wsb, None)


COMMON = [(dict(dtype=2), -3), (dict(bits=16), -3), (dict(temp=0.0), -6), (dict(temp=-1.0), -6), (dict(temp=float("nan")), -6),
          (dict(temp=float("inf")), -6), (dict(temp=1e-45), -6), (dict(rows=-1), -4), (dict(n=-1), -4), (dict(n=(1 << 30) + 1, ld=1 << 31), -6),
          (dict(ld=7), -4), (dict(ld=1 << 41), -6), (dict(scores=NULL), -1), (dict(action=NULL), -1), (dict(scores=ODD), -2), (dict(action=4100), -2),
          (dict(n_cand=ODD), -2)]
POLICY = [(dict(lo=-0.1), -6), (dict(lo=1.1), -6), (dict(hi=-0.1), -6), (dict(hi=float("nan")), -6), (dict(kl_coef=-1.0), -6), (dict(loss=NULL), -1),
          (dict(old=NULL), -1), (dict(adv=NULL), -1), (dict(logp=NULL), -1), (dict(kl=NULL), -1), (dict(d=NULL), -1), (dict(ldd=7), -4),
          (dict(ref=ODD), -2), (dict(weight=ODD), -2), (dict(d=ODD), -2), (dict(ws=NULL), -1), (dict(ws=4104), -2), (dict(wsb=0), -5)]


@needs_lib
@pytest.mark.parametrize("fn,kw,code", [("kge_log_prob", *c) for c in COMMON + [(dict(logp=NULL), -1), (dict(stats=NULL), -1), (dict(wsb=0), -5)]] +
                         [("kge_log_prob_backward", *c) for c in [(dict(stats=NULL), -1), (dict(adv=NULL), -1), (dict(d=NULL), -1), (dict(ldd=7), -4)]] +
                         [("kge_policy_loss", *c) for c in POLICY])
def test_candidate_refusals(fn, kw, code):
    try:
        device = _lib.lib().kge_check(None, (__import__("ctypes").c_int32 * 1)()) == 0
    except Exception:
        device = False
    got = cand(fn, **kw)
    # without a device a call whose first checks pass is refused for that (-7) before the later ones
    assert got == code or (not device and got == -7)
    if got == code:
        assert _lib.lib().kge_last_error().startswith(fn.encode() + b": ")


def test_python_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        losses.preference_loss(torch.zeros(2), torch.zeros(2, 3))
    with pytest.raises(ValueError, match="CUDA"):
        losses.log_prob(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="reduction"):
        losses._scale("max", 3)
    assert losses._scale("mean", 0) == 1.0 and losses._scale("mean", 4) == 0.25
    with pytest.raises(ValueError, match="float32"):
        losses._floats(torch.zeros(3, dtype=torch.float64), 3, "x")


# ---- preference loss ------------------------------------------------------------------------------------------------------
def pref64(pos, neg, rpos, rneg, mask, weight, kind, beta, margin, smoothing, scale):
    h = pos[:, None] - neg
    if rpos is not None:
        h = h - (rpos[:, None] - rneg)
    z = beta * h - margin
    valid = torch.ones_like(z, dtype=torch.bool) if mask is None else mask
    z = torch.where(valid, z, torch.zeros_like(z))
    sp = torch.nn.functional.softplus
    each = z * z if kind == "square" else (1 - smoothing) * -torch.nn.functional.logsigmoid(z) + (smoothing * -torch.nn.functional.logsigmoid(-z) if smoothing else 0)
    del sp
    cw = scale / valid.sum(1).clamp(min=1)
    if weight is not None:
        cw = cw * weight
    return (torch.where(valid, each, torch.zeros_like(each)) * cw[:, None]).sum(), z, cw


def pref_case(rows, n, ref, mask, weight, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + rows * 31 + n)
    r = lambda *s: torch.randn(*s, generator=g) * spread  # noqa: E731
    p = dict(pos=r(rows), neg=r(rows, n), rpos=r(rows) if ref else None, rneg=r(rows, n) if ref else None,
             mask=None, weight=(torch.rand(rows, generator=g) + 0.1) if weight else None)
    if mask:
        m = torch.rand(rows, n, generator=g) > 0.4
        m[::3] = torch.rand(m[::3].shape[0], 1, generator=g) > 0.5            # whole rows on or off
        p["mask"] = m
        for k in ("neg", "rneg"):                                             # what is masked out is not read
            if p[k] is not None:
                p[k] = torch.where(m, p[k], torch.tensor([float("nan"), float("inf"), float("-inf")]).repeat(rows * n)[: rows * n].view(rows, n))
    return p


def pref_check(p, kind="logistic", beta=1.0, margin=0.0, smoothing=0.0, reduction="sum", dev=None):
    rows, n = p["neg"].shape
    scale = 1.0 if reduction == "sum" else 1.0 / max(rows, 1)
    d = {k: None if v is None else v.cuda() for k, v in p.items()} if dev is None else dev
    loss, dpos, dneg = losses.preference_loss(d["pos"], d["neg"], d["rpos"], d["rneg"], mask=d["mask"], weight=d["weight"], kind=kind, beta=beta,
                                              margin=margin, smoothing=smoothing, reduction=reduction)
    valid = torch.ones(rows, n, dtype=torch.bool) if p["mask"] is None else p["mask"]
    q = {k: None if v is None else v.double() if v.dtype == torch.float32 else v for k, v in p.items()}
    for k in ("neg", "rneg"):
        if q[k] is not None:
            q[k] = torch.where(valid, q[k], torch.zeros_like(q[k]))
    q["pos"].requires_grad_(), q["neg"].requires_grad_()
    ref, z, cw = pref64(q["pos"], q["neg"], q["rpos"], q["rneg"], q["mask"], q["weight"], kind, beta, margin, smoothing, scale)
    gp, gn = torch.autograd.grad(ref, (q["pos"], q["neg"]))
    # z: four roundings of terms up to |pos| + |neg| + ..., times beta; l and l' then follow with slope <= 1 (logistic; the
    # exponential, logarithm and division add < 8 roundings of values <= 1 + |z|) or 2|z| (square)
    size = q["pos"].detach().abs()[:, None] + q["neg"].detach().abs()
    if q["rpos"] is not None:
        size = size + q["rpos"].abs()[:, None] + q["rneg"].abs()
    dz = 6 * EPS * (abs(beta) * size + abs(margin))
    zz = z.detach().abs()
    # the exponential's argument carries |z| roundings: e^-|z| is off by (4 + 2|z|) EPS relative, always below 4 EPS absolute + ...
    el = 2 * zz * dz + 4 * EPS * zz * zz if kind == "square" else dz + EPS * (12 + 4 * zz)
    ed = 2 * dz + 4 * EPS * zz if kind == "square" else dz + 12 * EPS
    cw = cw.detach()[:, None].abs()
    tn = abs(beta) * cw * ed + 6 * EPS * gn.abs()
    tn = torch.where(valid, tn, torch.zeros_like(tn))
    # sums of n terms a row: at most n - 1 roundings of the running sum
    tp = tn.sum(1) + (n + 8) * EPS * gn.abs().sum(1)
    each = zz * zz if kind == "square" else 1 + zz
    tl = (cw * torch.where(valid, el + (n + 8) * EPS * each, torch.zeros_like(el))).sum() + EPS * ref.abs()
    assert ((dneg.view(rows, n).cpu().double() - gn).abs() <= tn + 1e-37).all()
    assert ((dpos.view(-1).cpu().double() - gp).abs() <= tp + 1e-37).all()
    assert abs(loss.item() - ref.item()) <= tl.item() + 1e-37
    return loss, dpos, dneg


@gpu
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 1), (1000, 1), (257, 2), (33, 3), (65, 7), (5, 31), (4, 32), (9, 33), (130, 64), (3, 1000), (17, 1024),
                                    (2, 4099), (1, 20000), (2500, 12), (1, 70001)])
@pytest.mark.parametrize("ref,mask,weight", [(False, False, False), (True, False, True), (True, True, True), (False, True, False)])
def test_preference_logistic(rows, n, ref, mask, weight):
    p = pref_case(rows, n, ref, mask, weight)
    a = pref_check(p, beta=0.7, margin=0.2, smoothing=0.1)
    pref_check(p, beta=1.0, reduction="mean")
    b = pref_check(p, beta=0.7, margin=0.2, smoothing=0.1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("rows,n", [(300, 8), (301, 24), (130, 25), (100, 61), (4800, 68), (4740, 131), (1200, 200), (1190, 333), (40, 300), (800, 701),
                                    (40, 2044), (7, 9001), (5, 8200), (160, 4100)])
@pytest.mark.parametrize("mask", [False, True])
def test_preference_every_group_of_threads(rows, n, mask):
    pref_check(pref_case(rows, n, True, mask, True), beta=0.7, margin=0.2, smoothing=0.1)
    pref_check(pref_case(rows, n, False, mask, False), kind="square", beta=0.3)


@gpu
@pytest.mark.parametrize("rows,n,mask", [(7, 1, False), (64, 20, True), (3, 1111, True)])
def test_preference_square(rows, n, mask):
    pref_check(pref_case(rows, n, True, mask, True), kind="square", beta=0.3, margin=0.5)


@gpu
def test_preference_pitched_chunked_and_empty():
    rows, n = 24, 20
    p = pref_case(rows, n, True, True, True, seed=4)
    want = pref_check(p, smoothing=0.05)
    d = {k: v.cuda() for k, v in p.items()}
    for ld, off in ((28, 0), (21, 1), (24, 4), (33, 3)):
        for k in ("neg", "rneg", "mask"):
            wide = torch.zeros(rows * ld + off, dtype=p[k].dtype, device="cuda")
            v = wide[off:off + rows * ld].view(rows, ld)[:, :n]
            v.copy_(p[k])
            d[k] = v
        got = pref_check(p, smoothing=0.05, dev=d)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
    c = {k: v.cuda() for k, v in p.items()}
    loss, dpos, dneg = losses.preference_loss(c["pos"], c["neg"].view(3, 8, n), c["rpos"], c["rneg"].view(3, 8, n), mask=c["mask"].view(3, 8, n),
                                              weight=c["weight"], smoothing=0.05)
    assert dneg.shape == (3, 8, n) and torch.equal(dneg.view(rows, n), want[2]) and torch.equal(loss, want[0])
    loss, dpos, dneg = losses.preference_loss(c["pos"][:0], c["neg"][:0])
    assert loss.item() == 0 and dpos.numel() == 0 and dneg.shape == (0, n)
    loss, dpos, dneg = losses.preference_loss(c["pos"], c["neg"][:, :0])
    assert loss.item() == 0 and (dpos == 0).all() and dneg.shape == (rows, 0)
    loss, dpos, dneg = losses.preference_loss(c["pos"], c["neg"], mask=torch.zeros(rows, n, dtype=torch.bool, device="cuda"))
    assert loss.item() == 0 and (dpos == 0).all() and (dneg == 0).all()
    loss, dpos, dneg = losses.preference_loss(c["pos"], torch.full((rows, n), float("nan"), device="cuda"), weight=torch.zeros(rows, device="cuda"))
    assert loss.item() == 0 and (dpos == 0).all() and (dneg == 0).all()


@gpu
def test_preference_extremes():
    """A rejected triple of score -infinity costs nothing, large margins neither overflow nor lose the small side."""
    pos = torch.zeros(6, device="cuda")
    neg = torch.tensor([[float("-inf")], [-3e38], [3e38], [100.0], [-100.0], [-30.0]], device="cuda")
    loss, dpos, dneg = losses.preference_loss(pos[:2], neg[:2])
    assert loss.item() == 0 and (dneg == 0).all()
    loss, dpos, dneg = losses.preference_loss(pos[2:4], neg[2:4])
    assert torch.equal(dneg, torch.ones_like(dneg)) and loss.item() == torch.tensor(3e38).item()
    _, _, dneg = losses.preference_loss(pos[5:], neg[5:])
    assert abs(dneg.item() / np.exp(-30.0) - 1) < 100 * EPS


@gpu
def test_preference_against_differences():
    """Central differences of the 64-bit loss: h^2 / 6 |l'''| <= 1e-8 / 6 with h = 1e-4, and 1e-16 / h of rounding."""
    p = pref_case(5, 4, True, True, True, seed=9)
    loss, dpos, dneg = losses.preference_loss(*(p[k].cuda() for k in ("pos", "neg", "rpos", "rneg")), mask=p["mask"].cuda(), weight=p["weight"].cuda(),
                                              beta=0.8, smoothing=0.2)
    q = {k: v.double() if v.dtype == torch.float32 else v for k, v in p.items()}
    f = lambda: pref64(*(torch.where(q["mask"], q[k], torch.zeros_like(q[k])) if k in ("neg", "rneg") else q[k]  # noqa: E731
                         for k in ("pos", "neg", "rpos", "rneg")), q["mask"], q["weight"], "logistic", 0.8, 0.0, 0.2, 1.0)[0].item()
    h = 1e-4
    for b in range(5):
        for t, grad, at in [(q["pos"], dpos, (b,))] + [(q["neg"], dneg, (b, j)) for j in range(4)]:
            old = t[at].item()
            t[at] = old + h
            up = f()
            t[at] = old - h
            down = f()
            t[at] = old
            assert abs((up - down) / (2 * h) - grad[at].item()) < 3e-6


# ---- candidates -------------------------------------------------------------------------------------------------------------
def cand_case(rows, n, dtype, ragged, seed=0, spread=3.0, id_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + 7 * rows + n)
    s = (torch.randn(rows, n, generator=g) * spread).to(dtype)
    cnt = torch.full((rows,), n, dtype=torch.int64)
    if ragged:
        cnt = (torch.rand(rows, generator=g) * (n + 1)).long().clamp(max=n)
        cnt[0] = n
        s = torch.where(torch.arange(n)[None] < cnt[:, None], s, torch.tensor(float("nan"), dtype=dtype))     # padding is not read into anything
    act = (torch.rand(rows, generator=g) * cnt).long()
    act = torch.where(cnt > 0, torch.minimum(act, (cnt - 1).clamp(min=0)), torch.full_like(act, -1))
    if rows > 3:
        act[2] = -1
    return s, act.to(id_dtype), cnt.to(torch.int32) if ragged else None, cnt, g


def logits64(s, cnt, temp):
    x = s.double() / temp
    return x.masked_fill(torch.arange(s.shape[1])[None] >= cnt[:, None], float("-inf"))


def cand_ref(s, act, cnt, temp):
    """(live, logp, p): 64-bit log-probability (0 where a row takes no part) and probabilities (0 there and at padding)."""
    x = logits64(s, cnt, temp)
    live = (act >= 0) & ~(torch.isneginf(x).all(1))
    lse = torch.where(live, torch.logsumexp(x, 1), torch.zeros(len(act), dtype=torch.float64))
    lp = torch.where(live, x.gather(1, act.long().clamp(min=0)[:, None])[:, 0] - lse, torch.zeros_like(lse))
    return live, lp, torch.where(live[:, None], torch.exp(x - lse[:, None]), torch.zeros_like(x))


def rel_bound(s, cnt, temp):
    """Relative error of a row's exponentials and of their sum: the argument (s - m) / T log2(e) is rounded three times
    (2 A ln2 half-steps each, A its size), the exponential itself is good to 4 half-steps, n / 32 + 24 additions follow."""
    x = logits64(s, cnt, temp)
    x = torch.where(torch.isinf(x), torch.zeros_like(x), x)
    A = (x.max(1).values - x.min(1).values) if s.shape[1] else torch.zeros(s.shape[0], dtype=torch.float64)
    return EPS * (6 * A + 8 + s.shape[1] / 32 + 24)


def check_gradient(d, s, act, p, live, coef, dcoef, E, n):
    """d against coef (1[j = a] - p); coef (rows,) with absolute error dcoef."""
    d = d.cpu().double()
    onehot = torch.zeros_like(p)
    onehot.scatter_(1, act.long().clamp(min=0)[:, None], live.double()[:, None])
    rest = torch.where(onehot > 0, 1 - p, p)                       # |1[j = a] - p_j|
    if n > 1:                                                      # 1 - p without cancellation
        other = (p * (1 - onehot)).sum(1, keepdim=True)
        rest = torch.where(onehot > 0, other, p)
    ref = coef[:, None] * torch.where(onehot > 0, rest, -rest)
    tol = (dcoef[:, None] + coef.abs()[:, None] * (3 * E[:, None] + 8 * EPS)) * rest + 1e-37 * (1 + coef.abs()[:, None])
    if s.dtype == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * ref.abs()
    bad = ~((d - ref).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:4], d[bad][:4], ref[bad][:4])


SHAPES = [(1, 1), (1, 2), (5, 2), (300, 3), (64, 31), (33, 64), (7, 129), (40, 250), (9, 1000), (8, 1024), (6, 1350), (5, 2049), (3, 5003), (2, 15000),
          (3, 40001), (1, 100000), (2, 200003), (1200, 40)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_log_prob(rows, n, ragged, dtype):
    s, act, n_cand, cnt, g = cand_case(rows, n, dtype, ragged, id_dtype=torch.int32 if rows % 2 else torch.int64)
    temp = 0.8
    ds, da, dn = s.cuda(), act.cuda(), None if n_cand is None else n_cand.cuda()
    logp, stats = losses.log_prob(ds, da, n_cand=dn, temperature=temp)
    live, lp, p = cand_ref(s, act, cnt, temp)
    E = rel_bound(s, cnt, temp)
    assert ((logp.cpu().double() - lp).abs() <= E + 2 * EPS * lp.abs()).all()
    dl = torch.randn(rows, generator=g)
    d = losses.log_prob_backward(ds, da, stats, dl.cuda(), n_cand=dn, temperature=temp)
    coef = torch.where(live, dl.double() / temp, torch.zeros(rows, dtype=torch.float64))
    check_gradient(d, s, act, p, live, coef, 4 * EPS * coef.abs(), E, n)
    again, stats2 = losses.log_prob(ds, da, n_cand=dn, temperature=temp)
    assert torch.equal(logp, again) and torch.equal(d, losses.log_prob_backward(ds, da, stats2, dl.cuda(), n_cand=dn, temperature=temp))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(2400, 300), (2400, 700), (2369, 513)])
def test_candidates_of_many_rows(rows, n, dtype):
    """More rows than the GPU holds warps."""
    s, act, n_cand, cnt, g = cand_case(rows, n, dtype, True)
    policy_check(s, act, n_cand, cnt, g)
    logp, stats = losses.log_prob(s.cuda(), act.cuda(), n_cand=n_cand.cuda(), temperature=0.8)
    live, lp, p = cand_ref(s, act, cnt, 0.8)
    assert ((logp.cpu().double() - lp).abs() <= rel_bound(s, cnt, 0.8) + 2 * EPS * lp.abs()).all()


def policy64(lp, live, old, adv, ref, w, lo, hi, beta, scale):
    ratio = torch.exp(lp - old)
    l = -torch.minimum(ratio * adv, ratio.clamp(1 - lo, 1 + hi) * adv)
    kl = torch.zeros_like(lp)
    if ref is not None:
        kl = torch.exp(ref - lp) - (ref - lp) - 1
        l = l + beta * kl
    m = live.double() * (1 if w is None else w)
    return scale * (l * m).sum(), torch.where(live, kl, torch.zeros_like(kl)), ratio


def policy_check(s, act, n_cand, cnt, g, temp=1.3, lo=0.2, hi=0.3, beta=0.1, ref=True, weight=True, reduction="mean", dev=None):
    rows, n = s.shape
    live, lp, p = cand_ref(s, act, cnt, temp)
    delta = 0.3 * torch.randn(rows, generator=g).double()
    for edge in (np.log(1 - lo), np.log(1 + hi)):                       # a ratio on a border has no defined gradient
        delta = torch.where((delta - edge).abs() < 2e-3, delta + 8e-3, delta)
    old = (lp - delta).float()
    rp = (lp + 0.3 * torch.randn(rows, generator=g).double()).float() if ref else None
    adv = torch.randn(rows, generator=g)
    w = torch.rand(rows, generator=g).round(decimals=1) if weight else None
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    loss, logp, kl, d = losses.policy_loss(c(s) if dev is None else dev, c(act), c(old), c(adv), ref_logp=c(rp), n_cand=c(n_cand), weight=c(w), temperature=temp,
                                           clip_low=lo, clip_high=hi, kl_coef=beta if ref else 0.0, reduction=reduction)
    scale = 1.0 / rows if reduction == "mean" else 1.0
    w64 = None if w is None else w.double()
    lo32, hi32, b32 = (float(np.float32(v)) for v in (lo, hi, beta))    # the call takes fp32 settings
    x = lp.clone().requires_grad_()
    total, kl64, ratio = policy64(x, live, old.double(), adv.double(), None if rp is None else rp.double(), w64, lo32, hi32, b32, scale)
    coef = torch.autograd.grad(total, x)[0]
    E = rel_bound(s, cnt, temp) + 4 * EPS
    e = torch.exp(rp.double() - lp) if ref else torch.zeros_like(lp)
    ww = live.double() * (1 if w is None else w64)
    assert ((logp.cpu().double() - lp).abs() <= E + 2 * EPS * lp.abs()).all()
    assert ((kl.cpu().double() - kl64.detach()).abs() <= live * ((e - 1).abs() * E + E * E * e + 4 * EPS * kl64.detach())).all()
    term = ((ratio.detach() * adv.double()).abs() * E + b32 * ((e - 1).abs() * E + E * E * e)) * ww * scale
    assert abs(loss.item() - total.item()) <= term.sum().item() + 8 * EPS * (abs(total.item()) + scale * (ww * (ratio.detach() * adv.double()).abs()).sum().item())
    dcoef = ((ratio.detach() * adv.double()).abs() + b32 * e) * ww * scale * (E + 8 * EPS)
    check_gradient(d, s, act, p, live, coef.detach() / temp, dcoef / temp, E, n)
    return loss, logp, kl, d


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_policy_loss(rows, n, ragged, dtype):
    s, act, n_cand, cnt, g = cand_case(rows, n, dtype, ragged)
    policy_check(s, act, n_cand, cnt, g)
    policy_check(s, act, n_cand, cnt, g, ref=False, weight=False, reduction="sum", lo=0.1, hi=0.1)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,ld,off", [(9, 50, 56, 0), (9, 50, 53, 3), (6, 1000, 1001, 1), (5, 3001, 3008, 8), (3, 30000, 30007, 5), (2, 150001, 150004, 2)])
def test_pitched_rows_and_in_place(rows, n, ld, off, dtype):
    s, act, n_cand, cnt, g = cand_case(rows, n, dtype, False, seed=3)
    wide = torch.full((rows * ld + off,), 7.0, dtype=dtype, device="cuda")
    v = wide[off:off + rows * ld].view(rows, ld)[:, :n]
    v.copy_(s)
    state = g.get_state()
    want = policy_check(s, act, n_cand, cnt, g)
    g.set_state(state)
    got = policy_check(s, act, n_cand, cnt, g, dev=v)
    logp, stats = losses.log_prob(v, act.cuda(), temperature=0.9)
    dl = torch.randn(rows, device="cuda")
    grad = losses.log_prob_backward(v, act.cuda(), stats, dl, temperature=0.9)
    E = rel_bound(s, cnt, 1.3)
    assert ((got[1] - want[1]).abs().cpu().double() <= 2 * E + 4 * EPS * want[1].abs().cpu().double()).all()
    # the gradient over the scores themselves: the same values, what lies beside the rows untouched
    rest = wide.clone()
    L, c = _lib.lib(), (lambda t: t.data_ptr())
    da = act.cuda()
    from cuke_b200.scoring import _stream
    _lib.check(L.kge_log_prob_backward(c(v), 0 if dtype == torch.float32 else 1, ld, rows, n, None, c(da), 64, 0.9, c(stats), c(dl), c(v), ld, _stream()))
    assert torch.equal(v, grad)
    rest[off:off + rows * ld].view(rows, ld)[:, :n].copy_(grad)
    assert torch.equal(wide, rest)
    v.copy_(s)
    old, adv = torch.zeros(rows, device="cuda") - 3, torch.ones(rows, device="cuda")
    ws = torch.empty(L.kge_candidates_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")

    def step(d):         # the gradient into a buffer of the same pitch and offset, or over the scores: the same bits
        loss, lp, kl = (torch.empty(k, device="cuda") for k in (1, rows, rows))
        _lib.check(L.kge_policy_loss(c(v), 0 if dtype == torch.float32 else 1, ld, rows, n, None, c(da), 64, 1.0, c(old), None, c(adv), None, 0.2, 0.2, 0.0,
                                     1.0 / rows, c(loss), c(lp), c(kl), c(d), ld, c(ws), ws.numel(), _stream()))
        return loss, lp, kl

    other = rest.clone()
    apart = other[off:off + rows * ld].view(rows, ld)[:, :n]
    ref = step(apart)
    assert all(torch.equal(a, b) for a, b in zip(step(v), ref)) and torch.equal(v, apart)
    assert torch.equal(wide, other)
    packed = losses.policy_loss(apart.copy_(s), da, old, adv)        # another alignment may add in another order
    assert (packed[3].double() - v.double()).abs().max() <= (2.0 ** -7 if dtype == torch.bfloat16 else 4 * E.max().item()) * v.double().abs().max()


@gpu
@pytest.mark.parametrize("n", [4, 700, 9000, 60000, 300000])
def test_rows_that_take_no_part(n):
    """-infinity, the type's lowest value, NaN and +infinity in scores; ids outside the row; counts outside [0, n]."""
    from cuke_b200 import scoring
    scoring.device_flags()
    low, inf, nan = torch.finfo(torch.float32).min, float("inf"), float("nan")
    s = torch.randn(10, n, generator=torch.Generator().manual_seed(1))
    s[0] = -inf                    # nothing to choose
    s[1] = low                     # uniform
    s[2, 1:] = -inf                # one candidate left
    s[3, 1:] = low                 # the same through the lowest value
    s[4, 2] = nan
    s[5, 2] = inf
    act = torch.tensor([0, 1, 0, 0, 1, 1, -1, n, -7, 1])
    cnt = torch.tensor([n, n, n, n, n, n, n, n, n, -5], dtype=torch.int32)
    c = lambda t: t.cuda()  # noqa: E731
    logp, stats = losses.log_prob(c(s), c(act), n_cand=c(cnt))
    assert scoring.device_flags() == _lib.ERR_ID_RANGE
    lp = logp.cpu()
    assert lp[0] == 0 and abs(lp[1].item() + np.log(n)) < 1e-4 and lp[2] == 0 and lp[3] == 0 and torch.isnan(lp[4]) and torch.isnan(lp[5])
    assert (lp[6:] == 0).all()
    d = losses.log_prob_backward(c(s), c(act), stats, torch.ones(10, device="cuda"), n_cand=c(cnt)).cpu()
    scoring.device_flags()
    assert (d[0] == 0).all() and (d[2] == 0).all() and (d[3] == 0).all() and torch.isnan(d[4]).all() and (d[6:] == 0).all()
    assert (d[1, 0] + 1 / n).abs() < 1e-6 and (d[1, 1] - 1 + 1 / n).abs() < 1e-6
    old, adv = torch.zeros(10), torch.ones(10)
    loss, lp, kl, d = losses.policy_loss(c(s), c(act), c(old), c(adv), n_cand=c(cnt), weight=torch.tensor([1., 1, 1, 1, 0, 0, 1, 1, 1, 1]).cuda())
    assert scoring.device_flags() == _lib.ERR_ID_RANGE
    assert torch.isfinite(loss).all() and torch.isfinite(d).all() and (d[4:] == 0).all() and (d[0] == 0).all()
    empty = losses.policy_loss(c(s[:, :0]), torch.full((10,), -1, device="cuda"), c(old), c(adv))
    assert empty[0].item() == 0 and empty[3].shape == (10, 0)
    none = losses.policy_loss(c(s[:0]), c(act[:0]), c(old[:0]), c(adv[:0]))
    assert none[0].item() == 0 and none[3].shape == (0, n)


@gpu
@pytest.mark.parametrize("rows,n", [(3, 5), (2, 3000)])
def test_policy_against_differences(rows, n):
    """Central differences of the 64-bit loss with respect to a few scores (error h^2 / 6 |f'''| < 1e-7 at h = 1e-3)."""
    s, act, n_cand, cnt, g = cand_case(rows, n, torch.float32, False, seed=11)
    live, lp, p = cand_ref(s, act, cnt, 1.0)
    old, ref, adv = (lp - 0.05).float(), (lp + 0.1).float(), torch.randn(rows, generator=g)
    c = lambda t: t.cuda()  # noqa: E731
    d = losses.policy_loss(c(s), c(act), c(old), c(adv), ref_logp=c(ref), kl_coef=0.5)[3].cpu()
    f = lambda x: policy64(cand_ref(x, act, cnt, 1.0)[1], live, old.double(), adv.double(), ref.double(), None, 0.2, 0.2, 0.5, 1.0 / rows)[0].item()  # noqa: E731
    for r in range(rows):
        for j in {int(act[r]), 0, n // 2, n - 1}:
            x = s.double()
            x[r, j] += 1e-3
            up = f(x)
            x[r, j] -= 2e-3
            assert abs((up - f(x)) / 2e-3 - d[r, j].item()) < 1e-6


@gpu
def test_two_graphs_and_two_streams():
    """Calls captured into two graphs and calls on two streams share nothing: replays in any order give the eager results."""
    jobs = []
    for k, (rows, n) in enumerate([(64, 50), (70, 5000)]):
        s, act, _, _, g = cand_case(rows, n, torch.float32, False, seed=k)
        old, adv = torch.randn(rows, generator=g) - 5, torch.randn(rows, generator=g)
        jobs.append([t.cuda() for t in (s, act, old, adv)])
    eager = [losses.policy_loss(*j) for j in jobs]
    pe = [losses.preference_loss(j[2], j[0]) for j in jobs]
    graphs, outs, side = [], [], torch.cuda.Stream()
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append((losses.policy_loss(*j), losses.preference_loss(j[2], j[0])))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, e, q in zip(outs, eager, pe):
            assert all(torch.equal(a, b) for a, b in zip(o[0], e)) and all(torch.equal(a, b) for a, b in zip(o[1], q))
            for t in (*o[0], *o[1]):
                t.fill_(3)
        torch.cuda.synchronize()
    got = []
    for j, st in zip(jobs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([losses.policy_loss(*j) for _ in range(20)][-1])
    torch.cuda.synchronize()
    for o, e in zip(got, eager):
        assert all(torch.equal(a, b) for a, b in zip(o, e))
