"""Every form of the kernels of the losses over scores: sums in which a single omitted or doubled candidate shows, and the forms for
long rows against the definitions in 64 bits, with counts that cut anywhere, any alignment, and gradients over the scores."""
import math

import pytest
import torch

from cuke_b200 import _lib, losses
from cuke_b200.scoring import _stream

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                            # half a step of fp32, relative
BF = 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


def form(rows, n, dtype, policy):
    """The form that scores (rows, n) take where the gradient has the alignment of the scores: lanes in registers, threads of a row in
    shared memory and CTAs that share it, or passes."""
    nv = n // (4 if dtype == F32 else 8)
    for lim, name in ((8, "8 lanes, 1"), (16, "8 lanes, 2"), (32, "8 lanes, 4"), (64, "8 lanes, 8")):
        if nv <= lim:
            return name
    if nv <= 128 and rows <= 148 * 16:
        return "32 lanes"
    if nv <= (128 if dtype == F32 else 96):
        return "16 lanes"
    for lim, name in ((512, "32 threads"), (1024, "64 threads"), (2048, "128 threads")):
        if nv <= lim:
            return name
    ctas = next((c for c in (1, 2, 4, 8) if nv <= c * 4608), 16)
    if ctas > 8 or rows * ctas < 32 or (not policy and ctas > 1 and rows * ctas >= 148 * 3):
        return "passes"
    return f"256 threads x {ctas}"


# rows, n in fp32, the form of the policy loss; bf16 has twice as many candidates (and another odd one)
SHAPES = [(40, 35, "8 lanes, 1"), (40, 67, "8 lanes, 2"), (40, 127, "8 lanes, 4"), (40, 251, "8 lanes, 8"), (40, 509, "32 lanes"),
          (2400, 381, "16 lanes"), (40, 701, "32 threads"), (40, 2049, "32 threads"), (40, 4093, "64 threads"), (40, 8190, "128 threads"),
          (40, 9001, "256 threads x 1"), (40, 15000, "256 threads x 1"), (40, 18431, "256 threads x 1"), (40, 30001, "256 threads x 2"),
          (60, 36863, "256 threads x 2"), (40, 60003, "256 threads x 4"), (40, 120001, "256 threads x 8"), (3, 147455, "passes"),
          (2, 9001, "passes"), (2, 200003, "passes")]


def shape(k, dtype):
    rows, n, name = SHAPES[k]
    n = n if dtype == F32 else 2 * n + (1 if rows < 1000 else 0)
    assert form(rows, n, dtype, True) == name
    return rows, n, name


def launches(call):
    before = _lib.lib().kge_launch_count()
    out = call()
    return out, _lib.lib().kge_launch_count() - before


def counts(rows, n, dtype, g):
    """Counts that cut a row everywhere: at the ends, around every eighth of its vectors, and at random."""
    V = 4 if dtype == F32 else 8
    cnt = (torch.rand(rows, generator=g) * (n + 1)).long().clamp(max=n)
    step = max(1, (n // V + 7) // 8) * V
    edges = [n, n - 1, 1, 0, 2, V, n - V] + [e for k in range(1, 8) for e in (k * step - 1, k * step, k * step + 1, k * step + 3)]
    for i, e in enumerate(edges[: max(1, rows - 6)]):
        cnt[i] = min(max(e, 0), n)
    return cnt


def chosen(cnt, g):
    """A chosen candidate of every row that has one: first, last, or anywhere; none in one row."""
    act = (torch.rand(len(cnt), generator=g) * cnt).long()
    act[::5] = 0
    act[1::5] = cnt[1::5] - 1
    act = torch.minimum(act, cnt - 1).clamp(min=0)
    act[cnt == 0] = -1
    if len(cnt) > 9:
        act[9] = -1
    return act


def layout(s, pad, off):
    """s in a buffer with rows `pad` elements apart and `off` elements into it, and what lies beside them."""
    rows, n = s.shape
    wide = torch.full((off + rows * (n + pad),), 7.0, dtype=s.dtype, device="cuda")
    v = wide[off:].view(rows, n + pad)[:, :n]
    v.copy_(s)
    return wide, v


def policy_over_scores(v, act, cnt, old, adv, temp):
    """The policy loss with its gradient written over the scores v (any pitch)."""
    L, p = _lib.lib(), (lambda t: t.data_ptr())
    rows, n = v.shape
    ws = torch.empty(L.kge_candidates_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    loss, lp, kl = (torch.empty(k, device="cuda") for k in (1, rows, rows))
    ld = v.stride(0)
    _lib.check(L.kge_policy_loss(p(v), 0 if v.dtype == F32 else 1, ld, rows, n, None if cnt is None else p(cnt), p(act), 64, temp, p(old), None, p(adv), None,
                                 0.2, 0.2, 0.0, 1.0, p(loss), p(lp), p(kl), p(v), ld, p(ws), ws.numel(), _stream()))
    return loss, lp, kl, v


PASSES, ROWS = (2, 4), (1, 2)               # launches of log_prob and of the policy loss


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("k", range(len(SHAPES)))
def test_equal_scores(k, ragged, dtype):
    """Equal scores: S counts the candidates exactly (fp32 holds integers up to 2^24), so one too few or too many moves logp = -log(count)
    by 1 / count.  The logarithm is good to 2^-22 (two steps of one exponential), the result is rounded once to fp32."""
    rows, n, name = shape(k, dtype)
    g = torch.Generator().manual_seed(k)
    cnt = counts(rows, n, dtype, g) if ragged else torch.full((rows,), n)
    act = chosen(cnt, g)
    live = act >= 0
    s = torch.full((rows, n), 1.5, dtype=dtype)
    s[torch.arange(n)[None] >= cnt[:, None]] = float("nan")
    da, dc = act.cuda(), cnt.to(torch.int32).cuda() if ragged else None
    ones = torch.ones(rows, device="cuda")
    live, many = live.cuda(), cnt.cuda()[:, None].double().clamp(min=1)
    want = torch.where(live, -torch.log(many[:, 0]), torch.zeros_like(many[:, 0]))
    onehot = torch.zeros(rows, n, dtype=torch.float64, device="cuda").scatter_(1, da.clamp(min=0)[:, None], live[:, None].double())
    valid = (torch.arange(n, device="cuda")[None] < cnt.cuda()[:, None]) & live[:, None]
    unit = torch.where(onehot > 0, (many - 1) / many, -1 / many) * valid

    def check(logp, d, factor):
        assert ((logp.double() - want).abs() <= 2.0 ** -22 + EPS * want.abs()).all()
        d, ref = d.double(), factor.double()[:, None] * unit
        # the row's exponential of logp (2 steps), 1 / S, four factors, and the output's rounding
        assert ((d - ref).abs() <= (16 * EPS + (BF if dtype == BF16 else 0)) * ref.abs()).all()
        if dtype == F32 and n > 1:           # the others lose the same each, and together what the chosen one gains, to three roundings
            others = d * (1 - onehot)
            each = others.gather(1, others.abs().argmax(1, keepdim=True))
            assert torch.equal(others[valid & (onehot == 0)], each.expand(rows, n)[valid & (onehot == 0)])
            gain = (d * onehot).sum(1)
            assert ((gain + each[:, 0] * (many[:, 0] - 1)).abs() <= 4 * EPS * gain.abs()).all()

    old, adv = want.float(), ones
    factor = torch.exp(want - old.double()).neg()              # d(loss)/d(logp) = -ratio
    for pad, off in ((0, 0), (3, 1)):
        _, v = layout(s, pad, off)
        (logp, stats), used = launches(lambda: losses.log_prob(v, da, n_cand=dc))
        lname = form(rows, n, dtype, False)
        assert used == (PASSES if lname == "passes" else ROWS)[0]
        check(logp, losses.log_prob_backward(v, da, stats, ones, n_cand=dc), ones)
        (loss, lp, kl, d), used = launches(lambda: policy_over_scores(v, da, dc, old, adv, 1.0))
        assert used == (PASSES if name == "passes" else ROWS)[1] or used == 1
        check(lp, d, factor)
    _, v = layout(s, 3, 1)                   # the gradient at another alignment: passes
    if n > 1:
        loss, lp, kl, d = losses.policy_loss(v, da, old, adv, n_cand=dc, reduction="sum")
        check(lp, d, factor)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("k", [i for i, q in enumerate(SHAPES) if q[2].startswith("256") or q[2] == "passes"])
def test_long_rows_against_64_bits(k, ragged, dtype):
    """log_prob, its gradient and the policy loss, packed and pitched, with the gradient over the scores.

    Relative error of a row's sum: arguments of the exponentials 6 A half-steps (A the spread of scores / T; rescalings by new maxima
    telescope within it), each exponential 4, at most 33 additions behind one another, 14 rescalings of 5: 6 A + 112.  So for logp, absolute."""
    rows, n, name = shape(k, dtype)
    g = torch.Generator().manual_seed(100 + k)
    temp = 0.8
    cnt = counts(rows, n, dtype, g) if ragged else torch.full((rows,), n)
    act = chosen(cnt, g)
    s = (torch.randn(rows, n, generator=g) * 3).to(dtype)
    inside = torch.arange(n)[None] < cnt[:, None]
    s[~inside] = float("nan")
    if rows > 4:                             # half of a row without probability, and a whole one
        s[rows - 3, : n // 2] = -float("inf")
        act[rows - 3] = cnt[rows - 3] - 1
        s[rows - 4] = -float("inf")
    da, dc, inside = act.cuda(), cnt.to(torch.int32).cuda() if ragged else None, inside.cuda()
    x = (s.cuda().double() / temp).masked_fill(~inside, -float("inf"))
    live = (da >= 0) & (x > -float("inf")).any(1)
    lse = torch.where(live, torch.logsumexp(x, 1), torch.zeros_like(x[:, 0]))
    want = torch.where(live, x.gather(1, da.clamp(min=0)[:, None])[:, 0] - lse, torch.zeros_like(lse))
    p = torch.where(live[:, None] & inside, torch.exp(x - lse[:, None]), torch.zeros_like(x))
    onehot = torch.zeros_like(p).scatter_(1, da.clamp(min=0)[:, None], live[:, None].double())
    rest = torch.where(onehot > 0, (p * (1 - onehot)).sum(1, keepdim=True), -p)
    top = x.masked_fill(x == -float("inf"), -1e30).max(1).values
    low = x.masked_fill(x == -float("inf"), 1e30).min(1).values
    A = torch.where(live, top - low, torch.zeros_like(top)).clamp(min=0)
    E = EPS * (6 * A + 112)

    def check(logp, d, coef, dcoef):
        assert ((logp.double() - want).abs() <= E + 2 * EPS * want.abs()).all()
        ref = coef[:, None] * rest
        tol = (dcoef[:, None] + coef.abs()[:, None] * (3 * E[:, None] + 8 * EPS)) * rest.abs() + 1e-37 * (1 + coef.abs()[:, None])
        if dtype == BF16:
            tol = 1.01 * tol + BF * ref.abs()
        assert ((d.double() - ref).abs() <= tol).all()

    r = lambda: torch.randn(rows, generator=g).cuda()  # noqa: E731
    dlogp, adv = r(), r()
    delta = 0.3 * torch.randn(rows, generator=g).double().cuda()
    for edge in (math.log(0.8), math.log(1.2)):              # a ratio on a border has no defined gradient
        delta = torch.where((delta - edge).abs() < 2e-3, delta + 8e-3, delta)
    old = (want - delta).float()
    ratio, A64 = torch.exp(want - old.double()), adv.double()
    held = ((A64 > 0) & (ratio > 1.2)) | ((A64 < 0) & (ratio < 0.8))
    coef = torch.where(held | ~live, torch.zeros_like(ratio), -ratio * A64) / temp
    term = torch.where(live, -torch.minimum(ratio * A64, ratio.clamp(0.8, 1.2) * A64), torch.zeros_like(ratio))
    for pad, off in ((0, 0), (5, 3)):
        wide, v = layout(s, pad, off)
        rim = wide.clone()
        (logp, stats), used = launches(lambda: losses.log_prob(v, da, n_cand=dc, temperature=temp))
        assert used == (PASSES if form(rows, n, dtype, False) == "passes" else ROWS)[0]
        c = torch.where(live, dlogp.double() / temp, torch.zeros_like(ratio))
        check(logp, losses.log_prob_backward(v, da, stats, dlogp, n_cand=dc, temperature=temp), c, 4 * EPS * c.abs())
        (loss, lp, kl, d), used = launches(lambda: policy_over_scores(v, da, dc, old, adv, temp))
        assert used == (PASSES if name == "passes" else ROWS)[1]
        check(lp, d, coef, (ratio * A64).abs() / temp * (E + 8 * EPS))
        assert (kl == 0).all()
        assert abs(loss.item() - term.sum().item()) <= (((ratio * A64).abs() * (E + 8 * EPS) * live).sum() + 8 * EPS * term.abs().sum()).item()
        rim[off:].view(rows, n + pad)[:, :n].copy_(d)        # what lies beside the rows is as it was
        assert torch.equal(rim.view(torch.int32 if dtype == F32 else torch.int16), wide.view(torch.int32 if dtype == F32 else torch.int16))


PREFERENCE = [(300, 1), (300, 4), (301, 23), (300, 24), (130, 61), (130, 64), (4800, 68), (4740, 131), (4740, 447), (1200, 200), (1190, 333), (1190, 2047),
              (40, 300), (800, 701), (800, 8191), (40, 2044), (7, 9001), (5, 8200), (160, 4100), (200, 40001), (310, 33000), (2, 70001)]


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("rows,n", PREFERENCE)
def test_equal_preferences(rows, n, mask):
    """z = 1 under the square loss: every term is 1, every slope 2, and their sums are exact in fp32, so that one pair too few or too many
    moves d(pos) by 1 / count.  Three roundings: w / count, times 2 beta (exact), times the sum."""
    g = torch.Generator().manual_seed(n)
    m = torch.ones(rows, n, dtype=torch.bool)
    if mask:
        m = torch.rand(rows, n, generator=g) > 0.4
        m[::7] = False
        m[1::7] = True
    neg = torch.where(m, torch.zeros(rows, n), torch.full((rows, n), float("nan")))
    w = torch.rand(rows, generator=g) + 0.5
    cnt = m.sum(1).double()
    w64 = torch.where(cnt > 0, w.double(), torch.zeros(rows, dtype=torch.float64))
    for pad, off in ((0, 0), (4, 4), (3, 1)):
        _, v = layout(neg, pad, off)
        dm = layout(m, pad, off)[1] if mask else None
        loss, dpos, dneg = losses.preference_loss(torch.ones(rows, device="cuda"), v, mask=dm, weight=w.cuda(), kind="square")
        assert ((dpos.cpu().double() - 2 * w64).abs() <= 3 * EPS * 2 * w64).all()
        want = torch.where(m, (-2 * w64 / cnt.clamp(min=1))[:, None].expand(rows, n), torch.zeros(rows, n, dtype=torch.float64))
        assert ((dneg.cpu().double() - want).abs() <= 3 * EPS * want.abs()).all()
        assert abs(loss.item() - w64.sum().item()) <= 3 * EPS * w64.sum().item()


@pytest.mark.parametrize("rows,n", [(300, 3), (301, 24), (130, 61), (4740, 131), (1200, 200), (40, 300), (7, 9001), (160, 4100), (1, 70000)])
@pytest.mark.parametrize("kind", ["logistic", "square"])
def test_preference_gradient_over_the_scores(rows, n, kind):
    """dneg may be neg itself: the bits of the call with a buffer of its own, and nothing beside the rows changes."""
    L, p = _lib.lib(), (lambda t: None if t is None else t.data_ptr())
    g = torch.Generator().manual_seed(n + rows)
    neg, pos, weight = torch.randn(rows, n, generator=g), torch.randn(rows, generator=g).cuda(), torch.rand(rows, generator=g).cuda()
    m = (torch.rand(rows, n, generator=g) > 0.3).cuda()
    code = _lib.PREFERENCE_KINDS[kind]
    ws = torch.empty(L.kge_preference_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    for pad, off in ((0, 0), (4, 4), (3, 1)):
        for mask in (None, m):
            wide, v = layout(neg, pad, off)
            other, apart = layout(neg, pad, off)

            def call(d):
                loss, dpos = torch.empty(1, device="cuda"), torch.empty(rows, device="cuda")
                _lib.check(L.kge_preference_loss(p(pos), None, p(v), n + pad, None, 0, p(mask), n, p(weight), rows, n, code, 0.7, 0.1, 0.0, 1.0, p(loss),
                                                 p(dpos), p(d), n + pad, p(ws), ws.numel(), _stream()))
                return loss, dpos

            want = call(apart)
            got = call(v)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(wide, other)
