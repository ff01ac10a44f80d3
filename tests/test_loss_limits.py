"""Losses over scores at the limits of their terms: coefficients of zero beside infinities, rows that take no part."""
import math

import pytest
import torch

from cuke_b200 import losses

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                            # half a step of fp32, relative
INF = float("inf")


def policy_case(rows=6, n=50, seed=0):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(rows, n, generator=g)
    act = torch.randint(0, n, (rows,), generator=g)
    lp = torch.log_softmax(s.double(), 1).gather(1, act[:, None])[:, 0]
    return s.cuda(), act.cuda(), lp, torch.log_softmax(s.double(), 1)


def test_kl_of_coefficient_zero_is_only_reported():
    """ref - logp of 100, +-infinity and beyond fp32's exponential: the call without a reference, bit for bit, and kl beside it."""
    s, act, lp, _ = policy_case()
    gap = torch.tensor([0.1, 100.0, INF, -INF, -1e30, 88.0])
    ref = (lp + gap.double()).float()
    old, adv = (lp - 0.05).float().cuda(), torch.tensor([1.0, -1.0, 0.5, -0.5, 2.0, 0.0]).cuda()
    loss, logp, kl, d = losses.policy_loss(s, act, old, adv, ref_logp=ref.cuda(), kl_coef=0.0)
    want = losses.policy_loss(s, act, old, adv)
    assert torch.isfinite(loss).all() and torch.isfinite(d).all()
    assert torch.equal(loss, want[0]) and torch.equal(logp, want[1]) and torch.equal(d, want[3])
    assert kl[1] == INF and kl[2] == INF and kl[3] == INF and (kl[[0, 4, 5]] > 0).all() and torch.isfinite(kl[[0, 4, 5]]).all()


def test_advantage_of_zero_beside_a_ratio_past_fp32():
    """exp(100) times an advantage of 0 is 0: the row gives what it gives at a ratio of 1."""
    s, act, lp, _ = policy_case(seed=1)
    ref, zero = (lp + 0.2).float().cuda(), torch.zeros(6, device="cuda")
    for kl_coef in (0.0, 0.3):
        want = losses.policy_loss(s, act, lp.float().cuda(), zero, ref_logp=ref, kl_coef=kl_coef)
        got = losses.policy_loss(s, act, (lp - 100).float().cuda(), zero, ref_logp=ref, kl_coef=kl_coef)
        assert torch.isfinite(got[0]).all() and all(torch.equal(a, b) for a, b in zip(got, want))
    s[2, 3] = float("nan")                  # a row of NaN stays one
    loss, logp, kl, d = losses.policy_loss(s, act, (lp - 100).float().cuda(), zero)
    assert torch.isnan(loss).all() and torch.isnan(logp[2]) and torch.isnan(d[2]).all() and (d[[0, 1, 3, 4, 5]] == 0).all()


def test_kl_gradient_far_below_the_reference():
    """d = ref - logp far below zero: the slope kl_coef (e^d - 1) tends to -kl_coef, down to ref = -infinity.

    Relative error of the gradient: 128 half-steps (argument of the exponentials 6 A with A = 8, sums of 50 terms, the factors)."""
    temp, kl_coef = 0.8, 0.5
    g = torch.Generator().manual_seed(2)
    gap = torch.tensor([2.0, 50.0, 1e4, 1e7, 1e30, 3e38, INF])
    rows, n = len(gap), 50
    s = torch.randn(rows, n, generator=g)
    act = torch.randint(0, n, (rows,), generator=g)
    x = torch.log_softmax(s.double() / temp, 1)
    lp = x.gather(1, act[:, None])[:, 0]
    ref = (lp - gap.double()).float()
    d = ref.double() - lp
    zero, old = torch.zeros(rows, device="cuda"), lp.float().cuda()
    for upto, finite in ((rows, False), (rows - 1, True)):
        c = lambda t: t[:upto].cuda()  # noqa: E731
        loss, _, kl, grad = losses.policy_loss(c(s), c(act), old[:upto], zero[:upto], ref_logp=c(ref), temperature=temp, kl_coef=kl_coef, reduction="sum")
        slope = kl_coef * -torch.expm1(d[:upto])
        onehot = torch.zeros(upto, n, dtype=torch.float64).scatter_(1, act[:upto, None], 1.0)
        want = slope[:, None] / temp * (onehot - torch.exp(x[:upto]))
        assert ((grad.cpu().double() - want).abs() <= 128 * EPS * want.abs()).all()
        kl64 = torch.expm1(d[:upto]) - d[:upto]
        near = torch.where(torch.isinf(kl64), torch.zeros_like(kl64), kl64)
        assert torch.equal(torch.isinf(kl.cpu()), torch.isinf(kl64)) and (kl.cpu().double()[~torch.isinf(kl64)] - near[~torch.isinf(kl64)]).abs().le(
            16 * EPS * near[~torch.isinf(kl64)] + 16 * EPS).all()
        assert torch.isinf(loss).item() is not finite and not torch.isnan(loss).item()


def chosen_of_probability_zero():
    s, act, lp, _ = policy_case(seed=3)
    s[torch.arange(6, device="cuda"), act] = -INF
    return s, act, lp.float().cuda(), (lp + 0.1).float().cuda(), torch.ones(6, device="cuda")


def test_kl_of_a_chosen_candidate_of_probability_zero():
    """logp = -infinity: infinitely far from any reference (kl = +infinity, not NaN)."""
    s, act, old, ref, adv = chosen_of_probability_zero()
    loss, logp, kl, d = losses.policy_loss(s, act, old, adv, ref_logp=ref, kl_coef=0.1)
    assert (logp == -INF).all() and (kl == INF).all() and loss.item() == INF


def test_kl_of_coefficient_zero_beside_a_probability_of_zero():
    s, act, old, ref, adv = chosen_of_probability_zero()
    loss, logp, kl, d = losses.policy_loss(s, act, old, adv, ref_logp=ref)
    assert (logp == -INF).all() and (kl == INF).all() and loss.item() == 0 and (d == 0).all()


@pytest.mark.parametrize("n", [50, 700, 20000])
@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
def test_log_prob_gradient_of_rows_without_a_distribution(n, bad):
    """A row that takes no part has a zero gradient whatever d(logp) holds there."""
    s = torch.randn(5, n, generator=torch.Generator().manual_seed(4)).cuda()
    s[1] = -INF
    act = torch.tensor([0, 1, -1, 0, 2], device="cuda")
    cnt = torch.tensor([n, n, n, 0, n], dtype=torch.int32, device="cuda")
    act[3] = -1
    logp, stats = losses.log_prob(s, act, n_cand=cnt)
    dlogp = torch.tensor([1.0, bad, bad, bad, 1.0], device="cuda")
    d = losses.log_prob_backward(s, act, stats, dlogp, n_cand=cnt)
    assert (logp[1:4] == 0).all() and (d[1:4] == 0).all() and torch.isfinite(d).all() and (d[[0, 4]] != 0).any()


@pytest.mark.parametrize("n", [1, 3, 40])
def test_preference_smoothing_of_one_beside_infinities(n):
    """smoothing = 1 leaves softplus(z): z = -infinity costs nothing, as z = +infinity does without smoothing."""
    pos = torch.zeros(2, device="cuda")
    for value, smoothing in ((INF, 1.0), (3e38, 1.0), (-INF, 0.0), (-3e38, 0.0)):
        neg = torch.full((2, n), value, device="cuda")
        loss, dpos, dneg = losses.preference_loss(pos, neg, smoothing=smoothing, beta=2.0)         # (2 x 3e38 overflows)
        assert loss.item() == 0 and (dpos == 0).all() and (dneg == 0).all()
    loss, dpos, dneg = losses.preference_loss(pos, torch.full((2, n), -INF, device="cuda"), smoothing=1.0)
    assert loss.item() == INF and (dneg != 0).all()


@pytest.mark.parametrize("rows,n,mask", [(1, 1 << 24, False), (2, (1 << 24) + 3, True), (1, 40_000_001, False), (300, 1 << 18, True)])
def test_preference_sums_over_long_rows(rows, n, mask):
    """Equal pairs: the loss is that of one pair and d(pos) its slope, whatever the number of pairs.

    At most 64 additions in fp32 follow one another in a thread before they go to 64 bits; 5 more add a warp and 31 a row's warps; the
    pair itself is good to 16 half-steps (of 1): 120 half-steps of 1 cover all."""
    z, beta = 0.3, 1.0
    pos = torch.full((rows,), z, device="cuda")
    neg = torch.zeros(rows, n, device="cuda")
    m = None
    if mask:
        m = torch.rand(rows, n, device="cuda") > 0.3
        neg = neg.masked_fill(~m, float("nan"))
    loss, dpos, dneg = losses.preference_loss(pos, neg, mask=m, beta=beta, reduction="mean")
    z64 = float(torch.tensor(z, dtype=torch.float32))
    want, slope = math.log1p(math.exp(-z64)), -1 / (1 + math.exp(z64))
    assert abs(loss.item() - want) <= 120 * EPS
    assert ((dpos.double() * rows - slope).abs() <= 120 * EPS).all()
    loss, dpos, _ = losses.preference_loss(pos, neg, mask=m, kind="square", reduction="mean")
    assert abs(loss.item() - z64 * z64) <= 120 * EPS * z64 * z64 and ((dpos.double() * rows - 2 * z64).abs() <= 120 * EPS).all()
