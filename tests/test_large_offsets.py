"""The operators over features and losses on tensors of more than 2^31 elements: the last rows, whose offsets pass 32 bits, are what
a call on those rows alone gives."""
import numpy as np
import pytest
import torch

from cuke_b200 import features, losses, scoring
from oracle import sampler_model

pytestmark = pytest.mark.gpu
BF, F32 = 2.0 ** -8, 2.0 ** -24


def test_dropout():
    n = (1 << 31) + 4109
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = features.dropout(x, 0.25, 99, 4, 7)
    first = (n - 4101) // 4 * 4
    q = np.arange(first // 4, (n + 3) // 4, dtype=np.uint64)
    full = lambda v: np.full(q.shape, v, dtype=np.uint64)  # noqa: E731
    w = sampler_model.philox4x32_10(q & np.uint64(0xFFFFFFFF), q >> np.uint64(32), full(4), full(0x80000007), 99, 0)
    keep = (np.stack(w, 1).reshape(-1)[: n - first] >= np.uint64(1 << 30))
    want = torch.from_numpy(np.where(keep, np.float32(1 / 0.75), np.float32(0))).to(torch.bfloat16)      # one rounding of the same product
    assert torch.equal(y[first:].cpu(), want)
    # rows with a pitch: the same mask, by row-major element number
    rows, dim = 1 << 19, 4100
    wide = torch.ones(rows, dim + 4, dtype=torch.bfloat16, device="cuda")[:, :dim]
    got = features.dropout(wide, 0.25, 99, 4, 7, out=torch.empty(rows, dim + 4, dtype=torch.bfloat16, device="cuda")[:, :dim])
    assert rows * dim > n and torch.equal(got[: n // dim].reshape(-1), y[: n // dim * dim])


def test_preference():
    rows, n = 36000, 60000
    pos, neg = torch.randn(rows, device="cuda"), torch.randn(rows, n, device="cuda")
    loss, dpos, dneg = losses.preference_loss(pos, neg, beta=0.5)
    l2, p2, n2 = losses.preference_loss(pos[-3:].contiguous(), neg[-3:], beta=0.5)
    assert torch.equal(dneg[-3:], n2) and ((dpos[-3:] - p2).abs() <= n * F32 * p2.abs()).all()
    l1 = sum(losses.preference_loss(pos[i:i + 9000].contiguous(), neg[i:i + 9000], beta=0.5)[0].double().item() for i in range(0, rows, 9000))
    assert abs(loss.item() - l1) <= 8 * F32 * l1 + n * F32 * l1


@pytest.mark.parametrize("rows,n", [(2200, 1_000_000), (8_600_000, 250), (144_000, 15_000)])
def test_candidates(rows, n):
    s = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda").normal_()
    a = torch.randint(0, n, (rows,), device="cuda")
    old, adv = torch.randn(rows, device="cuda") - 8, torch.randn(rows, device="cuda")
    loss, logp, kl, d = losses.policy_loss(s, a, old, adv, reduction="sum")
    lp, stats = losses.log_prob(s, a)
    back = losses.log_prob_backward(s, a, stats, adv)
    # the form of the kernel follows the number of rows, and with it the order of additions: n additions of a sum at most
    tail = slice(rows - 5, rows)
    x = torch.log_softmax(s[tail].double(), 1)
    want = x.gather(1, a[tail, None])[:, 0]
    assert ((logp[tail].double() - want).abs() <= (n / 32 + 64) * F32 + 2 * F32 * want.abs()).all()
    assert ((lp[tail].double() - want).abs() <= (n / 32 + 64) * F32 + 2 * F32 * want.abs()).all()
    p = torch.exp(x)
    onehot = torch.zeros_like(p).scatter_(1, a[tail, None], 1.0)
    ratio = torch.exp(want - old[tail].double())
    A = adv[tail].double()
    dl = torch.where(((A > 0) & (ratio > 1.2)) | ((A < 0) & (ratio < 0.8)), torch.zeros_like(A), -ratio * A)
    E = (n / 32 + 200) * F32                 # of a row's exponentials and their sum, and so of the ratio
    near = ((ratio - 1.2).abs() <= 4 * E * ratio) | ((ratio - 0.8).abs() <= 4 * E * ratio)
    for got, coef, skip in ((d, dl, near), (back, A, torch.zeros_like(near))):
        ref = coef[:, None] * (onehot - p)
        ok = (got[tail].double() - ref).abs() <= (BF + 4 * E) * ref.abs() + 1e-37
        assert ok[~skip].all()
    assert scoring.device_flags() == 0


def test_linear():
    m, k, n = (1 << 20) + 300, 8, 2056
    x, w, b = torch.randn(m, k, device="cuda").bfloat16(), torch.randn(k, n, device="cuda").bfloat16(), torch.randn(n, device="cuda").bfloat16()
    out, slope = features.linear(x, w, b, act="gelu", save_preact=True)
    o2, s2 = features.linear(x[-300:], w, b, act="gelu", save_preact=True)
    assert torch.equal(out[-300:], o2) and torch.equal(slope[-300:], s2)         # eight products a sum: one order
    dx, dw, db = features.linear_backward(out, x, w, slope, act="gelu")
    dz = out[-300:].double() * slope[-300:].double()
    want, size = dz @ w.double().T, dz.abs() @ w.double().abs().T
    # dz rounded to bf16 before the product, n additions, the result's rounding
    assert ((dx[-300:].double() - want).abs() <= (BF + n * 2 * F32) * size + BF * want.abs()).all()
    # zeros and ones: sums below 2^24 are exact in fp32 whatever their order, so only the result's rounding is left
    x, dy = (torch.randint(0, 2, (m, q), device="cuda", dtype=torch.int8).to(torch.bfloat16) for q in (k, n))
    dx, dw, db = features.linear_backward(dy, x, w, need_dx=False)
    want = sum(x[i:i + 65536].double().T @ dy[i:i + 65536].double() for i in range(0, m, 65536))
    assert dx is None and ((dw.double() - want).abs() <= BF * want).all()
    want = sum(dy[i:i + 65536].sum(0, dtype=torch.float64) for i in range(0, m, 65536))
    assert ((db.double() - want).abs() <= BF * want).all()
