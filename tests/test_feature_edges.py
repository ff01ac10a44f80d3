"""Calls at the edges of what the operators over features and losses allow: nothing in them, several host threads, refused layouts."""
import threading

import pytest
import torch

from cuke_b200 import _lib, features, losses, scoring

pytestmark = pytest.mark.gpu


def ids(rows, value=0, dtype=torch.int64):
    return torch.full((rows,), value, dtype=dtype, device="cuda")


def test_nothing_in_them():
    none = torch.empty(0, 7, device="cuda")
    zero = torch.zeros(0, device="cuda")
    loss, logp, kl, d = losses.policy_loss(none, ids(0), zero, zero)
    assert loss.item() == 0 and logp.numel() == kl.numel() == 0 and d.shape == (0, 7)
    empty, ones = torch.empty(3, 0, device="cuda"), torch.ones(3, device="cuda")
    loss, logp, kl, d = losses.policy_loss(empty, ids(3, -1), ones, ones)
    assert loss.item() == 0 and (logp == 0).all() and (kl == 0).all() and d.shape == (3, 0)
    logp, stats = losses.log_prob(empty, ids(3, -1))
    assert (logp == 0).all() and losses.log_prob_backward(empty, ids(3, -1), stats, ones).shape == (3, 0)
    loss, dpos, dneg = losses.preference_loss(ones, empty)
    assert loss.item() == 0 and (dpos == 0).all() and dneg.shape == (3, 0)
    assert features.dropout(none, 0.5, 1).shape == (0, 7)
    assert features.dropout(torch.ones(2, 3, 4, device="cuda"), 0.0, 1).eq(1).all()
    assert scoring.device_flags() == 0


def test_refused_layouts():
    q = torch.ones(3, 4, device="cuda")
    x, w = torch.randn(20, 16, device="cuda").bfloat16(), torch.randn(16, 16, device="cuda").bfloat16()
    for call, error in ((lambda: losses.preference_loss(torch.ones(6, device="cuda")[::2], q), ValueError),
                        (lambda: losses.log_prob(q.t(), ids(4)), ValueError),
                        (lambda: losses.log_prob(q[:1].expand(3, 4), ids(3)), ValueError),
                        (lambda: losses.log_prob(q, ids(3).cpu()), ValueError),
                        (lambda: losses.log_prob(q, ids(3, dtype=torch.int16)), TypeError),
                        (lambda: losses.log_prob(q.half(), ids(3)), TypeError),
                        (lambda: losses.log_prob(q, ids(3), temperature=0.0), _lib.KgeError),
                        (lambda: features.linear(x, w, out=x), _lib.KgeError),
                        (lambda: features.linear(torch.randn(321, device="cuda").bfloat16()[1:].view(20, 16), w), _lib.KgeError),
                        (lambda: features.linear(x[:, :12], w[:12]), _lib.KgeError)):
        with pytest.raises(error):
            call()


def work(seed, out):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        for i in range(12):
            m, k, n = [(300, 136, 264), (17, 64, 72), (5000, 72, 200)][(i + seed) % 3]
            x, w, b = r(m, k).bfloat16(), r(k, n).bfloat16(), r(n).bfloat16()
            y, s = features.linear(x, w, b, act="silu", save_preact=True)
            scores = r(400, 999)
            action = torch.randint(0, 999, (400,), generator=g, device="cuda")
            out += [y, *features.linear_backward(y, x, w, s, act="silu"),
                    *losses.policy_loss(scores, action, torch.zeros(400, device="cuda"), torch.ones(400, device="cuda")),
                    *losses.preference_loss(scores[:, 0].contiguous(), scores), features.dropout(scores, 0.3, seed, 1, i)]
    stream.synchronize()


def test_two_host_threads_on_streams_of_their_own():
    alone, together = [[], []], [[], []]
    for seed in (0, 1):
        work(seed, alone[seed])
    threads = [threading.Thread(target=work, args=(seed, together[seed])) for seed in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, together):
        assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))
