"""An output may lie over its input with the same row pitch only: the C interface refuses another one before anything is launched."""
import os

import pytest

from cuke_b200 import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
A, B = 4096, 8192                           # stand-ins for device addresses: a refused call never follows them


def error():
    return _lib.lib().kge_last_error()


@pytest.mark.parametrize("x,residual,out", [(A, None, A), (A, B, B), (A, A, A)])
def test_dropout(x, residual, out):
    L = _lib.lib()
    ldx, ldr = (9, 8) if out == x else (8, 9)
    assert L.kge_dropout(x, 0, 4, 8, ldx, residual, ldr, out, 8, 0.5, 1, 0, 0, None, None) == -4
    assert error() == b"kge_dropout: out may be x or residual only with the same row pitch"


def test_preference():
    rc = _lib.lib().kge_preference_loss(A, None, B, 8, None, 0, None, 0, None, 4, 8, 0, 1.0, 0.0, 0.0, 1.0, A, A, B, 9, A, 1 << 20, None)
    assert rc == -4 and error() == b"kge_preference_loss: dneg may be neg only with the same row pitch"


@pytest.mark.gpu                            # without a device these calls are refused for that first
@pytest.mark.parametrize("fn", ["kge_policy_loss", "kge_log_prob_backward"])
def test_candidates(fn):
    L = _lib.lib()
    head = (A, 0, 8, 4, 8, None, B, 64, 1.0)
    if fn == "kge_policy_loss":
        rc = L.kge_policy_loss(*head, B, None, B, None, 0.2, 0.2, 0.0, 1.0, B, B, B, A, 9, B, 1 << 26, None)
    else:
        rc = L.kge_log_prob_backward(*head, B, B, A, 9, None)
    assert rc == -4 and error() == fn.encode() + b": dscores may be scores only with the same row pitch"
