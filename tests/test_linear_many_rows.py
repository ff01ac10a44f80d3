"""The bias gradient of the matrix product over the most rows a call admits."""
import pytest
import torch

from cuke_b200 import _lib
from cuke_b200.scoring import _stream

pytestmark = pytest.mark.gpu


def test_bias_gradient_of_equal_rows():
    """2^30 rows of one value: the sum is exact in 64 bits, so only its rounding to bf16 (2^-8 relative) and 64 + 16 half-steps of fp32 are
    left.  33/64: 64 of them make 33, of which a running fp32 sum past 2^24 (in steps of 2) takes 32 every time."""
    m, n, L = 1 << 30, 8, _lib.lib()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    dout = torch.full((m, n), 33 / 64, dtype=torch.bfloat16, device="cuda")
    db = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(L.kge_linear_workspace_bytes(m, 8, n, 0, 1), dtype=torch.uint8, device="cuda")
    _lib.check(L.kge_linear_backward(dout.data_ptr(), n, None, 8, None, n, None, m, 8, n, 0, None, 8, None, db.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
    want = m * 33 / 64
    assert ((db.double() - want).abs() <= (2.0 ** -8 + 80 * 2.0 ** -24) * want).all()
