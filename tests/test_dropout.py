"""Dropout with a counter-based mask (kge_dropout, cuke_b200.features.dropout) against a 64-bit statement of it."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

from cuke_b200 import _lib, features
from oracle import sampler_model

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
NULL, SOME, ODD = None, 4096, 4097          # stand-ins for device addresses: a refused call never follows them


def call(x=SOME, dtype=0, rows=4, dim=8, ldx=8, res=NULL, ldr=0, out=SOME, ldo=8, p=0.1, step_dev=NULL):
    return _lib.lib().kge_dropout(x, dtype, rows, dim, ldx, res, ldr, out, ldo, p, 1, 2, 3, step_dev, None)


@needs_lib
@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), -3), (dict(p=1.0), -6), (dict(p=-0.1), -6), (dict(p=float("nan")), -6), (dict(rows=-1), -4), (dict(dim=-1), -4),
    (dict(ldx=7), -4), (dict(ldo=7), -4), (dict(res=SOME, ldr=7), -4), (dict(x=NULL), -1), (dict(out=NULL), -1), (dict(x=ODD), -2),
    (dict(out=ODD, dtype=1), -2), (dict(res=ODD, ldr=8), -2), (dict(step_dev=4100), -2),
    (dict(rows=1 << 58, dim=8, ldx=8, ldo=8), -6)])
def test_refusals(kw, code):
    assert call(**kw) == code
    assert _lib.lib().kge_last_error().startswith(b"kge_dropout: ")


@needs_lib
def test_nothing_to_do():
    assert call(rows=0, x=NULL, out=NULL) == 0 and call(dim=0, x=NULL, out=NULL) == 0


def test_python_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        features.dropout(torch.zeros(2, 2), 0.1, 0)
    with pytest.raises(ValueError, match="contiguous"):
        features.pitch(torch.zeros(4, 4).t(), "x")
    with pytest.raises(ValueError, match="overlap"):
        features.pitch(torch.zeros(1, 4).expand(3, 4), "x")
    assert features.pitch(torch.zeros(4, 6)[:, :5], "x") == 6 and features.pitch(torch.zeros(1, 5), "x") == 5


def keep64(n, p, seed, stream, step):
    """Bool mask of elements 0..n-1."""
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    c = np.full(q.shape, stream, dtype=np.uint64)
    s = np.full(q.shape, 0x80000000 | (step & 0x7FFFFFFF), dtype=np.uint64)
    w = sampler_model.philox4x32_10(q & np.uint64(0xFFFFFFFF), q >> np.uint64(32), c, s, seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    return np.stack(w, 1).reshape(-1)[:n] >= np.uint64(int(p * 2 ** 32))


def check(x, y, keep, p, res=None):
    """Off by the rounding of 1 / (1 - p), of the product and of the sum (2^-24 each, relative to the terms) and by one
    rounding to 16 bits (2^-8 relative to the result)."""
    x64, y64 = x.double().cpu().numpy().reshape(-1), y.double().cpu().numpy().reshape(-1)
    r = np.zeros_like(x64) if res is None else res.double().cpu().numpy().reshape(-1)
    t = np.where(keep, x64 / (1 - p), 0.0)
    ref = t + r
    tol = 3 * 2.0 ** -24 * (np.abs(t) + np.abs(r)) + (2.0 ** -8 * np.abs(ref) if x.dtype == torch.bfloat16 else 0)
    assert (np.abs(y64 - ref) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 3), (3, 1), (5, 7), (2, 1023), (64, 128), (33, 400), (257, 36), (4097, 20), (1, 70001)])
@pytest.mark.parametrize("p,residual", [(0.0, False), (0.1, True), (0.5, False), (0.999, True)])
def test_values(rows, dim, dtype, p, residual):
    g = torch.Generator(device="cuda").manual_seed(rows * 1000 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    r = torch.randn(rows, dim, generator=g, device="cuda").to(dtype) if residual else None
    seed, stream, step = (7 << 40) + 12345, 9, 77
    y = features.dropout(x, p, seed, stream, step, residual=r)
    check(x, y, keep64(rows * dim, p, seed, stream, step), p, r)
    assert torch.equal(y, features.dropout(x, p, seed, stream, step, residual=r))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,ld,off", [(16, 24, 0), (12, 20, 4), (8, 8, 1), (7, 9, 0), (64, 65, 3), (1, 5, 2), (24, 32, 8)])
def test_pitches_and_offsets(dim, ld, off, dtype):
    """Views into wider buffers: values as for the packed tensor, the columns beside the view untouched."""
    rows, p, seed = 37, 0.3, 5
    g = torch.Generator(device="cuda").manual_seed(dim * 100 + ld)
    view = lambda b: b.view(-1)[off:off + rows * ld].view(rows, ld)[:, :dim]  # noqa: E731
    bx, br = (torch.randn(rows * ld + 16, generator=g, device="cuda").to(dtype) for _ in range(2))
    bo = torch.full((rows * ld + 16,), 3.0, device="cuda", dtype=dtype)
    x, r, o = view(bx), view(br), view(bo)
    y = features.dropout(x, p, seed, residual=r, out=o)
    assert y is o
    check(x.contiguous(), o.contiguous(), keep64(rows * dim, p, seed, 0, 0), p, r.contiguous())
    rest = torch.full_like(bo, 3.0)
    view(rest).copy_(o)
    assert torch.equal(bo, rest)
    # mixed pitches: a pitched input into a packed output
    assert torch.equal(features.dropout(x, p, seed, residual=r.contiguous()), o.contiguous())


@pytest.mark.gpu
def test_in_place_and_other_ranks():
    x = torch.randn(6, 5, 8, device="cuda")
    ref = features.dropout(x.view(-1), 0.4, 11, 2, 3)
    assert torch.equal(features.dropout(x, 0.4, 11, 2, 3).view(-1), ref)
    y = x.clone()
    features.dropout(y, 0.4, 11, 2, 3, out=y)
    assert torch.equal(y.view(-1), ref)
    r = torch.randn_like(x)
    want = features.dropout(x, 0.4, 11, 2, 3, residual=r)
    features.dropout(x, 0.4, 11, 2, 3, residual=r, out=r)
    assert torch.equal(r, want)
    assert features.dropout(x[:0], 0.4, 1).shape == (0, 5, 8)
    wide = torch.randn(4, 16, device="cuda")
    with pytest.raises(ValueError, match="pitch"):
        features.dropout(wide[:, :8], 0.1, 0, out=torch.as_strided(wide, (4, 8), (8, 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropped_elements_hide_infinities(dtype):
    keep = keep64(4096, 0.5, 3, 0, 0)
    x = torch.ones(4096, device="cuda", dtype=dtype)
    bad = torch.from_numpy(~keep).cuda()
    x[bad] = torch.tensor([float("inf"), float("nan")], device="cuda", dtype=dtype).repeat(4096)[: int(bad.sum())]
    y = features.dropout(x, 0.5, 3)
    assert torch.equal(y, torch.where(bad, 0.0, 2.0).to(dtype))


@pytest.mark.gpu
def test_gradient_and_rate():
    """The map is linear: <dropout(x), dy> = <x, dropout(dy)>, and a share 1 - p of the elements is kept."""
    n, p = 1 << 20, 0.25
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    y, dx = features.dropout(x, p, 42, 1, 2), features.dropout(dy, p, 42, 1, 2)
    a, b = (y.double() * dy.double()), (x.double() * dx.double())
    assert (a - b).abs().max() <= 4 * 2.0 ** -24 * a.abs().max()         # two roundings a side
    kept = int((y != 0).sum())
    assert abs(kept - n * (1 - p)) < 6 * (n * p * (1 - p)) ** 0.5           # six standard deviations
    for other in ((43, 1, 2), (42, 2, 2), (42, 1, 3)):                      # another seed, stream or step: another mask
        assert abs(int(((features.dropout(x, p, *other) != 0) == (y != 0)).sum()) / n - (p * p + (1 - p) ** 2)) < 0.01


@pytest.mark.gpu
def test_step_on_the_device_and_replay():
    x = torch.randn(1000, 9, device="cuda")
    step = torch.tensor([5], dtype=torch.int64, device="cuda")
    assert torch.equal(features.dropout(x, 0.2, 8, 1, step), features.dropout(x, 0.2, 8, 1, 5))
    with pytest.raises(ValueError):
        features.dropout(x, 0.2, 8, 1, step.to(torch.int32))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            y = features.dropout(x, 0.2, 8, 1, step)
    torch.cuda.current_stream().wait_stream(s)
    for k in (0, 1, 1000):
        step.fill_(k)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, features.dropout(x, 0.2, 8, 1, k))
