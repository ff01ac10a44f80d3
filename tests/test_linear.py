"""Matrix product with bias, activation and residual, and its gradient (cuke_b200.features) against 64-bit definitions."""
import math
import os

import pytest
import torch

from cuke_b200 import _lib, features

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
NULL, SOME, ODD = None, 4096, 4104          # stand-ins for device addresses: a refused call never follows them
ACC = 2.0 ** -23                            # one addition of the fp32 accumulator, truncated
BF = 2.0 ** -8                              # one rounding to bf16
gpu = pytest.mark.gpu


def fwd(x=SOME, ldx=16, w=SOME, ldw=24, bias=NULL, res=NULL, ldr=0, m=4, k=16, n=24, act=0, out=SOME, ldo=24, slope=NULL, ws=SOME, wsb=1 << 30):
    return _lib.lib().kge_linear_forward(x, ldx, w, ldw, bias, res, ldr, m, k, n, act, out, ldo, slope, ws, wsb, None)


def bwd(dout=SOME, ldd=24, x=SOME, ldx=16, w=SOME, ldw=24, slope=SOME, m=4, k=16, n=24, act=1, dx=SOME, lddx=16, dw=SOME, db=SOME, ws=SOME, wsb=1 << 30):
    return _lib.lib().kge_linear_backward(dout, ldd, x, ldx, w, ldw, slope, m, k, n, act, dx, lddx, dw, db, ws, wsb, None)


SIZES = [(dict(act=4), -3), (dict(act=-1), -3), (dict(m=-1), -4), (dict(k=0), -4), (dict(n=0), -4), (dict(k=12), -3), (dict(n=20), -3),
         (dict(m=(1 << 30) + 8), -6), (dict(k=(1 << 20) + 8), -6), (dict(n=(1 << 20) + 8), -6), (dict(x=NULL), -1), (dict(w=NULL), -1), (dict(x=ODD), -2),
         (dict(w=ODD), -2), (dict(ldx=8), -4), (dict(ldx=20), -2), (dict(ldw=16), -4), (dict(ldw=28), -2), (dict(ldx=1 << 33), -6)]


@needs_lib
@pytest.mark.parametrize("kw,code", SIZES + [(dict(out=NULL), -1), (dict(out=ODD), -2), (dict(ldo=16), -4), (dict(ldo=25), -2), (dict(bias=ODD), -2),
                                             (dict(res=ODD, ldr=24), -2), (dict(res=SOME, ldr=16), -4), (dict(slope=ODD), -2)])
def test_forward_refusals(kw, code):
    assert fwd(**kw) == code
    assert _lib.lib().kge_last_error().startswith(b"kge_linear_forward: ")


@needs_lib
@pytest.mark.parametrize("kw,code", SIZES + [(dict(dout=NULL), -1), (dict(slope=NULL), -1), (dict(ldd=16), -4), (dict(ldd=25), -2), (dict(dx=ODD), -2),
                                             (dict(lddx=8), -4), (dict(dw=ODD), -2), (dict(db=ODD), -2), (dict(ws=NULL), -1), (dict(ws=4112), -2), (dict(wsb=0), -5)])
def test_backward_refusals(kw, code):
    assert bwd(**kw) == code
    assert _lib.lib().kge_last_error().startswith(b"kge_linear_backward: ")


@needs_lib
def test_outputs_over_inputs_are_refused():
    x, w, out, res, dy, ws = (4096 * i for i in range(1, 7))
    assert fwd(x=x, w=w, out=x, ws=ws) == -3 and fwd(x=x, w=w, out=w, ws=ws) == -3
    assert fwd(x=x, w=w, out=out, res=out, ldr=32, ldo=24, ws=ws) == -4
    for kw in (dict(dx=dy, dw=out), dict(dx=x, dw=out), dict(dx=w, dw=out), dict(dx=out, dw=res), dict(dx=NULL, dw=x)):
        assert bwd(dout=dy, x=x, w=w, slope=res, ws=ws, db=NULL, **kw) == -3


@needs_lib
def test_workspace_sizes():
    W = _lib.lib().kge_linear_workspace_bytes
    assert W(0, 16, 16, 1, 1) == 0 and W(8, 12, 16, 1, 1) == 0 and fwd(m=0, x=NULL, out=NULL) == 0
    assert W(1 << 16, 1024, 1024, 0, 0) == 0                                   # enough tiles: nothing is split
    assert W(1 << 16, 1024, 1024, 3, 1) >= 2 * (1 << 26)                       # dz
    assert W(128, 4096, 256, 0, 0) % (4 * 128 * 256) == 0 and W(128, 4096, 256, 0, 0) > 0


def test_python_refusals():
    z = torch.zeros(8, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        features.linear(z, z)
    with pytest.raises(ValueError, match="CUDA"):
        features.linear_backward(z, z, z)
    with pytest.raises(TypeError, match="bfloat16"):
        features._matrix(z.float(), "x", 8, 8)
    with pytest.raises(ValueError, match="must be"):
        features._matrix(z, "x", 8, 16)
    with pytest.raises(ValueError, match="act is one of"):
        features._act("tanh")


def act64(z, act):
    if act == "none":
        return z * 1
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def make(m, k, n, act, bias=True, residual=False, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 5 * n)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    wide = lambda a, b: r(a, b + pad)[:, :b]  # noqa: E731
    return dict(x=wide(m, k), w=(wide(k, n).float() / math.sqrt(k)).to(torch.bfloat16) if not pad else wide(k, n), b=r(n) if bias else None,
                res=wide(m, n) if residual else None, dy=wide(m, n))


def check(c, act, backward=True):
    """Forward: K additions of the accumulator over sum |x w|, the activation's own error (slope at most 1.13, evaluation
    2^-20 relative to 1 + |z|), one rounding.  slope: |act''| <= 1.2 times the error of z, one rounding to fp16 (2^-11).
    dz then carries |dout| times that and one rounding, which the products sum up beside their own N or M additions."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x, w, b, res, dy = (d(c[q]) for q in ("x", "w", "b", "res", "dy"))
    m, k, n = x.shape[0], x.shape[1], w.shape[1]
    out, slope = features.linear(c["x"], c["w"], c["b"], act=act, residual=c["res"], save_preact=True)
    assert torch.equal(out, features.linear(c["x"], c["w"], c["b"], act=act, residual=c["res"]))
    z = (x @ w + (0 if b is None else b)).requires_grad_()
    zerr = (k + 4) * ACC * (x.abs() @ w.abs() + (0 if b is None else b.abs()))
    y = act64(z, act)
    ref = y.detach() + (0 if res is None else res)
    zz = z.detach()
    tol = 1.13 * zerr + (2.0 ** -20 * (1 + zz.abs()) if act in ("silu", "gelu") else 0) + BF * ref.abs() + 2 * ACC * (zz.abs() + (0 if res is None else res.abs()))
    assert out.shape == (m, n) and ((out.double() - ref).abs() <= tol).all()
    sl = torch.autograd.grad(y.sum(), z, retain_graph=True)[0]
    serr = torch.zeros_like(zz)
    if act != "none":
        serr = 1.2 * zerr + 2.0 ** -20 * (1 + zz.abs()) + 2.0 ** -11 * sl.abs() + 2.0 ** -25
        if act == "relu":
            serr = (zz.abs() <= zerr).double()              # either side of the kink
        assert ((slope.double() - sl).abs() <= serr).all()
    else:
        assert slope is None
    if not backward:
        return out
    dx, dw, db = features.linear_backward(c["dy"], c["x"], c["w"], slope, act=act)
    dz = dy * sl
    dzerr = dy.abs() * serr + (BF * (dz.abs() + dy.abs() * serr) if act != "none" else 0)
    for got, want, err in ((dx, dz @ w.T, dzerr @ w.abs().T + (n + 4) * ACC * (dz.abs() @ w.abs().T)),
                           (dw, x.T @ dz, x.abs().T @ dzerr + (m + 4) * ACC * (x.abs().T @ dz.abs())),
                           (db, dz.sum(0), (dy.abs() * serr).sum(0) + (m + 4) * ACC * dz.abs().sum(0))):
        bad = ~((got.double() - want).abs() <= err + BF * (want.abs() + err) + 1e-30)
        assert not bad.any(), (bad.nonzero()[:4], got[bad][:4], want[bad][:4])
    again = features.linear_backward(c["dy"], c["x"], c["w"], slope, act=act)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    return out


@gpu
@pytest.mark.parametrize("m,k,n", [(9, 64, 64), (128, 64, 16), (256, 128, 256), (1, 8, 8), (3, 40, 24), (300, 200, 400), (257, 64, 264), (513, 1000, 136),
                                   (100, 2048, 64), (17, 1024, 1024), (2049, 72, 520), (5000, 136, 200), (1024, 24, 1032)])
@pytest.mark.parametrize("act,residual", [("none", False), ("relu", True), ("silu", False), ("gelu", True)])
def test_values(m, k, n, act, residual):
    from cuke_b200 import scoring
    check(make(m, k, n, act, bias=act != "none", residual=residual), act)
    assert scoring.device_flags() == 0


@gpu
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 16])
@pytest.mark.parametrize("k,n", [(8, 8), (1024, 512), (72, 136), (2048, 1024), (4096, 72), (264, 2056)])
def test_few_rows(m, k, n):
    c = make(m, k, n, "gelu", residual=True)
    check(c, "gelu", backward=m in (1, 9))
    c["res"] = None
    check(c, "relu", backward=False)


@gpu
@pytest.mark.parametrize("m,k,n,pad", [(5, 64, 72, 8), (300, 72, 136, 8), (513, 256, 256, 24), (64, 128, 512, 56)])
def test_pitched_rows(m, k, n, pad):
    c = make(m, k, n, "silu", residual=True, pad=pad)
    assert c["x"].stride(0) == k + pad
    out = check(c, "silu")
    wide = torch.full((m, n + pad), 5.0, dtype=torch.bfloat16, device="cuda")
    features.linear(c["x"], c["w"], c["b"], act="silu", residual=c["res"], out=wide[:, :n])
    assert torch.equal(wide[:, :n], out) and (wide[:, n:] == 5).all()
    r = c["res"].contiguous()
    features.linear(c["x"], c["w"], c["b"], act="silu", residual=r, out=r)           # the residual updated in place
    assert torch.equal(r, out)


@gpu
def test_parts_of_the_gradient_and_no_rows():
    c = make(300, 64, 72, "gelu")
    out, s = features.linear(c["x"], c["w"], c["b"], act="gelu", save_preact=True)
    full = features.linear_backward(c["dy"], c["x"], c["w"], s, act="gelu")
    for want in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        part = features.linear_backward(c["dy"], c["x"], c["w"], s, act="gelu", need_dx=want[0], need_dw=want[1], need_dbias=want[2])
        assert all((p is None) if not need else torch.equal(p, f) for p, f, need in zip(part, full, want))
    e = c["x"][:0]
    out, s = features.linear(e, c["w"], c["b"], act="gelu", save_preact=True)
    dx, dw, db = features.linear_backward(c["dy"][:0], e, c["w"], s, act="gelu")
    assert out.shape == (0, 72) and dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    with pytest.raises(ValueError, match="preact"):
        features.linear_backward(c["dy"], c["x"], c["w"], None, act="gelu")


@gpu
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("m", [2, 200])
def test_infinite_and_large_preactivations(act, m):
    """One product per output: z = x w runs through +-infinity, the type's largest values and NaN."""
    v = torch.tensor([float("inf"), float("-inf"), 3e38, -3e38, 1e20, -1e20, 100.0, -100.0, 0.0, -0.0, float("nan"), 1.0, -1.0, 8.0, -8.0, 20.0], device="cuda")
    x = torch.zeros(m, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(8, 16, dtype=torch.bfloat16, device="cuda")
    b = v.to(torch.bfloat16)
    out, s = features.linear(x, w, b, act=act, save_preact=True)
    z = b.double()
    y = {"relu": torch.relu(z), "silu": torch.where(z < -700, 0.0, z * torch.sigmoid(z)),
         "gelu": torch.where(z < -100, 0.0, 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))))}[act]
    y = torch.where(torch.isneginf(z), torch.zeros_like(y), y)
    fine = torch.isfinite(y)
    got = out[0].double()
    assert torch.equal(torch.isnan(got), torch.isnan(y)) and torch.equal(torch.isposinf(got), torch.isposinf(y))
    assert ((got - y)[fine].abs() <= BF * y[fine].abs() + 1e-4).all()
    assert torch.isfinite(s[0][~torch.isnan(v)]).all() and (s[0][v >= 20] == 1).all() and (s[0][v <= -100].float().abs() < 1e-3).all()
    assert torch.equal(out[:1].expand(m, 16).float().nan_to_num(7), out.float().nan_to_num(7))


@gpu
def test_against_differences():
    """Central differences of the 64-bit loss sum(dy * out) with respect to a few inputs; the gradients are bf16 (2^-8 of
    their size) from a bf16 dz (2^-8 of sum |dz||w|)."""
    c = make(6, 16, 24, "gelu", residual=True, seed=3)
    _, s = features.linear(c["x"], c["w"], c["b"], act="gelu", residual=c["res"], save_preact=True)
    dx, dw, db = features.linear_backward(c["dy"], c["x"], c["w"], s, act="gelu")
    x, w, b, dy = (c[q].double() for q in ("x", "w", "b", "dy"))
    f = lambda: (act64(x @ w + b, "gelu") * dy).sum().item()  # noqa: E731
    h = 1e-4
    for t, g, at, size in ((x, dx, (2, 5), (dy.abs() @ w.abs().T)[2, 5]), (w, dw, (7, 11), (x.abs().T @ dy.abs())[7, 11]), (b, db, (3,), dy.abs().sum(0)[3])):
        old = t[at].item()
        t[at] = old + h
        up = f()
        t[at] = old - h
        down = f()
        t[at] = old
        assert abs((up - down) / (2 * h) - g[at].item()) <= 3 * BF * 1.13 * size.item() + 1e-5


@gpu
def test_two_graphs_and_two_streams():
    jobs = [make(64, 1024, 64, "gelu", seed=1), make(700, 72, 136, "gelu", seed=2)]

    def step(c):
        out, s = features.linear(c["x"], c["w"], c["b"], act="gelu", save_preact=True)
        return [out, *features.linear_backward(c["dy"], c["x"], c["w"], s, act="gelu")]

    eager = [step(c) for c in jobs]
    side, graphs, outs = torch.cuda.Stream(), [], []
    for c in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(c))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(o, e))
    got = []
    for c, st in zip(jobs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([step(c) for _ in range(10)][-1])
    torch.cuda.synchronize()
    for o, e in zip(got, eager):
        assert all(torch.equal(a, b) for a, b in zip(o, e))
