"""evkcu_linear, evkcu_gated_ffn and evkcu_qk_norm_rope, forward and backward,
against their formulas in 64 bits.

Tolerances are bounds, element by element, with u = eps / 2 of the storage type
(bf16 2^-8, fp16 2^-11) and t = the type's smallest step (fp16 subnormals):
  - one rounding of a value v: u |v| + t / 2;
  - an fp32 sum of K products a b: (K + 2) 2^-23 sum |a| |b| (a truncating
    adder's bound, twice that of a rounding one);
  - an operand that was itself rounded (hidden, dpre) adds its own error times
    the other operand, summed: |e| @ |w|;
  - act and act' from ex2 and a reciprocal: the exponential's error grows with
    its argument (2 + 1.2 |x| units of 2^-23); 2^-16 |act| and 2^-15 bound them
    wherever the value is not below the type's smallest step.
"""
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import evk_b200 as evk
from conftest import ROOT, u16

pytestmark = pytest.mark.gpu

F64 = torch.float64
ACTS = {"none": evk.ACT_NONE, "relu": evk.ACT_RELU, "gelu": evk.ACT_GELU, "silu": evk.ACT_SILU}
DTYPES = [torch.float16, torch.bfloat16]


def unit(dt):
    return torch.finfo(dt).eps / 2


def step(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, dt, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)


class Guarded:
    """An output inside a larger buffer whose margins must stay as they were."""

    def __init__(self, dt, *shape, fill=None):
        n = math.prod(shape)
        self.buf = torch.full((n + 512,), 77.0, dtype=dt, device="cuda")
        self.t = self.buf[256:256 + n].view(*shape)
        if fill is not None:
            self.t.copy_(fill)

    def check(self):
        torch.cuda.synchronize()
        assert bool((self.buf[:256] == 77).all()) and bool((self.buf[-256:] == 77).all()), "written out of bounds"


def act64(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0 * z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z) if name == "silu" else z


def dact64(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def rounded(ref, err, dt):
    """Bound of a value with error `err` after one rounding."""
    return err + unit(dt) * (ref.abs() + err) + step(dt) / 2


def prod_err(aabs, babs, k):
    return (k + 2) * 2.0 ** -23 * (aabs @ babs)


def check(got, ref, tol, what):
    diff = (got.double() - ref).abs()
    bad = ~(diff <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                                 f"{float((diff / tol).max()):.3g} of the bound")


def lin_ref(x, w, bias, res, act, dt):
    """(z, its error, y, its bound) of the linear operator."""
    x, w = x.double(), w.double()
    z = x @ w
    ez = prod_err(x.abs(), w.abs(), x.shape[1])
    if bias is not None:
        z = z + bias.double()
        ez = ez + 2.0 ** -23 * (bias.double().abs() + z.abs())
    y = act64(z, act)
    e = 1.13 * ez + 2.0 ** -16 * y.abs()
    if res is not None:
        y = y + res.double()
        e = e + 2.0 ** -23 * y.abs()
    return z, ez, y, rounded(y, e, dt)


ROWS = [1, 2, 15, 16, 17, 33, 64, 65, 127, 128, 129, 300]
KN = [(8, 8), (64, 56), (72, 136), (264, 72), (520, 264), (1024, 520)]
LINEAR = [(r, *KN[(i + j) % len(KN)], list(ACTS)[(i + j) % 4], DTYPES[(i // 2 + j) % 2], bool((i + j) % 2),
           bool(i % 3), bool((i + j) % 3 == 1), bool((i // 3 + j) % 2)) for i, r in enumerate(ROWS) for j in range(4)]

# Outputs of many tiles: several rounds of a persistent grid, ragged at every edge.
LINEAR += [(4100, 72, 4104, "gelu", torch.bfloat16, True, True, True, False),
           (4100, 200, 4104, "none", torch.float16, True, False, False, True),
           (2305, 1024, 1800, "silu", torch.float16, False, True, False, False),
           (129, 264, 16392, "relu", torch.bfloat16, False, False, True, True),
           (16385, 64, 264, "none", torch.bfloat16, False, True, False, False)]


@pytest.mark.parametrize("rows,K,N,act,dt,bias,res,pre,nk", LINEAR)
def test_linear(rows, K, N, act, dt, bias, res, pre, nk):
    g = gen(rows * 7 + K)
    x, w = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=K ** -0.5)
    b = rnd(g, dt, N) if bias else None
    r = rnd(g, dt, rows, N) if res else None
    y, z = Guarded(dt, rows, N), Guarded(dt, rows, N)
    evk.linear(x, w.t().contiguous() if nk else w, y.t, bias=b, residual=r, act=ACTS[act], pre=z.t if pre else None,
               transpose_w=nk)
    y.check(), z.check(), evk.check_device_error()
    zr, ez, yr, tol = lin_ref(x, w, b, r, act, dt)
    check(y.t, yr, tol, "y")
    if pre:
        check(z.t, zr, rounded(zr, ez, dt), "pre")
    else:
        assert bool((z.t == 77).all())


@pytest.mark.parametrize("dt", DTYPES)
def test_linear_residual_may_be_the_output(dt):
    for rows, K, N in ((5, 264, 136), (200, 264, 136), (2048, 512, 2304)):
        g = gen(rows)
        x, w, r = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=K ** -0.5), rnd(g, dt, rows, N)
        y = r.clone()
        evk.linear(x, w, y, residual=y)
        _, _, yr, tol = lin_ref(x, w, None, r, "none", dt)
        check(y, yr, tol, f"y in place, {rows} rows")


def back_ref(x, w, z, dy, act, dt):
    """dz and the gradients with their bounds."""
    x, w, dy = x.double(), w.double(), dy.double()
    if act == "none":
        dz, ez, eu = dy, torch.zeros_like(dy), torch.zeros_like(dy)
    else:
        dz = dy * dact64(z.double(), act)
        eu = 2.0 ** -15 * dy.abs()  # unrounded
        ez = rounded(dz, eu, dt)
    dx = dz @ w.t()
    edx = ez @ w.abs().t() + prod_err(dz.abs() + ez, w.abs().t(), w.shape[1])
    dw = x.t() @ dz
    edw = x.abs().t() @ ez + prod_err(x.abs().t(), dz.abs() + ez, x.shape[0])
    db = dz.sum(0)
    edb = eu.sum(0) + (x.shape[0] + 2) * 2.0 ** -23 * (dz.abs() + eu).sum(0)
    return dz, ez, (dx, edx), (dw, edw), (db, edb)


BACK = [(r, *KN[(i + 2 * j) % len(KN)], list(ACTS)[(i + j) % 4], DTYPES[(i // 2 + j) % 2], bool((i // 2 + j) % 2),
         bool(i % 2 == j)) for i, r in enumerate([1, 7, 64, 100, 129, 257, 1000]) for j in range(2)]

BACK += [(1001, 2056, 1800, "gelu", torch.bfloat16, False, False), (300, 4104, 2056, "silu", torch.float16, True, True),
         (5000, 264, 520, "relu", torch.float16, False, True), (2305, 1800, 2056, "none", torch.bfloat16, True, False)]


@pytest.mark.parametrize("rows,K,N,act,dt,nk,acc", BACK)
def test_linear_backward(rows, K, N, act, dt, nk, acc):
    g = gen(rows * 3 + N)
    x, w, dy = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=N ** -0.5), rnd(g, dt, rows, N)
    z = rnd(g, dt, rows, N) if act != "none" else None
    old = [rnd(g, dt, rows, K), rnd(g, dt, *((N, K) if nk else (K, N))), rnd(g, dt, N)]
    dx, dw, db = (Guarded(dt, *o.shape, fill=o) for o in old)
    dz = Guarded(dt, rows, N)
    evk.linear_backward(x, w.t().contiguous() if nk else w, dy, dx=dx.t, dw=dw.t, dbias=db.t, act=ACTS[act], pre=z,
                        dpre=dz.t if z is not None else None, transpose_w=nk, acc=acc)
    for o in (dx, dw, db, dz):
        o.check()
    evk.check_device_error()
    dzr, ez, *grads = back_ref(x, w, z, dy, act, dt)
    if z is not None:
        check(dz.t, dzr, ez, "dpre")
    for got, o, (ref, e), name in zip((dx, dw, db), old, grads, ("dx", "dw", "dbias")):
        if nk and name == "dw":
            ref, e = ref.t(), e.t()
        if acc:
            ref = ref + o.double()
            e = e + 2.0 ** -23 * ref.abs()
        check(got.t, ref, rounded(ref, e, dt), name)


def test_linear_backward_in_place_and_partial():
    """dpre may be pre or dy; each gradient may be left out."""
    dt = torch.bfloat16
    g = gen(5)
    x, w, dy, z = rnd(g, dt, 77, 72), rnd(g, dt, 72, 136, std=0.1), rnd(g, dt, 77, 136), rnd(g, dt, 77, 136)
    dzr, ez, (dxr, edx), (dwr, edw), (dbr, edb) = back_ref(x, w, z, dy, "gelu", dt)
    for where in ("pre", "dy"):
        zz, dd = z.clone(), dy.clone()
        dx = torch.empty_like(x)
        evk.linear_backward(x, w, dd, dx=dx, act=evk.ACT_GELU, pre=zz, dpre=zz if where == "pre" else dd)
        check(zz if where == "pre" else dd, dzr, ez, "dpre in place")
        check(dx, dxr, rounded(dxr, edx, dt), "dx")
    dw, db, dz = torch.empty_like(w), torch.empty(136, dtype=dt, device="cuda"), torch.empty_like(z)
    evk.linear_backward(x, w, dy, dw=dw, act=evk.ACT_GELU, pre=z, dpre=dz)
    check(dw, dwr, rounded(dwr, edw, dt), "dw alone")
    evk.linear_backward(x, w, dy, dbias=db, act=evk.ACT_GELU, pre=z, dpre=dz)
    check(db, dbr, rounded(dbr, edb, dt), "dbias alone")


def ffn_ref(x, wi, wo, res, act, dt):
    x, wi, wo = x.double(), wi.double(), wo.double()
    F = wo.shape[0]
    z = x @ wi
    ez = prod_err(x.abs(), wi.abs(), x.shape[1])
    a, u = act64(z[:, :F], act), z[:, F:]
    ea = 1.13 * ez[:, :F] + 2.0 ** -16 * a.abs()
    h = a * u
    eh = rounded(h, ea * (u.abs() + ez[:, F:]) + a.abs() * ez[:, F:] + 2.0 ** -23 * h.abs(), dt)
    y = h @ wo
    e = eh @ wo.abs() + prod_err(h.abs() + eh, wo.abs(), F)
    if res is not None:
        y = y + res.double()
        e = e + 2.0 ** -23 * y.abs()
    return z, rounded(z, ez, dt), h, eh, y, rounded(y, e, dt)


DF = [(8, 8), (64, 72), (72, 200), (264, 136), (512, 1368)]
FFN = [(r, *DF[(i + j) % len(DF)], list(ACTS)[(i + 2 * j) % 4], DTYPES[(i + j) % 2], bool(i % 2), bool((i + j) % 3),
        bool((i // 2 + j) % 2)) for i, r in enumerate(ROWS) for j in range(3)]

FFN += [(2100, 520, 1368, "silu", torch.bfloat16, True, True, False),
        (1001, 72, 2056, "gelu", torch.float16, True, True, True),
        (4097, 264, 1032, "relu", torch.bfloat16, False, False, True),
        (300, 2056, 4104, "silu", torch.float16, True, False, False)]


@pytest.mark.parametrize("rows,D,F,act,dt,res,pre,nk", FFN)
def test_gated_ffn(rows, D, F, act, dt, res, pre, nk):
    g = gen(rows * 5 + F)
    x, wi, wo = rnd(g, dt, rows, D), rnd(g, dt, D, 2 * F, std=D ** -0.5), rnd(g, dt, F, D, std=F ** -0.5)
    r = rnd(g, dt, rows, D) if res else None
    y, h, z = Guarded(dt, rows, D), Guarded(dt, rows, F), Guarded(dt, rows, 2 * F)
    t = (lambda m: m.t().contiguous()) if nk else (lambda m: m)
    evk.gated_ffn(x, t(wi), t(wo), y.t, h.t, act=ACTS[act], residual=r, pre=z.t if pre else None, transpose_w=nk)
    y.check(), h.check(), z.check(), evk.check_device_error()
    zr, tz, hr, th, yr, ty = ffn_ref(x, wi, wo, r, act, dt)
    check(h.t, hr, th, "hidden")
    check(y.t, yr, ty, "y")
    if pre:
        check(z.t, zr, tz, "pre")


def ffn_back_ref(x, wi, wo, z, dy, act, dt):
    x, wi, wo, z, dy = (t.double() for t in (x, wi, wo, z, dy))
    F = wo.shape[0]
    g, u = z[:, :F], z[:, F:]
    dh = dy @ wo.t()
    edh = prod_err(dy.abs(), wo.abs().t(), dy.shape[1])
    a, da = act64(g, act), dact64(g, act)
    ea, eda = 2.0 ** -16 * a.abs(), 2.0 ** -15
    dz = torch.cat([dh * u * da, dh * a], 1)
    eg = edh * u.abs() * (da.abs() + eda) + (dh * u).abs() * eda
    eu = edh * (a.abs() + ea) + dh.abs() * ea
    ez = rounded(dz, torch.cat([eg, eu], 1) + 2.0 ** -22 * dz.abs(), dt)
    h = a * u
    eh = rounded(h, ea * u.abs() + 2.0 ** -23 * h.abs(), dt)
    dx = dz @ wi.t()
    edx = ez @ wi.abs().t() + prod_err(dz.abs() + ez, wi.abs().t(), 2 * F)
    dwi = x.t() @ dz
    edwi = x.abs().t() @ ez + prod_err(x.abs().t(), dz.abs() + ez, x.shape[0])
    dwo = h.t() @ dy
    edwo = eh.t() @ dy.abs() + prod_err((h.abs() + eh).t(), dy.abs(), x.shape[0])
    return (dz, ez), (h, eh), (dx, edx), (dwi, edwi), (dwo, edwo)


FFNB = [(r, *DF[(i + j) % len(DF)], list(ACTS)[(i + 2 * j) % 4], DTYPES[(i + j) % 2], bool((i // 2 + j) % 2),
         bool(i % 2 == j)) for i, r in enumerate([1, 7, 64, 100, 129, 257, 1000]) for j in range(2)]

FFNB += [(2100, 520, 1368, "silu", torch.bfloat16, False, False), (1001, 72, 2056, "gelu", torch.float16, True, True),
         (4097, 264, 1032, "relu", torch.bfloat16, True, False), (300, 2056, 4104, "silu", torch.float16, False, True)]


@pytest.mark.parametrize("rows,D,F,act,dt,nk,acc", FFNB)
def test_gated_ffn_backward(rows, D, F, act, dt, nk, acc):
    g = gen(rows * 11 + F)
    x, wi, wo = rnd(g, dt, rows, D), rnd(g, dt, D, 2 * F, std=F ** -0.5), rnd(g, dt, F, D, std=D ** -0.5)
    z, dy = rnd(g, dt, rows, 2 * F), rnd(g, dt, rows, D)
    t = (lambda m: m.t().contiguous()) if nk else (lambda m: m)
    old = [rnd(g, dt, rows, D), t(rnd(g, dt, D, 2 * F)), t(rnd(g, dt, F, D))]
    outs = [Guarded(dt, *o.shape, fill=o) for o in old]
    dz, h = Guarded(dt, rows, 2 * F), Guarded(dt, rows, F)
    evk.gated_ffn_backward(x, t(wi), t(wo), z, dy, dz.t, h.t, dx=outs[0].t, dw_in=outs[1].t, dw_out=outs[2].t,
                           act=ACTS[act], transpose_w=nk, acc=acc)
    for o in outs + [dz, h]:
        o.check()
    evk.check_device_error()
    (dzr, ez), (hr, eh), *grads = ffn_back_ref(x, wi, wo, z, dy, act, dt)
    check(dz.t, dzr, ez, "dpre")
    check(h.t, hr, eh, "hidden")
    for got, o, (ref, e), name in zip(outs, old, grads, ("dx", "dw_in", "dw_out")):
        if name != "dx":
            ref, e = t(ref), t(e)
        if acc:
            ref = ref + o.double()
            e = e + 2.0 ** -23 * ref.abs()
        check(got.t, ref, rounded(ref, e, dt), name)


@pytest.mark.parametrize("rows", [9, 200, 2100])
def test_gated_ffn_alone_and_gradient_in_place(rows):
    """y = None stops at hidden (a gated linear unit); dpre may be pre."""
    dt, g, D, F = torch.bfloat16, gen(rows), 264, 1368
    x, wi, wo = rnd(g, dt, rows, D), rnd(g, dt, D, 2 * F, std=D ** -0.5), rnd(g, dt, F, D, std=F ** -0.5)
    h, z = Guarded(dt, rows, F), Guarded(dt, rows, 2 * F)
    assert evk.gated_ffn(x, wi, None, None, h.t, pre=z.t) is h.t
    h.check(), z.check()
    zr, tz, hr, th, _, _ = ffn_ref(x, wi, wo, None, "silu", dt)
    check(h.t, hr, th, "hidden")
    check(z.t, zr, tz, "pre")
    dy, pre = rnd(g, dt, rows, D), z.t.clone()
    dx, dz, d2 = torch.empty_like(x), torch.empty_like(pre), torch.empty_like(x)
    evk.gated_ffn_backward(x, wi, wo, pre, dy, dz, None, dx=dx)
    evk.gated_ffn_backward(x, wi, wo, pre, dy, pre, None, dx=d2)
    assert torch.equal(pre, dz) and torch.equal(dx, d2)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradients_against_differences(act):
    """The kernels' gradients of L = sum(y * dy) against central differences of
    the 64-bit formula along random directions.  The step 1e-5 leaves a
    truncation error near 1e-10 of the third derivative; the gradients'
    bounds, summed over the direction, cover the rest."""
    dt = torch.float16
    g = gen(3)
    rows, D, F = 40, 64, 72
    x, wi, wo = rnd(g, dt, rows, D), rnd(g, dt, D, 2 * F, std=0.1), rnd(g, dt, F, D, std=0.1)
    dy = rnd(g, dt, rows, D)
    y, h, z = (torch.empty(rows, n, dtype=dt, device="cuda") for n in (D, F, 2 * F))
    evk.gated_ffn(x, wi, wo, y, h, act=ACTS[act], pre=z)
    dz, grads = torch.empty_like(z), [torch.empty_like(t) for t in (x, wi, wo)]
    evk.gated_ffn_backward(x, wi, wo, z, dy, dz, h, dx=grads[0], dw_in=grads[1], dw_out=grads[2], act=ACTS[act])

    def loss(x, wi, wo):
        p = x @ wi
        return float((((act64(p[:, :F], act) * p[:, F:]) @ wo) * dy.double()).sum())

    base = [t.double() for t in (x, wi, wo)]
    # The saved pre-activations are rounded: their half step moves dz by at
    # most the second derivatives (below 1.2 |dh| (1 + |u|)) times it.
    zr = x.double() @ wi.double()
    ezr = rounded(zr, prod_err(x.double().abs(), wi.double().abs(), D), dt)
    (dzr, ez), (hr, eh), (_, edx), (_, edwi), (_, edwo) = ffn_back_ref(x, wi, wo, z, dy, act, dt)
    dh = (dy.double() @ wo.double().t()).abs()
    eg, eu = ezr[:, :F], ezr[:, F:]
    more = torch.cat([1.2 * dh * ((1 + z[:, F:].double().abs()) * eg + eu), 1.2 * dh * eg], 1)
    moreh = 1.2 * z[:, F:].double().abs() * eg + (act64(z[:, :F].double(), act).abs() + 1.2 * eg) * eu
    extra = [more @ wi.double().abs().t(), x.double().abs().t() @ more, moreh.t() @ dy.double().abs()]
    for i, (got, e) in enumerate(zip(grads, (edx, edwi, edwo))):
        d = torch.randn(got.shape, generator=g, device="cuda", dtype=F64)
        hi = [t + (1e-5 * d if j == i else 0) for j, t in enumerate(base)]
        lo = [t - (1e-5 * d if j == i else 0) for j, t in enumerate(base)]
        num = (loss(*hi) - loss(*lo)) / 2e-5
        tol = float(((rounded(got.double(), e, dt) + extra[i]) * d.abs()).sum()) + 1e-6 * abs(num)
        assert abs(num - float((got.double() * d).sum())) <= tol, (i, num, tol)


@pytest.mark.parametrize("rows", [3, 130, 600])
def test_nan_and_infinity_stay_in_their_rows(rows):
    dt = torch.bfloat16
    g = gen(9)
    x, w = rnd(g, dt, rows, 72), rnd(g, dt, 72, 136)
    y0, y1 = (torch.empty(rows, 136, dtype=dt, device="cuda") for _ in range(2))
    evk.linear(x, w, y0, act=evk.ACT_SILU)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    evk.linear(x, w, y1, act=evk.ACT_SILU)
    assert bool(torch.isnan(y1[1]).all()) and not bool(torch.isfinite(y1[2]).all())
    keep = [r for r in range(rows) if r not in (1, 2)]
    assert torch.equal(y0[keep], y1[keep])
    big = torch.full((4, 72), 3e38, dtype=dt, device="cuda")  # activations and derivatives at the type's ends
    z = torch.tensor([3e38, -3e38, 60.0, -60.0, 0.0, 1e20, -1e20, 30.0], dtype=dt, device="cuda").repeat(4, 17)
    for act in ("relu", "gelu", "silu"):
        dz, dy = torch.empty_like(z), torch.ones_like(z)
        evk.linear_backward(big, w, dy, dbias=torch.empty(136, dtype=dt, device="cuda"), act=ACTS[act], pre=z, dpre=dz)
        assert torch.equal(dz[:, 0], torch.ones_like(dz[:, 0])) and not bool(dz[:, 1].any()), act
        assert bool(torch.isfinite(dz).all()), act


@pytest.mark.parametrize("dt", DTYPES)
def test_no_rows(dt):
    w, x = torch.ones(72, 136, dtype=dt, device="cuda"), torch.empty(0, 72, dtype=dt, device="cuda")
    y = torch.empty(0, 136, dtype=dt, device="cuda")
    evk.linear(x, w, y)
    dw, db = torch.ones_like(w), torch.ones(136, dtype=dt, device="cuda")
    evk.linear_backward(x, w, y, dw=dw, dbias=db, acc=True)
    assert bool((dw == 1).all()) and bool((db == 1).all())
    evk.linear_backward(x, w, y, dw=dw, dbias=db)
    assert not bool(dw.any()) and not bool(db.any())
    q = torch.empty(0, 5, 128, dtype=dt, device="cuda")
    dg = torch.ones(64, dtype=dt, device="cuda")
    evk.qk_norm_rope(q, q, q, q, 2)
    evk.qk_norm_rope_backward(q, None, q, None, q, None, 2, dgain_q=dg)
    assert not bool(dg.any())


def test_more_than_2_31_elements():
    """Offsets past 32 bits: outputs, saved tensors and a cache of 2.2e9
    elements, looked at near both ends."""
    dt, g = torch.bfloat16, gen(31)
    rows, K, N = 270001, 8, 8192
    x, w = rnd(g, dt, rows, K), rnd(g, dt, K, N)
    y = torch.empty(rows, N, dtype=dt, device="cuda")
    evk.linear(x, w, y, residual=None, act=evk.ACT_SILU)
    dx, dz = torch.empty_like(x), torch.empty_like(y)
    evk.linear_backward(x, w, y, dx=dx, act=evk.ACT_SILU, pre=y, dpre=dz)
    for at in (slice(0, 300), slice(rows - 300, rows)):
        _, _, yr, tol = lin_ref(x[at], w, None, None, "silu", dt)
        check(y[at], yr, tol, "y")
        dzr, ez, (dxr, edx), _, _ = back_ref(x[at], w, y[at], y[at], "silu", dt)
        check(dz[at], dzr, ez, "dpre")
        check(dx[at], dxr, rounded(dxr, edx, dt), "dx")
    del y, dz
    cache_len, heads, dh = 1100000, 16, 128
    kc, vc = (torch.zeros(1, cache_len, heads * dh, dtype=dt, device="cuda") for _ in range(2))
    k, v = rnd(g, dt, 1, 3, heads * dh), rnd(g, dt, 1, 3, heads * dh)
    pos = torch.tensor([[0, cache_len - 1, cache_len // 2]], dtype=torch.int32, device="cuda")
    evk.qk_norm_rope(k, k, torch.empty_like(k), kc, heads, v=v, v_out=vc, cache=True, positions=pos)
    kr, n, _, wt, _, spread = qk_ref(k, heads, None, pos, 0, False, 10000.0, 1e-5)
    tol = rounded(kr, 2 * qk_unit(dh) * spread(n * wt), dt)
    for t in range(3):
        check(kc[0, pos[0, t]].reshape(heads, dh), kr[0, t], tol[0, t], "cache row")
        assert torch.equal(vc[0, pos[0, t]], v[0, t])
    assert int(torch.count_nonzero(vc.view(torch.int16)[0].any(-1))) == 3


# ------------------------------------------------------------- qk_norm_rope --
def qk_ref(x, heads, gain, pos, rot, half_split, base, eps):
    """Normalised and rotated heads in 64 bits: (y, n, r, rotate)."""
    B, S, C = x.shape
    dh = C // heads
    x = x.double().reshape(B, S, heads, dh)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    rot = rot or dh
    i = torch.arange(rot // 2, device="cuda", dtype=F64)
    ang = pos.double()[..., None] * base ** (-2 * i / rot)
    c, s = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]

    def rotate(t, sign=1.0):
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half_split else (slice(0, rot, 2), slice(1, rot, 2))
        o = t.clone()
        o[..., a], o[..., b] = t[..., a] * c - sign * t[..., b] * s, sign * t[..., a] * s + t[..., b] * c
        return o

    # |a| + |b| of each pair, for the bounds
    def spread(t):
        t = t.abs()
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half_split else (slice(0, rot, 2), slice(1, rot, 2))
        o = t.clone()
        o[..., a] = o[..., b] = t[..., a] + t[..., b]
        return o

    w = gain.double() if gain is not None else torch.ones(dh, device="cuda", dtype=F64)
    return rotate(n * w), n, r, w, rotate, spread


# fp32: r from a sum of Dh squares (Dh 2^-24 at most, halved by the root) and
# rsqrt (2^-22); the products n, gain and the angle (2^-22 of a turn and the
# function's own 2^-22) come on top.
def qk_unit(dh):
    return dh * 2.0 ** -24 + 12 * 2.0 ** -23


QK = [(1, 1, 1, 1, 8, 0, False), (2, 3, 4, 2, 16, 0, False), (3, 7, 5, 1, 32, 16, True), (1, 129, 8, 8, 64, 0, True),
      (2, 65, 12, 4, 64, 32, True), (2, 33, 6, 3, 80, 0, True), (5, 9, 6, 2, 96, 48, False),
      (1, 300, 32, 8, 128, 0, False), (4, 31, 7, 7, 128, 64, True), (3, 17, 4, 1, 256, 0, False),
      (2, 40, 3, 3, 248, 16, True), (2, 6, 2, 2, 72, 72, False), (1, 2000, 2, 1, 128, 0, True),
      (2, 1, 200, 100, 64, 2, False), (2, 50, 3, 2, 128, 96, True), (1, 5000, 20, 4, 64, 48, True),
      (3, 2500, 12, 12, 128, 0, False)]


@pytest.mark.parametrize("B,S,H,Hk,dh,rot,half", QK)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("form", ["packed", "in place", "positions"])
def test_qk_norm_rope(B, S, H, Hk, dh, rot, half, dt, form):
    g = gen(B * 100 + S + dh)
    qkv = rnd(g, dt, B, S, (H + 2 * Hk) * dh, std=2.0)
    if B * S > 1:
        qkv[0, -1, :dh] = 0  # a head of zeros stays zero
    q, k, _ = qkv.split([H * dh, Hk * dh, Hk * dh], -1)
    gains = form != "in place"
    gq, gk = (rnd(g, dt, dh, std=0.2, mean=1.0) for _ in range(2)) if gains else (None, None)
    off = 0 if form == "packed" else 1048000
    pos = torch.arange(S, device="cuda")[None].expand(B, S) + off
    kw = dict(rot_dim=rot, half_split=half, base=500000.0, eps=1e-5, pos_offset=off)
    if form == "positions":
        pos = torch.randint(-5, 2 ** 31 - 1, (B, S), generator=g, device="cuda").int()
        kw.update(positions=pos, pos_offset=0)
    want = [qk_ref(t, h, w, pos, rot, half, 500000.0, 1e-5) for t, h, w in ((q, H, gq), (k, Hk, gk))]
    if form == "in place":
        before = qkv.clone()
        evk.qk_norm_rope(q, k, q, k, H, **kw)
        got = (q, k)
        assert torch.equal(qkv[..., (H + Hk) * dh:], before[..., (H + Hk) * dh:])
    else:
        outs = Guarded(dt, B, S, H * dh), Guarded(dt, B, S, Hk * dh)
        evk.qk_norm_rope(q, k, outs[0].t, outs[1].t, H, gain_q=gq, gain_k=gk, **kw)
        outs[0].check(), outs[1].check()
        got = (outs[0].t, outs[1].t)
    for t, (y, n, r, w, _, spread) in zip(got, want):
        # far positions: |pos| 2^-53 of a turn, below 2^-22 up to 2^31
        tol = rounded(y, 2 * qk_unit(dh) * spread(n * w), dt)
        check(t.reshape(y.shape), y, tol, form)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,S,H,Hk,dh,cache_len", [(8, 1, 32, 8, 128, 100), (3, 5, 4, 4, 64, 37), (1, 1, 1, 1, 80, 3),
                                                    (3, 2000, 8, 8, 128, 2100)])
def test_qk_norm_rope_into_a_cache(B, S, H, Hk, dh, cache_len, dt):
    g = gen(cache_len)
    qkv = rnd(g, dt, B, S, (H + 2 * Hk) * dh)
    q, k, v = qkv.split([H * dh, Hk * dh, Hk * dh], -1)
    pos = torch.stack([torch.randperm(cache_len, generator=g, device="cuda")[:S] for _ in range(B)]).int()
    if B > 1:
        pos[1, 0], pos[2, 0] = cache_len, -1  # outside: not stored
    old = rnd(g, dt, B, cache_len, Hk * dh), rnd(g, dt, B, cache_len, Hk * dh)
    kc, vc = (Guarded(dt, *o.shape, fill=o) for o in old)
    qo = torch.empty(B, S, H * dh, dtype=dt, device="cuda")
    evk.qk_norm_rope(q, k, qo, kc.t, H, v=v, v_out=vc.t, cache=True, positions=pos)
    kc.check(), vc.check()
    yk, n, _, w, _, spread = qk_ref(k, Hk, None, pos, 0, False, 10000.0, 1e-5)
    tol = rounded(yk, 2 * qk_unit(dh) * spread(n * w), dt)
    seen = torch.zeros(B, cache_len, dtype=torch.bool, device="cuda")
    for b in range(B):
        for t in range(S):
            p = int(pos[b, t])
            if 0 <= p < cache_len:
                seen[b, p] = True
                check(kc.t[b, p].reshape(Hk, dh), yk[b, t], tol[b, t], "cache row")
                assert torch.equal(vc.t[b, p], v[b, t])
    assert torch.equal(kc.t[~seen], old[0][~seen]) and torch.equal(vc.t[~seen], old[1][~seen])
    yq, n, _, w, _, spread = qk_ref(q, H, None, pos, 0, False, 10000.0, 1e-5)
    check(qo.reshape(yq.shape), yq, rounded(yq, 2 * qk_unit(dh) * spread(n * w), dt), "q")


@pytest.mark.parametrize("B,S,H,Hk,dh,rot,half", QK)
@pytest.mark.parametrize("dt", DTYPES)
def test_qk_norm_rope_backward(B, S, H, Hk, dh, rot, half, dt):
    g = gen(B * 10 + S + dh)
    qkv, dqkv = rnd(g, dt, B, S, (H + 2 * Hk) * dh, std=2.0), Guarded(dt, B, S, (H + 2 * Hk) * dh)
    q, k, _ = qkv.split([H * dh, Hk * dh, Hk * dh], -1)
    dq, dk, dv = dqkv.t.split([H * dh, Hk * dh, Hk * dh], -1)
    gq, gk = rnd(g, dt, dh, std=0.2, mean=1.0), None if dh == 96 else rnd(g, dt, dh, std=0.2, mean=1.0)
    dqo, dko = rnd(g, dt, B, S, H * dh), rnd(g, dt, B, S, Hk * dh)
    acc = dh == 64
    old = rnd(g, dt, dh), rnd(g, dt, dh)
    dgq, dgk = (Guarded(dt, dh, fill=o) for o in old)
    pos = torch.arange(S, device="cuda")[None].expand(B, S) + 7
    ws = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
    evk.qk_norm_rope_backward(q, k, dqo, dko, dq, dk, H, gain_q=gq, gain_k=gk, dgain_q=dgq.t, dgain_k=dgk.t,
                              workspace=ws, rot_dim=rot, half_split=half, pos_offset=7, acc_gain=acc)
    dqkv.check(), dgq.check(), dgk.check()
    assert bool((dv == 77).all())
    for x, dy, heads, gain, got, dg, o in ((q, dqo, H, gq, dq, dgq, old[0]), (k, dko, Hk, gk, dk, dgk, old[1])):
        _, n, r, w, rotate, spread = qk_ref(x, heads, gain, pos, rot, half, 10000.0, 1e-5)
        dy = dy.double().reshape(n.shape)
        t = rotate(dy, -1.0)
        dn = t * w
        m = (dn * n).mean(-1, keepdim=True)
        ref = r * (dn - n * m)
        # t carries the angle's error, n and m those of r and the sums
        su, e = spread(dy), 2 * qk_unit(dh)
        mabs = (su * w.abs() * n.abs()).mean(-1, keepdim=True)
        tol = 4 * e * r * (su * w.abs() + n.abs() * mabs)
        check(got.reshape(ref.shape), ref, rounded(ref, tol, dt), "dx")
        count = B * S * heads
        ref = (t * n).sum((0, 1, 2))
        # the longest chain of additions is under 2^11, whatever the count
        tol = (2 * e + min(count, 2048) * 2.0 ** -23) * (su * n.abs()).sum((0, 1, 2))
        if acc:
            ref = ref + o.double()
            tol = tol + 2.0 ** -23 * ref.abs()
        check(dg.t, ref, rounded(ref, tol, dt), "dgain")


def test_qk_norm_rope_backward_in_place_without_gains():
    dt = torch.bfloat16
    g = gen(77)
    q, k = rnd(g, dt, 2, 50, 4 * 64), rnd(g, dt, 2, 50, 2 * 64)
    a, b = rnd(g, dt, 2, 50, 4 * 64), rnd(g, dt, 2, 50, 2 * 64)
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    evk.qk_norm_rope_backward(q, k, a, b, dq, dk, 4)
    evk.qk_norm_rope_backward(q, k, a, b, a, b, 4)
    assert torch.equal(a, dq) and torch.equal(b, dk)
    evk.qk_norm_rope_backward(q, None, dq, None, dq, None, 4)  # queries only


def test_qk_gradient_against_differences():
    """Along random directions, as above: bound of the gradients plus 1e-6."""
    dt = torch.float16
    g = gen(21)
    B, S, H, dh = 2, 9, 3, 64
    x, gain, dy = rnd(g, dt, B, S, H * dh), rnd(g, dt, dh, std=0.2, mean=1.0), rnd(g, dt, B, S, H * dh)
    dx, dg = torch.empty_like(x), torch.empty_like(gain)
    ws = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
    evk.qk_norm_rope_backward(x, None, dy, None, dx, None, H, gain_q=gain, dgain_q=dg, workspace=ws, half_split=True)
    pos = torch.arange(S, device="cuda")[None].expand(B, S)

    def loss(x, w):
        return float((qk_ref(x, H, w, pos, 0, True, 10000.0, 1e-5)[0].reshape(x.shape) * dy.double()).sum())

    for got, i in ((dx, 0), (dg, 1)):
        base = [x.double(), gain.double()]
        d = torch.randn(got.shape, generator=g, device="cuda", dtype=F64)
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        num = (loss(*hi) - loss(*lo)) / 2e-5
        # each gradient: its rounding plus 2^-17 of the sums that cancel in it
        size = dy.double().abs().amax() * 8 if i == 0 else dy.double().abs().sum() / dh * 4
        tol = float(((unit(dt) * got.double().abs() + 2.0 ** -17 * size) * d.abs()).sum()) + 1e-6 * abs(num)
        assert abs(num - float((got.double() * d).sum())) <= tol, (i, num, tol)


# ------------------------------------------------------------------ together --
def _layer_state(dt, B, S, H, Hk, dh, F, seed, bias=True):
    g = gen(seed)
    D = H * dh
    s = dict(x=rnd(g, dt, B, S, D), wqkv=rnd(g, dt, D, (H + 2 * Hk) * dh, std=D ** -0.5),
             bqkv=rnd(g, dt, (H + 2 * Hk) * dh, std=0.1), gq=rnd(g, dt, dh, std=0.1, mean=1),
             gk=rnd(g, dt, dh, std=0.1, mean=1), wo=rnd(g, dt, D, D, std=D ** -0.5),
             wi=rnd(g, dt, D, 2 * F, std=D ** -0.5), wd=rnd(g, dt, F, D, std=F ** -0.5), dy=rnd(g, dt, B, S, D))
    e = lambda *sh: torch.empty(*sh, dtype=dt, device="cuda")  # noqa: E731
    s.update(xn=e(B, S, D), qkv=e(B, S, (H + 2 * Hk) * dh), q=e(B, S, D), k=e(B, S, Hk * dh), v=e(B, S, Hk * dh),
             att=e(B, S, D), x1=e(B, S, D), x1n=e(B, S, D), h=e(B, S, F), pre=e(B, S, 2 * F), y=e(B, S, D))
    return s


def _layer(s, H, Hk, dh):
    """One decoder layer's forward pass through the public entry points."""
    evk.rms_norm(s["x"], s["xn"], eps=1e-5)
    evk.linear(s["xn"], s["wqkv"], s["qkv"], bias=s["bqkv"])
    q, k, v = s["qkv"].split([H * dh, Hk * dh, Hk * dh], -1)
    evk.qk_norm_rope(q, k, s["q"], s["k"], H, gain_q=s["gq"], gain_k=s["gk"], v=v, v_out=s["v"])
    evk.flash_attention(s["q"], s["k"], s["v"], s["att"], heads=H, causal=True)
    evk.linear(s["att"], s["wo"], s["x1"], residual=s["x"])
    evk.rms_norm(s["x1"], s["x1n"], eps=1e-5)
    evk.gated_ffn(s["x1n"], s["wi"], s["wd"], s["y"], s["h"], residual=s["x1"], pre=s["pre"])
    return s["y"]


def _layer64(s, H, Hk, dh):
    w = {n: t.double() for n, t in s.items()}
    norm = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    x = w["x"]
    B, S, D = x.shape
    q, k, v = (norm(x) @ w["wqkv"] + w["bqkv"]).split([H * dh, Hk * dh, Hk * dh], -1)
    pos = torch.arange(S, device="cuda")[None].expand(B, S)
    q = qk_ref(q, H, w["gq"], pos, 0, False, 10000.0, 1e-5)[0].transpose(1, 2)
    k = qk_ref(k, Hk, w["gk"], pos, 0, False, 10000.0, 1e-5)[0].transpose(1, 2).repeat_interleave(H // Hk, 1)
    v = v.reshape(B, S, Hk, dh).transpose(1, 2).repeat_interleave(H // Hk, 1)
    sc = (q @ k.transpose(2, 3)) / math.sqrt(dh)
    sc = sc.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    x1 = x + (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(B, S, D) @ w["wo"]
    p = norm(x1) @ w["wi"]
    F = p.shape[-1] // 2
    return x1 + (act64(p[..., :F], "silu") * p[..., F:]) @ w["wd"]


@pytest.mark.parametrize("dt", DTYPES)
def test_decoder_layer(dt):
    """The operators together, as a decoder layer calls them.  Eight tensors
    are rounded on the way, each off by at most u relative to its own size;
    none is amplified by more than the layer's gain (about 1 by the weights'
    scale, doubled by the gated product): 2-norm within 16 u."""
    B, S, H, Hk, dh, F = 2, 192, 8, 2, 64, 1368
    s = _layer_state(dt, B, S, H, Hk, dh, F, 4)
    y = _layer(s, H, Hk, dh)
    evk.check_device_error()
    ref = _layer64(s, H, Hk, dh)
    err = float((y.double() - ref).norm() / ref.norm())
    assert err <= 16 * unit(dt), err


def test_layer_captured_replayed_and_on_two_streams():
    """Captured graphs and eager calls on two streams give the bits of a plain
    run: no call shares scratch with another, and equal calls are equal."""
    dt = torch.bfloat16
    B, S, H, Hk, dh, F = 1, 130, 4, 2, 64, 264
    sets = [_layer_state(dt, B, S, H, Hk, dh, F, n) for n in (1, 2)]

    def back(s):
        rows = B * S
        f = lambda t: t.view(rows, -1)  # noqa: E731
        if "dx" not in s:
            s["dpre"], s["dx"] = torch.empty_like(s["pre"]), torch.empty_like(s["x"])
            s["dwi"], s["dwd"] = torch.empty_like(s["wi"]), torch.empty_like(s["wd"])
            s["dq"], s["dgq"] = torch.empty_like(s["q"]), torch.empty_like(s["gq"])
            s["ws"] = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
        evk.gated_ffn_backward(f(s["x1n"]), s["wi"], s["wd"], f(s["pre"]), f(s["dy"]), f(s["dpre"]), f(s["h"]),
                               dx=f(s["dx"]), dw_in=s["dwi"], dw_out=s["dwd"])
        q = s["qkv"][..., :H * dh]
        evk.qk_norm_rope_backward(q, None, s["dx"], None, s["dq"], None, H, gain_q=s["gq"], dgain_q=s["dgq"],
                                  workspace=s["ws"])
        return [s[n] for n in ("y", "pre", "dx", "dwi", "dwd", "dq", "dgq")]

    want = []
    for s in sets:
        _layer(s, H, Hk, dh)
        want.append([t.clone() for t in back(s)])
    for _ in range(3):
        for s in sets:
            for n in ("y", "pre", "dx", "dwi", "dwd", "dq", "dgq"):
                s[n].fill_(3.0)
        streams = [torch.cuda.Stream() for _ in sets]
        torch.cuda.synchronize()
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                _layer(s, H, Hk, dh)
                back(s)
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(back(s), w))
    graphs = []
    for s in sets:
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            _layer(s, H, Hk, dh)
            outs = back(s)
        graphs.append((gph, outs))
    for _, outs in graphs:
        for t in outs:
            t.fill_(5.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(2):
        for (gph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gph.replay()
    torch.cuda.synchronize()
    for (_, outs), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_equal_calls_give_equal_bits(rows):
    dt = torch.float16
    g = gen(rows)
    x, wi, wo = rnd(g, dt, rows, 1024), rnd(g, dt, 1024, 1040, std=0.03), rnd(g, dt, 520, 1024, std=0.03)
    first = None
    for _ in range(4):
        y, h = torch.empty_like(x), torch.empty(rows, 520, dtype=dt, device="cuda")
        evk.gated_ffn(x, wi, wo, y, h)
        first = y if first is None else first
        assert torch.equal(y, first)


def test_binding_refuses_mismatched_tensors():
    dt = torch.float16
    e = lambda *s: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    x, w, y = e(4, 16), e(16, 24), e(4, 24)
    with pytest.raises(ValueError):
        evk.linear(e(4, 32)[:, ::2], w, y)  # not contiguous
    with pytest.raises(evk.EvkcuError):
        evk.linear(x, w, y, bias=e(16))
    with pytest.raises(evk.EvkcuError):
        evk.linear(x, w, y, residual=y.bfloat16())
    with pytest.raises(evk.EvkcuError):
        evk.linear(x, w, y, transpose_w=True)
    with pytest.raises(evk.EvkcuError):
        evk.linear(e(4, 12), e(12, 24), y)  # K not a multiple of 8
    with pytest.raises(evk.EvkcuError):
        evk.gated_ffn(x, e(16, 48), e(24, 16), e(4, 24), e(4, 24))
    q = e(2, 3, 128)
    with pytest.raises(evk.EvkcuError):
        evk.qk_norm_rope(q.transpose(0, 1), None, e(3, 2, 128), None, 2)  # rows not evenly spaced
    with pytest.raises(evk.EvkcuError):
        evk.qk_norm_rope(q, None, e(2, 3, 128), None, 2, positions=torch.zeros(6, device="cuda"))
    with pytest.raises(evk.EvkcuError):
        evk.qk_norm_rope(q, None, e(2, 3, 128), None, 3)
    with pytest.raises(evk.EvkcuError):
        evk.qk_norm_rope_backward(q, None, q, None, e(2, 3, 128), None, 2, dgain_q=e(64))  # no workspace


LAYER = os.path.join(ROOT, "evk_b200", "reftests", "layer_check")


@pytest.mark.skipif(not os.path.exists(LAYER), reason="layer_check not built")
def test_cpp_layer_gives_the_bits_of_the_c_abi(tmp_path):
    """evk_ai_ext.h's linear, gated_ffn and qk_norm_rope, forward and backward,
    through libevk_ai.so (shapes in layer_check.cpp) against the same calls
    through the Python binding: equal bits."""
    dt, g = torch.bfloat16, gen(99)
    B, S, D, F, H, Hk, dh = 2, 9, 256, 264, 4, 2, 64
    C = (H + 2 * Hk) * dh
    x, wqkv, bqkv = rnd(g, dt, B, S, D), rnd(g, dt, D, C, std=0.06), rnd(g, dt, C, std=0.1)
    gq, gk = (rnd(g, dt, dh, std=0.1, mean=1.0) for _ in range(2))
    wi, wo, dy = rnd(g, dt, D, 2 * F, std=0.06), rnd(g, dt, F, D, std=0.06), rnd(g, dt, B, S, D)
    fin, fout = tmp_path / "in.bin", tmp_path / "out.bin"
    fin.write_bytes(b"".join(u16(t).tobytes() for t in (x, wqkv, bqkv, gq, gk, wi, wo, dy)))
    r = subprocess.run([LAYER, str(fin), str(fout)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "LAYER_OK" in r.stdout, (r.stdout + r.stderr)[-3000:]
    e = lambda *s: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    qkv, q, k, v, kc, vc = e(B, S, C), e(B, S, D), e(B, S, 128), e(B, S, 128), e(B, 16, 128), e(B, 16, 128)
    evk.linear(x, wqkv, qkv, bias=bqkv)
    qi, ki, vi = qkv.split([H * dh, Hk * dh, Hk * dh], -1)
    rope = dict(half_split=True, pos_offset=5)
    evk.qk_norm_rope(qi, ki, q, k, H, gain_q=gq, gain_k=gk, v=vi, v_out=v, **rope)
    evk.qk_norm_rope(qi, ki, q, kc, H, gain_q=gq, gain_k=gk, v=vi, v_out=vc, cache=True, **rope)
    y, h, pre, dpre = e(B, S, D), e(B, S, F), e(B, S, 2 * F), e(B, S, 2 * F)
    evk.gated_ffn(x, wi, wo, y, h, residual=x, pre=pre)
    dx, dwi, dwo, dqkv = e(B, S, D), e(D, 2 * F), e(F, D), e(B, S, C)
    evk.gated_ffn_backward(x, wi, wo, pre, dy, dpre, h, dx=dx, dw_in=dwi, dw_out=dwo)
    dqi, dki, _ = dqkv.split([H * dh, Hk * dh, Hk * dh], -1)
    dgq, dgk, dxq, dwqkv, dbqkv = e(dh), e(dh), e(B, S, D), e(D, C), e(C)
    ws = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
    evk.qk_norm_rope_backward(qi, ki, q, k, dqi, dki, H, gain_q=gq, gain_k=gk, dgain_q=dgq, dgain_k=dgk, workspace=ws,
                              **rope)
    evk.linear_backward(x, wqkv, dqkv, dx=dxq, dw=dwqkv, dbias=dbqkv)
    got, at = np.fromfile(fout, np.uint16), 0
    names = "qkv q k v y pre dx dwi dwo dqkv dgq dgk dxq dwqkv dbqkv kc".split()
    for name, t in zip(names, (qkv, q, k, v, y, pre, dx, dwi, dwo, dqkv, dgq, dgk, dxq, dwqkv, dbqkv, kc)):
        want = u16(t).ravel()
        assert np.array_equal(got[at:at + want.size], want), name
        at += want.size
    assert at == got.size
