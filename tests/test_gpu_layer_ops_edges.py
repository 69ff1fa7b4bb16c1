"""Edges of evkcu_linear, evkcu_gated_ffn and evkcu_qk_norm_rope that
test_gpu_layer_ops.py does not reach, with its helpers and bounds."""
import math
import threading

import pytest
import torch

import evk_b200 as evk
from test_gpu_layer_ops import (ACTS, DTYPES, _layer, _layer_state, act64, back_ref, check, ffn_back_ref, gen, lin_ref,
                                qk_ref, qk_unit, rnd, rounded)

pytestmark = pytest.mark.gpu


# -------------------------------------------- order of loads, stores, waits --
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,D,F", [(1030, 520, 2056), (2305, 264, 1032)])
def test_staged_inputs_arrive_before_they_are_read(rows, D, F, dt):
    """Epilogues that load boxes (residual, saved pre-activations, gradients
    added to) in the large-product kernel, several tiles a CTA: right, and the
    same bits in every call."""
    g = gen(rows + D)
    x, wi, wo = rnd(g, dt, rows, D), rnd(g, dt, D, 2 * F, std=F ** -0.5), rnd(g, dt, F, D, std=D ** -0.5)
    z, dy, res = rnd(g, dt, rows, 2 * F), rnd(g, dt, rows, D), rnd(g, dt, rows, 2 * F)
    old = rnd(g, dt, rows, D)
    first = None
    for _ in range(6):
        dz, y, pre, dx = torch.empty_like(z), res.clone(), torch.empty_like(z), old.clone()
        evk.linear(x, wi, y, residual=y, act=evk.ACT_GELU, pre=pre)
        evk.gated_ffn_backward(x, wi, wo, z, dy, dz, None, dx=dx, acc=True)
        got = [y, pre, dz, dx]
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    evk.check_device_error()
    zr, ez, yr, tol = lin_ref(x, wi, None, res, "gelu", dt)
    check(first[0], yr, tol, "y")
    check(first[1], zr, rounded(zr, ez, dt), "pre")
    (dzr, ez), _, (dxr, edx), _, _ = ffn_back_ref(x, wi, wo, z, dy, "silu", dt)
    check(first[2], dzr, ez, "dpre")
    dxr = dxr + old.double()
    check(first[3], dxr, rounded(dxr, edx + 2.0 ** -23 * dxr.abs(), dt), "dx")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,K,N", [(3, 2048, 264), (13, 1024, 136), (16, 4096, 520), (21, 2048, 264),
                                      (63, 1024, 136), (64, 4096, 264), (101, 2048, 136), (127, 4096, 264)])
def test_split_sums(rows, K, N, dt):
    """Products of few tiles, K split over a cluster whose CTAs share out rows
    that do not divide evenly: right, and the same bits in every call."""
    g = gen(rows + K)
    x, w = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=K ** -0.5)
    first = None
    for _ in range(6):
        y = torch.empty(rows, N, dtype=dt, device="cuda")
        evk.linear(x, w, y)
        first = y if first is None else first
        assert torch.equal(y, first)
    evk.check_device_error()
    _, _, yr, tol = lin_ref(x, w, None, None, "none", dt)
    check(first, yr, tol, "y")


@pytest.mark.parametrize("rows", [1, 3, 9, 515, 1031])
@pytest.mark.parametrize("where", ["pre", "dy"])
def test_activation_gradient_in_place_of_ragged_rows(rows, where):
    """dpre over pre or over dy, rows that leave lanes without a row: the bits
    of separate buffers, and the column sums of the unrounded values."""
    dt, g, K, N = torch.bfloat16, gen(rows), 72, 136
    x, w = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=N ** -0.5)
    z, dy = rnd(g, dt, rows, N), rnd(g, dt, rows, N)
    dz, dx, db = torch.empty_like(z), torch.empty_like(x), torch.empty(N, dtype=dt, device="cuda")
    evk.linear_backward(x, w, dy, dx=dx, dbias=db, act=evk.ACT_SILU, pre=z, dpre=dz)
    dzr, ez, (dxr, edx), _, (dbr, edb) = back_ref(x, w, z, dy, "silu", dt)
    check(dz, dzr, ez, "dpre")
    check(dx, dxr, rounded(dxr, edx, dt), "dx")
    check(db, dbr, rounded(dbr, edb, dt), "dbias")
    for _ in range(4):
        zz, dd, d2, b2 = z.clone(), dy.clone(), torch.empty_like(x), torch.empty_like(db)
        over = zz if where == "pre" else dd
        evk.linear_backward(x, w, dd, dx=d2, dbias=b2, act=evk.ACT_SILU, pre=zz, dpre=over)
        assert torch.equal(over, dz) and torch.equal(d2, dx) and torch.equal(b2, db)


def test_many_small_products_back_to_back():
    """Short products one behind the other, so that a kernel starts where the
    one before has just left: equal bits to each call alone."""
    dt, g = torch.bfloat16, gen(17)
    calls = []
    for rows, K, N in ((300, 8, 2056), (1030, 64, 520), (5, 72, 264), (2305, 136, 1032), (40, 264, 136)):
        x, w = rnd(g, dt, rows, K), rnd(g, dt, K, N, std=K ** -0.5)
        r = rnd(g, dt, rows, N)
        y = torch.empty_like(r)
        evk.linear(x, w, y, residual=r)
        torch.cuda.synchronize()
        _, _, yr, tol = lin_ref(x, w, None, r, "none", dt)
        check(y, yr, tol, "y")
        calls.append((x, w, r, y))
    outs = []
    for _ in range(40):
        for x, w, r, _ in calls:
            outs.append(torch.empty_like(r))
            evk.linear(x, w, outs[-1], residual=r)
    evk.check_device_error()
    for i, o in enumerate(outs):
        assert torch.equal(o, calls[i % len(calls)][3])


# ------------------------------------------------------------- qk_norm_rope --
def qk_grad_ref(x, dy, heads, gain, pos, rot, half, eps):
    """(dx, its bound before rounding, dgain, its bound before rounding): the
    formulas and bounds of test_qk_norm_rope_backward."""
    _, n, r, w, rotate, spread = qk_ref(x, heads, gain, pos, rot, half, 10000.0, eps)
    dy = dy.double().reshape(n.shape)
    t = rotate(dy, -1.0)
    dn = t * w
    su, e = spread(dy), 2 * qk_unit(n.shape[-1])
    mabs = (su * w.abs() * n.abs()).mean(-1, keepdim=True)
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    count = n.shape[0] * n.shape[1] * n.shape[2]
    return (dx, 4 * e * r * (su * w.abs() + n.abs() * mabs), (t * n).sum((0, 1, 2)),
            (2 * e + min(count, 2048) * 2.0 ** -23) * (su * n.abs()).sum((0, 1, 2)))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("B,S,H,Hk,dh,rot,half", [(1, 1, 32, 8, 128, 0, False), (1, 1001, 32, 8, 128, 0, False),
                                                  (3, 7, 5, 1, 32, 16, True), (2, 33, 6, 3, 80, 0, True),
                                                  (1, 2, 3, 0, 256, 0, False)])
def test_gain_gradients_without_eps(B, S, H, Hk, dh, rot, half, eps, dt):
    """eps = 0, no head all zeros, rows and heads that leave groups of a block
    idle: gain gradients of the real rows alone."""
    g = gen(B * 10 + S + dh)
    dt_k = Hk * dh
    q, k = rnd(g, dt, B, S, H * dh, std=2.0), rnd(g, dt, B, S, dt_k, std=2.0) if Hk else None
    dqo, dko = rnd(g, dt, B, S, H * dh), rnd(g, dt, B, S, dt_k) if Hk else None
    gq, gk = (rnd(g, dt, dh, std=0.2, mean=1.0) for _ in range(2))
    dgq, dgk = torch.empty_like(gq), torch.empty_like(gk)
    dq, dk = torch.empty_like(q), torch.empty_like(k) if Hk else None
    ws = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
    evk.qk_norm_rope_backward(q, k, dqo, dko, dq, dk, H, gain_q=gq, gain_k=gk if Hk else None, dgain_q=dgq,
                              dgain_k=dgk if Hk else None, workspace=ws, rot_dim=rot, half_split=half, eps=eps)
    pos = torch.arange(S, device="cuda")[None].expand(B, S)
    for x, dy, heads, gain, dx, dg in ((q, dqo, H, gq, dq, dgq), (k, dko, Hk, gk, dk, dgk)):
        if x is None:
            continue
        xr, ex, gr, eg = qk_grad_ref(x, dy, heads, gain, pos, rot, half, eps)
        check(dx.reshape(xr.shape), xr, rounded(xr, ex, dt), "dx")
        check(dg, gr, rounded(gr, eg, dt), "dgain")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rot", [2, 20, 30, 70])
@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_unrotated_values_stay_apart(rot, bad, dt):
    """A rotated part that ends inside a vector of eight: values past it keep
    to themselves, so an infinity or NaN in one column of a gradient reaches
    no other column's gain gradient, nor in a gain another column's output."""
    g, dh, S, H = gen(rot), 80, 5, 3
    x, dy = rnd(g, dt, 1, S, H * dh), rnd(g, dt, 1, S, H * dh)
    gain, dgain, dx = rnd(g, dt, dh, std=0.2, mean=1.0), torch.empty(dh, dtype=dt, device="cuda"), torch.empty_like(x)
    ws = torch.empty(evk.qk_norm_rope_workspace(dh), dtype=torch.uint8, device="cuda")
    pos = torch.arange(S, device="cuda")[None]
    _, _, gr, eg = qk_grad_ref(x, dy, H, gain, pos, rot, False, 1e-5)
    yr, n, _, w, _, spread = qk_ref(x, H, gain, pos, rot, False, 10000.0, 1e-5)
    tol = rounded(yr, 2 * qk_unit(dh) * spread(n * w), dt)
    dyb, gainb, y = dy.clone(), gain.clone(), torch.empty_like(x)
    dyb.view(1, S, H, dh)[0, 2, 1, rot] = float(bad)
    gainb[rot] = float(bad)
    evk.qk_norm_rope_backward(x, None, dyb, None, dx, None, H, gain_q=gain, dgain_q=dgain, workspace=ws, rot_dim=rot)
    evk.qk_norm_rope(x, None, y, None, H, gain_q=gainb, rot_dim=rot)
    keep = [i for i in range(dh) if i != rot]
    check(dgain[keep], gr[keep], rounded(gr, eg, dt)[keep], "dgain")
    assert not bool(torch.isfinite(dgain[rot]))
    check(y.reshape(yr.shape)[..., keep], yr[..., keep], tol[..., keep], "y")
    assert not bool(torch.isfinite(y.reshape(yr.shape)[..., rot]).any())


# --------------------------------------------------------------- activations --
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", DTYPES)
def test_activations_of_far_negative_values(act, dt):
    """Where exp(v) leaves fp32's normal range, v the sigmoid's argument, the
    result is still one of the storage type for a while: every value and
    derivative from -4 down.

    Relative error of the sigmoid there: the exponential's 2 + 1.2 |v| units of
    2^-23, 6 for the quotient and the products behind it, and for GELU six
    roundings of v itself, 3 |v| units; the derivatives' two terms of opposite
    sign stand 1 to 3.9 at least, (3.9 + 1) / (3.9 - 1) < 2."""
    lo = -100.0 if act == "silu" else -14.0
    z = torch.linspace(-4.0, lo, 8 * 4096, device="cuda").to(dt).view(512, 64)
    arg = z.double() if act == "silu" else math.sqrt(8 / math.pi) * (z.double() + 0.044715 * z.double() ** 3)
    rel = (8 + (1.2 if act == "silu" else 4.2) * arg.abs()) * 2.0 ** -23
    eye = torch.eye(64, dtype=dt, device="cuda")
    y = torch.empty_like(z)
    evk.linear(z, eye, y, act=ACTS[act])  # z itself is the product
    ref = act64_far(z.double(), act)
    check(y, ref, rounded(ref, rel * ref.abs(), dt), "act")
    dz, db = torch.empty_like(z), torch.empty(64, dtype=dt, device="cuda")
    evk.linear_backward(z, eye, torch.ones_like(z), dbias=db, act=ACTS[act], pre=z, dpre=dz)
    leaf = z.double().requires_grad_(True)
    ref, = torch.autograd.grad(act64_far(leaf, act).sum(), leaf)
    check(dz, ref, rounded(ref, 2 * rel * ref.abs(), dt), "act'")


def act64_far(z, name):
    """act64 without tanh's cancellation: z sigmoid(z), z sigmoid(2 u)."""
    return z * torch.sigmoid(z if name == "silu" else math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))


# ------------------------------------------------------------------ together --
def layer_ref(s, H, Hk, dh, dt=None, leave_out=()):
    """The decoder layer of test_gpu_layer_ops.py in 64 bits: as it is, with
    every stored tensor (and the attention's weights) rounded to dt, or without
    some of its parts."""
    w = {n: t.double() for n, t in s.items()}
    for n in ("gq", "gk"):
        if n in leave_out:
            w[n] = torch.ones_like(w[n])
    r = (lambda t: t.to(dt).double()) if dt else (lambda t: t)
    norm = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    x = w["x"]
    B, S, D = x.shape
    pos = torch.arange(S, device="cuda")[None].expand(B, S) * (0 if "rotation" in leave_out else 1)
    qkv = r(r(norm(x)) @ w["wqkv"] + (0 if "bias" in leave_out else w["bqkv"]))
    q, k, v = qkv.split([H * dh, Hk * dh, Hk * dh], -1)
    q = r(qk_ref(q, H, w["gq"], pos, 0, False, 10000.0, 1e-5)[0]).transpose(1, 2)
    k = r(qk_ref(k, Hk, w["gk"], pos, 0, False, 10000.0, 1e-5)[0]).transpose(1, 2).repeat_interleave(H // Hk, 1)
    v = v.reshape(B, S, Hk, dh).transpose(1, 2).repeat_interleave(H // Hk, 1)
    sc = (q @ k.transpose(2, 3)) / math.sqrt(dh)
    sc = sc.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    att = r((r(torch.softmax(sc, -1)) @ v).transpose(1, 2).reshape(B, S, D))
    x1 = r(att @ w["wo"] + (0 if "first residual" in leave_out else x))
    p = r(norm(x1)) @ w["wi"]
    F = p.shape[-1] // 2
    h = r((p[..., :F] if "activation" in leave_out else act64(p[..., :F], "silu")) * p[..., F:])
    return r(h @ w["wd"] + (0 if "second residual" in leave_out else x1))


@pytest.mark.parametrize("dt", DTYPES)
def test_decoder_layer_would_show_a_missing_part(dt):
    """The layer with gains and a bias that matter.  e is what rounding every
    stored tensor does to the 64-bit layer; the kernels round the same tensors,
    and their fp32 sums add little (K 2^-23 against 2^-11), so 3 e bounds them
    in the 2-norm.  Leaving any part out moves the result by 6 e at least."""
    B, S, H, Hk, dh, F = 2, 192, 8, 2, 64, 1368
    s = _layer_state(dt, B, S, H, Hk, dh, F, 4)
    g = gen(5)
    s["gq"], s["gk"] = (rnd(g, dt, dh, std=0.5, mean=1.0) for _ in range(2))
    s["bqkv"], s["wo"] = rnd(g, dt, (H + 2 * Hk) * dh, std=0.5), rnd(g, dt, H * dh, H * dh, std=2 * (H * dh) ** -0.5)
    y = _layer(s, H, Hk, dh).double()
    evk.check_device_error()
    ref = layer_ref(s, H, Hk, dh)
    far = lambda t: float((t - ref).norm())  # noqa: E731
    e = far(layer_ref(s, H, Hk, dh, dt))
    assert far(y) <= 3 * e, (far(y), e)
    for part in ("gq", "gk", "rotation", "bias", "first residual", "second residual", "activation"):
        assert far(layer_ref(s, H, Hk, dh, leave_out=(part,))) >= 6 * e, part


def test_calls_from_threads_of_their_own():
    """Host threads whose first CUDA call is an operator's, all at once: no
    refusal, and the bits of calls from the main thread."""
    dt, K, N = torch.bfloat16, 264, 520
    sets = []
    for rows in (1, 40, 130, 1030):
        g = gen(rows)
        x, w, wi, wo = rnd(g, dt, rows, K), rnd(g, dt, K, N), rnd(g, dt, K, 2 * N, std=0.1), rnd(g, dt, N, K, std=0.1)
        dy, q = rnd(g, dt, rows, N), rnd(g, dt, 1, rows, 128)
        e = lambda t: torch.empty_like(t)  # noqa: E731
        sets.append((x, w, wi, wo, dy, q, e(dy), e(x), e(w), e(x), e(dy), e(q), torch.cuda.Stream()))

    def work(x, w, wi, wo, dy, q, y, dx, dw, z, h, qo, stream):
        evk.linear(x, w, y, act=evk.ACT_SILU, stream=stream)
        evk.linear_backward(x, w, dy, dx=dx, dw=dw, stream=stream)
        evk.gated_ffn(x, wi, wo, z, h, stream=stream)
        evk.qk_norm_rope(q, None, qo, None, 2, stream=stream)
        stream.synchronize()
        return [t.clone() for t in (y, dx, dw, z, h, qo)]

    want = [work(*s) for s in sets]
    for s in sets:
        for t in s[6:12]:
            t.fill_(3.0)
    torch.cuda.synchronize()
    errors = []

    def thread(s):
        try:
            for _ in range(10):
                work(*s)
        except Exception as e:  # noqa: BLE001 - shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(s,)) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(s[6:12], w))
