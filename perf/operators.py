"""Cases of the decoder-layer operators around attention: `linear` (matrix
product with bias, activation and residual), `gated_ffn` (gated feed-forward
block) and `qk_norm_rope` (per-head query / key RMSNorm with the position
rotation), each forward and backward.

A case names one pass through one operator.  `run` computes it either in plain
form (elementary torch operations in 32 bits, one rounding at the end) or,
with `own`, through this package's entry points; `exact` computes the same
values in 64 bits from the definitions.
"""
import math

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases --
def _linear(name, rows, d_in, d_out, act, dtype, bias=True, residual=False, save_pre=False, nk=False):
    return dict(name=name, op="linear", rows=rows, d_in=d_in, d_out=d_out, act=act, dtype=dtype, bias=bias,
                residual=residual, save_pre=save_pre, nk=nk)


def _linear_bwd(name, rows, d_in, d_out, act, dtype, bias=True, nk=False):
    return dict(name=name, op="linear_backward", rows=rows, d_in=d_in, d_out=d_out, act=act, dtype=dtype, bias=bias,
                nk=nk)


def _ffn(name, rows, d, hidden, act, dtype, residual=True, save_pre=False, nk=False):
    return dict(name=name, op="gated_ffn", rows=rows, d=d, hidden=hidden, act=act, dtype=dtype, residual=residual,
                save_pre=save_pre, nk=nk)


def _ffn_bwd(name, rows, d, hidden, act, dtype, nk=False):
    return dict(name=name, op="gated_ffn_backward", rows=rows, d=d, hidden=hidden, act=act, dtype=dtype, nk=nk)


def _qk(name, batch, seq, heads, kv_heads, head_dim, dtype, rot_dim=0, half_split=False, gains=True, pos_offset=0,
        base=10000.0, cache_len=0):
    return dict(name=name, op="qk_norm_rope", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, rot_dim=rot_dim, half_split=half_split, gains=gains,
                pos_offset=pos_offset, base=base, cache_len=cache_len)


def _qk_bwd(name, batch, seq, heads, kv_heads, head_dim, dtype, rot_dim=0, half_split=False, gains=True,
            pos_offset=0, base=10000.0):
    c = _qk(name, batch, seq, heads, kv_heads, head_dim, dtype, rot_dim, half_split, gains, pos_offset, base)
    del c["cache_len"]
    c["op"] = "qk_norm_rope_backward"
    return c


def listed():
    return [
        # One decode step of the 512-wide decoder: its MLP's first projection for a single token.
        _linear("linear 1 token 512", 1, 512, 2048, "gelu", "fp16"),
        # Prefill of 8 x 2048 tokens of the 2048-wide decoder: the MLP's second projection with bias and residual.
        _linear("linear prefill 16384", 16384, 8192, 2048, "none", "bf16", residual=True),
        # Training step of the 2048-wide decoder's MLP: gradients of its first projection, 4 x 1024 tokens.
        _linear_bwd("linear backward 4096", 4096, 2048, 8192, "gelu", "bf16"),
        # The 512-wide decoder in training on a ragged batch of 1001 tokens, weights stored [out, in].
        _linear_bwd("linear backward ragged", 1001, 512, 2048, "relu", "fp16", nk=True),
        # One decode step of the 4096-wide decoder (hidden 14336), a single sequence.
        _ffn("ffn 1 token 4096", 1, 4096, 14336, "silu", "bf16"),
        # Training forward of the 2048-wide decoder's block: the pre-activations are kept for the backward pass.
        _ffn("ffn train 4096", 4096, 2048, 8192, "silu", "bf16", save_pre=True),
        # A short prompt through a small block with an odd hidden size, weights stored [out, in].
        _ffn("ffn ragged 333", 333, 512, 1368, "gelu", "fp16", nk=True),
        # Its training step's backward pass: gradients of the input and of all three weights.
        _ffn_bwd("ffn backward 4096", 4096, 2048, 8192, "silu", "bf16"),
        # One decode step of 8 sequences with grouped keys: keys and values go to their rows of the cache.
        _qk("qk decode 8", 8, 1, 32, 8, 128, "bf16", base=500000.0, cache_len=480),
        # Prefill of 8 x 2048 tokens of the 2048-wide decoder.
        _qk("qk prefill 16384", 8, 2048, 16, 16, 128, "bf16"),
        # A ragged batch with half-split pairs, a part of the head rotated, at far positions.
        _qk("qk ragged partial", 3, 777, 12, 4, 64, "fp16", rot_dim=32, half_split=True, pos_offset=120000),
        # Training step: gradients of queries, keys and both gains, 4 x 2048 tokens.
        _qk_bwd("qk backward 8192", 4, 2048, 32, 8, 128, "bf16"),
    ]


# The dearest listed cases, which bound the drawn ones.
_MAX_FLOPS = 12.0 * 4096 * 2048 * 8192
_MAX_ELEMS = 8 * 2048 * 48 * 128


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "gated_ffn", "gated_ffn", "gated_ffn_backward",
                     "qk_norm_rope", "qk_norm_rope", "qk_norm_rope_backward"])
    dtype = rng.choice(["fp16", "bf16"])
    if op.startswith("qk"):
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        half_split = rng.random() < 0.5
        rot = rng.choice([0, 0, dh // 2 // 16 * 16])
        batch = _log_int(rng, 1, 64)
        cap = max(1, _MAX_ELEMS // ((heads + 2 * kv) * dh * batch))
        pos = rng.choice([0, rng.randrange(5000), rng.randrange(1000000)])
        base = rng.choice([10000.0, 500000.0])
        gains = rng.random() < 0.8
        if op == "qk_norm_rope_backward":
            c = _qk_bwd("", batch, _log_int(rng, 1, min(cap, 4096)), heads, kv, dh, dtype, rot, half_split, gains,
                        pos, base)
        elif rng.random() < 0.4:
            c = _qk("", batch, 1, heads, kv, dh, dtype, rot, half_split, gains, 0, base,
                    _log_int(rng, 16, max(17, min(2048, 3900000 // (batch * kv * dh)))))
        else:
            c = _qk("", batch, _log_int(rng, 1, min(cap, 4096)), heads, kv, dh, dtype, rot, half_split, gains, pos,
                    base)
    else:
        per = {"linear": 2, "linear_backward": 4, "gated_ffn": 6, "gated_ffn_backward": 12}[op]
        d = _log_int(rng, 64, 4096, 8)
        e = _log_int(rng, 64, 14336, 8)
        top = int(min(16384, _MAX_FLOPS // (per * d * e)))
        decode = op in ("linear", "gated_ffn") and rng.random() < 0.4
        rows = _log_int(rng, 1, min(top, 64 if decode else top))
        act = rng.choice(["gelu", "silu", "relu"])
        nk = rng.random() < 0.3
        if op == "linear":
            c = _linear("", rows, d, e, rng.choice([act, "none"]), dtype, rng.random() < 0.6, rng.random() < 0.5,
                        rng.random() < 0.3, nk)
        elif op == "linear_backward":
            c = _linear_bwd("", rows, d, e, rng.choice([act, "none"]), dtype, rng.random() < 0.6, nk)
        elif op == "gated_ffn":
            c = _ffn("", rows, d, e, act, dtype, rng.random() < 0.6, rng.random() < 0.4, nk)
        else:
            c = _ffn_bwd("", rows, d, e, act, dtype, nk)
    del c["name"]
    return c


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]

    def n(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)

    def empty(*shape):
        return torch.empty(*shape, dtype=dt, device="cuda")

    def weight(a, b):  # a x b, or stored transposed
        return n(b, a, std=0.02) if case["nk"] else n(a, b, std=0.02)

    s = dict(case=case)
    op = case["op"]
    if op.startswith("linear"):
        m, k, o = case["rows"], case["d_in"], case["d_out"]
        s["x"], s["w"] = n(m, k), weight(k, o)
        if op == "linear":
            s["bias"] = n(o, std=0.1) if case["bias"] else None
            s["residual"] = n(m, o) if case["residual"] else None
            s["y"] = empty(m, o)
            s["pre"] = empty(m, o) if case["save_pre"] else None
        else:
            s["dy"] = n(m, o)
            s["pre"] = n(m, o) if case["act"] != "none" else None  # the forward pass's saved pre-activation
            s["dpre"] = empty(m, o) if case["act"] != "none" else None
            s["dx"], s["dw"] = empty(*s["x"].shape), empty(*s["w"].shape)
            s["dbias"] = empty(o) if case["bias"] else None
    elif op.startswith("gated_ffn"):
        m, d, f = case["rows"], case["d"], case["hidden"]
        s["x"], s["w_in"], s["w_out"] = n(m, d), weight(d, 2 * f), weight(f, d)
        s["hidden"] = empty(m, f)
        if op == "gated_ffn":
            s["residual"] = n(m, d) if case["residual"] else None
            s["y"] = empty(m, d)
            s["pre"] = empty(m, 2 * f) if case["save_pre"] else None
        else:
            s["pre"], s["dy"] = n(m, 2 * f), n(m, d)
            s["dpre"] = empty(m, 2 * f)
            s["dx"], s["dw_in"], s["dw_out"] = empty(m, d), empty(*s["w_in"].shape), empty(*s["w_out"].shape)
    else:
        b, t, h, kv, dh = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
        qkv = n(b, t, (h + 2 * kv) * dh)  # the fused projection's output
        s["q"], s["k"], s["v"] = qkv.split([h * dh, kv * dh, kv * dh], dim=-1)
        s["gain_q"] = n(dh, std=0.1, mean=1.0) if case["gains"] else None
        s["gain_k"] = n(dh, std=0.1, mean=1.0) if case["gains"] else None
        if op == "qk_norm_rope":
            s["q_out"] = empty(b, t, h * dh)
            if case["cache_len"]:
                s["positions"] = torch.randint(0, case["cache_len"], (b, t), generator=g, device="cuda",
                                               dtype=torch.int32)
                s["k_out"], s["v_out"] = n(b, case["cache_len"], kv * dh), n(b, case["cache_len"], kv * dh)
            else:
                s["positions"], s["k_out"] = None, empty(b, t, kv * dh)
        else:
            s["positions"] = None
            s["dq_out"], s["dk_out"] = n(b, t, h * dh), n(b, t, kv * dh)
            dqkv = empty(b, t, (h + 2 * kv) * dh)
            s["dq"], s["dk"], _ = dqkv.split([h * dh, kv * dh, kv * dh], dim=-1)
            s["dgain_q"] = empty(dh) if case["gains"] else None
            s["dgain_k"] = empty(dh) if case["gains"] else None
            s["workspace"] = torch.empty(8192 * dh, dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------- plain form --
def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _dact(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


def _w(t, c):
    return t.float().t() if c["nk"] else t.float()


def _plain_linear(s, c, dt):
    z = torch.matmul(s["x"].float(), _w(s["w"], c))
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(dt), pre=z.to(dt)) if c["save_pre"] else dict(y=y.to(dt))


def _plain_linear_backward(s, c, dt):
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _dact(s["pre"].float(), c["act"])
    dw = torch.matmul(s["x"].float().t(), dz)
    out = dict(dx=torch.matmul(dz, _w(s["w"], c).t()).to(dt), dw=(dw.t() if c["nk"] else dw).contiguous().to(dt))
    if c["bias"]:
        out["dbias"] = dz.sum(0).to(dt)
    return out


def _plain_gated_ffn(s, c, dt):
    z = torch.matmul(s["x"].float(), _w(s["w_in"], c))
    f = c["hidden"]
    y = torch.matmul(_act(z[:, :f], c["act"]) * z[:, f:], _w(s["w_out"], c))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(dt), pre=z.to(dt)) if c["save_pre"] else dict(y=y.to(dt))


def _plain_gated_ffn_backward(s, c, dt):
    f = c["hidden"]
    gate, up = s["pre"][:, :f].float(), s["pre"][:, f:].float()
    dy, a = s["dy"].float(), _act(gate, c["act"])
    dh = torch.matmul(dy, _w(s["w_out"], c).t())
    dpre = torch.cat([dh * up * _dact(gate, c["act"]), dh * a], dim=1)
    dw_out = torch.matmul((a * up).t(), dy)
    dw_in = torch.matmul(s["x"].float().t(), dpre)
    dx = torch.matmul(dpre, _w(s["w_in"], c).t())
    return dict(dx=dx.to(dt), dw_in=(dw_in.t() if c["nk"] else dw_in).contiguous().to(dt),
                dw_out=(dw_out.t() if c["nk"] else dw_out).contiguous().to(dt))


def _angles(s, c):
    """cos, sin [B or 1, S, 1, rot / 2] of each position's angles, in 64 bits until the end."""
    rot = c["rot_dim"] or c["head_dim"]
    if s["positions"] is not None:
        pos = s["positions"].double()
    else:
        pos = torch.arange(c["seq"], device="cuda", dtype=torch.float64)[None] + c["pos_offset"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    ang = pos[..., None] * torch.pow(torch.tensor(c["base"], device="cuda", dtype=torch.float64), -2 * i / rot)
    return torch.cos(ang).float()[:, :, None, :], torch.sin(ang).float()[:, :, None, :], rot


def _rotate(x, cos, sin, rot, half_split):
    out = x.clone()
    if half_split:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return out


_EPS = 1e-5


def _plain_qk(s, c, dt):
    cos, sin, rot = _angles(s, c)

    def one(x, heads, gain):
        x = x.float().reshape(c["batch"], c["seq"], heads, c["head_dim"])
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        if gain is not None:
            x = x * gain.float()
        return _rotate(x, cos, sin, rot, c["half_split"]).reshape(c["batch"], c["seq"], -1).to(dt)

    q, k = one(s["q"], c["heads"], s["gain_q"]), one(s["k"], c["kv_heads"], s["gain_k"])
    if not c["cache_len"]:
        return dict(q=q, k=k)
    at = (torch.arange(c["batch"], device="cuda")[:, None], s["positions"].long())
    s["k_out"][at] = k
    s["v_out"][at] = s["v"]
    return dict(q=q, kcache=s["k_out"], vcache=s["v_out"])


def _plain_qk_backward(s, c, dt):
    cos, sin, rot = _angles(s, c)

    def one(x, dy, heads, gain):
        shape = (c["batch"], c["seq"], heads, c["head_dim"])
        x, t = x.float().reshape(shape), _rotate(dy.float().reshape(shape), cos, -sin, rot, c["half_split"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        nrm = x * r
        dg = (t * nrm).sum((0, 1, 2))
        dn = t if gain is None else t * gain.float()
        dx = r * (dn - nrm * (dn * nrm).mean(-1, keepdim=True))
        return dx.reshape(c["batch"], c["seq"], -1).to(dt), dg.to(dt)

    dq, dgq = one(s["q"], s["dq_out"], c["heads"], s["gain_q"])
    dk, dgk = one(s["k"], s["dk_out"], c["kv_heads"], s["gain_k"])
    return dict(dq=dq, dk=dk, dgain_q=dgq, dgain_k=dgk) if c["gains"] else dict(dq=dq, dk=dk)


_PLAIN = {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "gated_ffn": _plain_gated_ffn,
          "gated_ffn_backward": _plain_gated_ffn_backward, "qk_norm_rope": _plain_qk,
          "qk_norm_rope_backward": _plain_qk_backward}


# ------------------------------------------------------------ the package's --
def _own(s, c):
    import evk_b200 as evk

    op = c["op"]
    if op.startswith("qk"):
        rope = dict(positions=s["positions"], rot_dim=c["rot_dim"], half_split=c["half_split"], eps=_EPS,
                    base=c["base"], pos_offset=c["pos_offset"])
        if op == "qk_norm_rope":
            if c["cache_len"]:
                evk.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], c["heads"], gain_q=s["gain_q"],
                                 gain_k=s["gain_k"], v=s["v"], v_out=s["v_out"], cache=True, **rope)
                return dict(q=s["q_out"], kcache=s["k_out"], vcache=s["v_out"])
            evk.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], c["heads"], gain_q=s["gain_q"],
                             gain_k=s["gain_k"], **rope)
            return dict(q=s["q_out"], k=s["k_out"])
        evk.qk_norm_rope_backward(s["q"], s["k"], s["dq_out"], s["dk_out"], s["dq"], s["dk"], c["heads"],
                                  gain_q=s["gain_q"], gain_k=s["gain_k"], dgain_q=s["dgain_q"],
                                  dgain_k=s["dgain_k"], workspace=s["workspace"], **rope)
        if c["gains"]:
            return dict(dq=s["dq"], dk=s["dk"], dgain_q=s["dgain_q"], dgain_k=s["dgain_k"])
        return dict(dq=s["dq"], dk=s["dk"])
    act = {"none": evk.ACT_NONE, "relu": evk.ACT_RELU, "gelu": evk.ACT_GELU, "silu": evk.ACT_SILU}[c["act"]]
    if op == "linear":
        evk.linear(s["x"], s["w"], s["y"], bias=s["bias"], residual=s["residual"], act=act, pre=s["pre"],
                   transpose_w=c["nk"])
        return dict(y=s["y"], pre=s["pre"]) if c["save_pre"] else dict(y=s["y"])
    if op == "linear_backward":
        evk.linear_backward(s["x"], s["w"], s["dy"], dx=s["dx"], dw=s["dw"], dbias=s["dbias"], act=act, pre=s["pre"],
                            dpre=s["dpre"], transpose_w=c["nk"])
        out = dict(dx=s["dx"], dw=s["dw"])
        if c["bias"]:
            out["dbias"] = s["dbias"]
        return out
    if op == "gated_ffn":
        evk.gated_ffn(s["x"], s["w_in"], s["w_out"], s["y"], s["hidden"], act=act, residual=s["residual"],
                      pre=s["pre"], transpose_w=c["nk"])
        return dict(y=s["y"], pre=s["pre"]) if c["save_pre"] else dict(y=s["y"])
    evk.gated_ffn_backward(s["x"], s["w_in"], s["w_out"], s["pre"], s["dy"], s["dpre"], s["hidden"], dx=s["dx"],
                           dw_in=s["dw_in"], dw_out=s["dw_out"], act=act, transpose_w=c["nk"])
    return dict(dx=s["dx"], dw_in=s["dw_in"], dw_out=s["dw_out"])


def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    return _PLAIN[c["op"]](state, c, _DT[c["dtype"]])


# -------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    if op.startswith("linear"):
        m, k, o = case["rows"], case["d_in"], case["d_out"]
        if op == "linear":
            elems = m * k + k * o + m * o * (1 + case["residual"] + case["save_pre"]) + o * case["bias"]
            return {"bytes": 2 * elems, "flops": 2 * m * k * o}
        elems = 2 * (m * k + k * o) + m * o * (1 + (case["act"] != "none")) + o * case["bias"]
        return {"bytes": 2 * elems, "flops": 4 * m * k * o}
    if op.startswith("gated_ffn"):
        m, d, f = case["rows"], case["d"], case["hidden"]
        if op == "gated_ffn":
            elems = m * d * (2 + case["residual"]) + 3 * d * f + 2 * m * f * case["save_pre"]
            return {"bytes": 2 * elems, "flops": 6 * m * d * f}
        return {"bytes": 2 * (3 * m * d + 6 * d * f + 2 * m * f), "flops": 12 * m * d * f}
    rows, h, kv, dh = case["batch"] * case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    if op == "qk_norm_rope":
        heads = h + (2 * kv if case["cache_len"] else kv)
        return {"bytes": 2 * (2 * rows * heads * dh + 2 * dh * case["gains"]), "flops": 9 * rows * (h + kv) * dh}
    return {"bytes": 2 * (3 * rows * (h + kv) * dh + 4 * dh * case["gains"]), "flops": 17 * rows * (h + kv) * dh}


# ------------------------------------------------------------------- exact --
def _exact_act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":  # 0.5 (1 + tanh u) = sigmoid(2 u)
        return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z * 1


def _exact_heads(x, heads, gain, c, pos):
    """norm and rotation of [B, S, heads * Dh] in 64 bits, the pairs as complex numbers."""
    dh, rot = c["head_dim"], c["rot_dim"] or c["head_dim"]
    x = x.view(c["batch"], c["seq"], heads, dh)
    x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / dh + _EPS)
    if gain is not None:
        x = x * gain
    freq = torch.exp(torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) * (-math.log(c["base"]) / rot))
    ang = torch.einsum("bs,f->bsf", pos, freq)[:, :, None]
    turn = torch.polar(torch.ones_like(ang), ang)
    head, rest = x[..., :rot], x[..., rot:]
    if c["half_split"]:
        z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat([head, rest], -1).reshape(c["batch"], c["seq"], heads * dh)


def exact(case, seed):
    s, c = prepare(case, seed), case
    s = {k: (v.double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    op = c["op"]
    tr = (lambda t: t.t()) if op[0] != "q" and c["nk"] else (lambda t: t)
    if op == "linear":
        z = s["x"] @ tr(s["w"])
        if s["bias"] is not None:
            z += s["bias"]
        y = _exact_act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"]
        return dict(y=y, pre=z) if c["save_pre"] else dict(y=y)
    if op == "linear_backward":
        dz = s["dy"]
        if c["act"] != "none":
            z = s["pre"].requires_grad_(True)
            dz, = torch.autograd.grad(_exact_act(z, c["act"]), z, s["dy"])
        w = s["w"]
        out = dict(dx=dz @ tr(w).t(), dw=dz.t() @ s["x"] if c["nk"] else s["x"].t() @ dz)
        if c["bias"]:
            out["dbias"] = torch.ones(1, dz.shape[0], device="cuda", dtype=torch.float64) @ dz
            out["dbias"] = out["dbias"][0]
        return out
    if op == "gated_ffn":
        z = s["x"] @ tr(s["w_in"])
        gate, up = z.chunk(2, dim=1)
        y = (_exact_act(gate, c["act"]) * up) @ tr(s["w_out"])
        if s["residual"] is not None:
            y += s["residual"]
        return dict(y=y, pre=z) if c["save_pre"] else dict(y=y)
    if op == "gated_ffn_backward":
        z = s["pre"].requires_grad_(True)
        w = s["w_out"].requires_grad_(True)
        gate, up = z.chunk(2, dim=1)
        y = (_exact_act(gate, c["act"]) * up) @ tr(w)
        dz, dw_out = torch.autograd.grad(y, (z, w), s["dy"])
        return dict(dx=dz @ tr(s["w_in"]).t(), dw_in=dz.t() @ s["x"] if c["nk"] else s["x"].t() @ dz, dw_out=dw_out)
    if s["positions"] is not None:
        pos = s["positions"].double()
    else:
        pos = (torch.arange(c["seq"], device="cuda", dtype=torch.float64) + c["pos_offset"]).expand(c["batch"], -1)
    if op == "qk_norm_rope":
        q = _exact_heads(s["q"].contiguous(), c["heads"], s["gain_q"], c, pos)
        k = _exact_heads(s["k"].contiguous(), c["kv_heads"], s["gain_k"], c, pos)
        if not c["cache_len"]:
            return dict(q=q, k=k)
        kc, vc = s["k_out"], s["v_out"]
        for b in range(c["batch"]):
            for t in range(c["seq"]):
                p = int(s["positions"][b, t])
                kc[b, p], vc[b, p] = k[b, t], s["v"][b, t]
        return dict(q=q, kcache=kc, vcache=vc)
    out = {}
    for x, heads in (("q", c["heads"]), ("k", c["kv_heads"])):
        leaf = s[x].contiguous().requires_grad_(True)
        gain = s["gain_" + x]
        gain = gain.requires_grad_(True) if gain is not None else None
        y = _exact_heads(leaf, heads, gain, c, pos)
        got = torch.autograd.grad(y, [leaf] + ([gain] if gain is not None else []), s["d%s_out" % x])
        out["d" + x] = got[0]
        if gain is not None:
            out["dgain_" + x] = got[1]
    return out
