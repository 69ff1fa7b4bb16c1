"""Refusals of the decoder-layer operators (evkcu_linear, evkcu_gated_ffn,
evkcu_qk_norm_rope and their backward passes): every bad call is turned away
with a status before any CUDA call, so these need no GPU.  The pointers are
never read."""
import ctypes

import pytest

import evk_b200 as evk

OK, SHAPE, ALIGN, ARG = 0, 1, 2, 7
P = [0x100000 * (i + 1) for i in range(16)]  # distinct, 16-byte aligned


@pytest.fixture(scope="module")
def lib():
    return evk.lib()


def _linear(lib, x=P[0], w=P[1], bias=P[2], res=P[3], y=P[4], pre=P[5], rows=4, K=16, N=24, act=0, flags=0, dtype=0):
    return lib.evkcu_linear(x, w, bias, res, y, pre, rows, K, N, act, flags, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), ARG), (dict(w=None), ARG), (dict(y=None), ARG), (dict(dtype=2), ARG), (dict(dtype=-1), ARG),
    (dict(act=4), ARG), (dict(act=-1), ARG), (dict(flags=1), ARG), (dict(flags=4), ARG), (dict(K=0), SHAPE),
    (dict(N=0), SHAPE), (dict(K=12), SHAPE), (dict(N=20), SHAPE), (dict(rows=(1 << 30) + 1), SHAPE),
    (dict(x=P[0] + 8), ALIGN), (dict(w=P[1] + 2), ALIGN), (dict(bias=P[2] + 4), ALIGN), (dict(res=P[3] + 8), ALIGN),
    (dict(y=P[4] + 8), ALIGN), (dict(pre=P[5] + 8), ALIGN), (dict(y=P[0]), ARG), (dict(y=P[1]), ARG),
    (dict(pre=P[4]), ARG), (dict(pre=P[0]), ARG), (dict(pre=P[3]), ARG), (dict(y=P[2]), ARG), (dict(rows=0), OK),
    (dict(rows=0, x=None, w=None, y=None), OK),
])
def test_linear_refuses(lib, kw, status):
    assert _linear(lib, **kw) == status
    if status:
        assert "evkcu_linear" in lib.evkcu_last_error().decode()


def _linear_bwd(lib, x=P[0], w=P[1], pre=P[2], dy=P[3], dpre=P[4], dx=P[5], dw=P[6], dbias=P[7], rows=4, K=16, N=24,
                act=2, flags=0, dtype=1):
    return lib.evkcu_linear_backward(x, w, pre, dy, dpre, dx, dw, dbias, rows, K, N, act, flags, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), ARG), (dict(w=None), ARG), (dict(dy=None), ARG), (dict(pre=None), ARG), (dict(dpre=None), ARG),
    (dict(flags=1), ARG), (dict(flags=8), ARG), (dict(act=9), ARG), (dict(dtype=7), ARG), (dict(K=4), SHAPE),
    (dict(N=9), SHAPE), (dict(dx=P[5] + 8), ALIGN), (dict(dw=P[6] + 8), ALIGN), (dict(dbias=P[7] + 8), ALIGN),
    (dict(dx=P[3]), ARG), (dict(dx=P[4]), ARG), (dict(dx=P[1]), ARG), (dict(dw=P[0]), ARG), (dict(dw=P[4]), ARG),
    (dict(dw=P[1]), ARG), (dict(dx=P[0]), ARG), (dict(dpre=P[0]), ARG), (dict(dw=P[5]), ARG), (dict(dbias=P[3]), ARG),
])
def test_linear_backward_refuses(lib, kw, status):
    assert _linear_bwd(lib, **kw) == status


def _ffn(lib, x=P[0], wi=P[1], wo=P[2], res=P[3], y=P[4], h=P[5], pre=P[6], rows=4, D=16, F=24, act=3, flags=0,
         dtype=1):
    return lib.evkcu_gated_ffn(x, wi, wo, res, y, h, pre, rows, D, F, act, flags, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), ARG), (dict(wi=None), ARG), (dict(wo=None), ARG), (dict(h=None), ARG), (dict(flags=4), ARG),
    (dict(act=5), ARG), (dict(dtype=3), ARG), (dict(D=0), SHAPE), (dict(F=0), SHAPE), (dict(F=12), SHAPE),
    (dict(D=20), SHAPE), (dict(F=(1 << 29) + 8), SHAPE), (dict(h=P[5] + 8), ALIGN), (dict(wi=P[1] + 8), ALIGN),
    (dict(h=P[0]), ARG), (dict(h=P[4]), ARG), (dict(pre=P[5]), ARG), (dict(pre=P[0]), ARG), (dict(pre=P[4]), ARG),
    (dict(pre=P[3]), ARG), (dict(h=P[3]), ARG), (dict(y=P[2]), ARG), (dict(rows=0), OK),
])
def test_gated_ffn_refuses(lib, kw, status):
    assert _ffn(lib, **kw) == status


def _ffn_bwd(lib, x=P[0], wi=P[1], wo=P[2], pre=P[3], dy=P[4], dpre=P[5], h=P[6], dx=P[7], dwi=P[8], dwo=P[9], rows=4,
             D=16, F=24, act=3, flags=0, dtype=0):
    return lib.evkcu_gated_ffn_backward(x, wi, wo, pre, dy, dpre, h, dx, dwi, dwo, rows, D, F, act, flags, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), ARG), (dict(wi=None), ARG), (dict(wo=None), ARG), (dict(pre=None), ARG), (dict(dy=None), ARG),
    (dict(dpre=None), ARG), (dict(h=None), ARG), (dict(flags=1), ARG), (dict(D=4), SHAPE), (dict(F=4), SHAPE),
    (dict(dx=P[7] + 8), ALIGN), (dict(dpre=P[5] + 8), ALIGN), (dict(dpre=P[4]), ARG), (dict(dx=P[5]), ARG),
    (dict(dx=P[4]), ARG), (dict(h=P[5]), ARG), (dict(h=P[3]), ARG), (dict(dwi=P[1]), ARG), (dict(dwo=P[2]), ARG),
    (dict(dwo=P[6]), ARG), (dict(dwi=P[8], dwo=P[8]), ARG), (dict(h=P[4]), ARG),
])
def test_gated_ffn_backward_refuses(lib, kw, status):
    assert _ffn_bwd(lib, **kw) == status


def _desc(**kw):
    d = dict(batch=2, seq_len=3, heads=4, kv_heads=2, head_dim=64, rot_dim=0, flags=0, pos_offset=0, cache_len=0,
             eps=1e-5, base=10000.0, positions=None, q_pitch=512, k_pitch=512, v_pitch=512, q_out_pitch=256,
             k_out_pitch=128, dq_pitch=256, dk_pitch=128)
    d.update(kw)
    return evk.QkNormRopeDesc(**d)


def _qk(lib, q=P[0], k=P[1], v=None, gq=P[2], gk=P[3], qo=P[4], ko=P[5], vo=None, dtype=1, **kw):
    return lib.evkcu_qk_norm_rope(ctypes.byref(_desc(**kw)), q, k, v, gq, gk, qo, ko, vo, dtype, None)


DESC_REFUSALS = [
    (dict(head_dim=0), SHAPE), (dict(head_dim=4), SHAPE), (dict(head_dim=68), SHAPE), (dict(head_dim=264), SHAPE),
    (dict(rot_dim=66), SHAPE), (dict(rot_dim=7), SHAPE), (dict(rot_dim=24, flags=1), SHAPE), (dict(flags=8), ARG),
    (dict(head_dim=72, flags=1, q_pitch=1024, k_pitch=1024, q_out_pitch=512, k_out_pitch=512), SHAPE),
    (dict(heads=0), SHAPE), (dict(heads=70000), SHAPE), (dict(kv_heads=70000), SHAPE), (dict(eps=-1.0), ARG),
    (dict(eps=float("nan")), ARG), (dict(base=0.0), ARG), (dict(base=float("inf")), ARG), (dict(dtype=2), ARG),
    (dict(base=float("nan")), ARG), (dict(pos_offset=0x7FFFFFFF), SHAPE), (dict(batch=1 << 20, seq_len=1 << 20), SHAPE),
    (dict(q=None), ARG), (dict(k=None), ARG), (dict(q=P[0] + 8), ALIGN), (dict(k=P[1] + 2), ALIGN),
    (dict(gq=P[2] + 8), ALIGN), (dict(q_pitch=248), SHAPE), (dict(k_pitch=132), SHAPE), (dict(k_out_pitch=120), SHAPE),
    (dict(q_out_pitch=260), SHAPE), (dict(positions=P[6] + 2), ALIGN),
]


@pytest.mark.parametrize("kw,status", DESC_REFUSALS + [
    (dict(flags=2), SHAPE), (dict(flags=4), ARG), (dict(v=P[6]), ARG), (dict(vo=P[7]), ARG),
    (dict(qo=None), ARG), (dict(ko=None), ARG), (dict(v=P[6], vo=P[7] + 8), ALIGN),
    (dict(v=P[6], vo=P[7], v_pitch=64), SHAPE),
    (dict(qo=P[0]), ARG), (dict(ko=P[1]), ARG), (dict(qo=P[5]), ARG), (dict(ko=P[2], gk=None), ARG),
    (dict(flags=2, cache_len=5, ko=P[1], k_pitch=128), ARG), (dict(batch=0), OK), (dict(seq_len=0), OK),
])
def test_qk_norm_rope_refuses(lib, kw, status):
    assert _qk(lib, **kw) == status


def test_qk_norm_rope_refuses_a_missing_descriptor(lib):
    assert lib.evkcu_qk_norm_rope(None, P[0], P[1], None, None, None, P[2], P[3], None, 0, None) == ARG


def _qk_bwd(lib, q=P[0], k=P[1], gq=P[2], gk=P[3], dqo=P[4], dko=P[5], dq=P[6], dk=P[7], dgq=P[8], dgk=P[9], ws=P[10],
            wbytes=1 << 20, dtype=1, **kw):
    return lib.evkcu_qk_norm_rope_backward(ctypes.byref(_desc(**kw)), q, k, gq, gk, dqo, dko, dq, dk, dgq, dgk, ws,
                                           wbytes, dtype, None)


@pytest.mark.parametrize("kw,status", DESC_REFUSALS + [
    (dict(flags=2), ARG), (dict(ws=None), ARG), (dict(wbytes=8192 * 64 - 1), ARG), (dict(ws=P[10] + 8), ALIGN),
    (dict(dqo=None), ARG), (dict(dko=None), ARG), (dict(dq=None), ARG), (dict(dk=None), ARG),
    (dict(dq_pitch=128), SHAPE), (dict(dk_pitch=120), SHAPE), (dict(dq=P[0]), ARG), (dict(dk=P[1]), ARG),
    (dict(dq=P[4], dq_pitch=512), ARG),
])
def test_qk_norm_rope_backward_refuses(lib, kw, status):
    assert _qk_bwd(lib, **kw) == status


def test_workspace_size(lib):
    assert evk.qk_norm_rope_workspace(128) == 8192 * 128


def test_python_binding_refuses_cpu_tensors():
    import torch

    x, w, y = torch.zeros(2, 16).half(), torch.zeros(16, 8).half(), torch.zeros(2, 8).half()
    with pytest.raises(ValueError):
        evk.linear(x, w, y)
    q = torch.zeros(1, 2, 64).half()
    with pytest.raises(ValueError):
        evk.qk_norm_rope(q, None, q.clone(), None, 1)
    with pytest.raises(evk.EvkcuError):
        evk.linear(x, w, torch.zeros(2, 16).half())  # w is not (16, 16)
    with pytest.raises(evk.EvkcuError):
        evk.linear(x, w.bfloat16(), y)
