"""Calls of the decoder-layer operators that the Python binding and the C++
layer turn away before anything is computed; none needs a GPU."""
import os
import signal
import subprocess

import pytest
import torch

import evk_b200 as evk
from conftest import ROOT

SHAPE, ARG = 1, 7
BIG = 1 << 32


def meta(*shape):
    """A tensor of that shape and type without memory."""
    return torch.empty(*shape, dtype=torch.float16, device="meta")


def refused(status, f, *a, **kw):
    with pytest.raises(evk.EvkcuError) as e:
        f(*a, **kw)
    assert e.value.status == status, e.value


@pytest.mark.parametrize("rows,K,N", [(BIG, 8, 8), (BIG + 5, 8, 16), (1, BIG, 8), (1, 8, BIG), (3, 8, BIG + 8)])
def test_sizes_past_32_bits_are_refused(rows, K, N):
    """The C ABI takes 32-bit sizes; a call must not be cut to its low bits."""
    x, w, y = meta(rows, K), meta(K, N), meta(rows, N)
    refused(SHAPE, evk.linear, x, w, y)
    refused(SHAPE, evk.linear, x.view(rows, 1, K), w, y.view(rows, 1, N))
    refused(SHAPE, evk.linear_backward, x, w, y, dx=meta(rows, K))
    refused(SHAPE, evk.gated_ffn, x, meta(K, 2 * N), meta(N, K), meta(rows, K), y)
    refused(SHAPE, evk.gated_ffn_backward, x, meta(K, 2 * N), meta(N, K), meta(rows, 2 * N), meta(rows, K),
            meta(rows, 2 * N), y, dx=meta(rows, K))


@pytest.mark.parametrize("B,S,H,dh", [(BIG, 1, 1, 8), (1, BIG + 3, 1, 8), (1, 1, BIG, 8), (2, 1, BIG + 2, 8)])
def test_qk_sizes_past_32_bits_are_refused(B, S, H, dh):
    q = meta(B, S, H * dh)
    refused(SHAPE, evk.qk_norm_rope, q, None, meta(B, S, H * dh), None, H)
    refused(SHAPE, evk.qk_norm_rope_backward, q, None, q, None, meta(B, S, H * dh), None, H)


def test_keys_and_caches_past_32_bits_are_refused():
    q, k = meta(1, 1, 8), meta(1, 1, 8)
    refused(SHAPE, evk.qk_norm_rope, q, meta(1, 1, 8 * BIG), meta(1, 1, 8), meta(1, 1, 8 * BIG), 1)
    refused(SHAPE, evk.qk_norm_rope, q, k, meta(1, 1, 8), meta(1, BIG + 4, 8), 1, cache=True)


def test_missing_tensors_are_refused():
    """None for a tensor that gives the binding a call's shapes: its error, with
    a status (the others are refused by the C ABI)."""
    t, w = meta(4, 8), meta(8, 8)
    for n in ("x", "y"):
        refused(ARG, evk.linear, **{**dict(x=t, w=w, y=t), n: None})
    for n in ("x", "dy"):
        refused(ARG, evk.linear_backward, **{**dict(x=t, w=w, dy=t), n: None})
    for n in ("x", "hidden"):
        refused(ARG, evk.gated_ffn, **{**dict(x=t, w_in=meta(8, 16), w_out=w, y=t, hidden=t), n: None})
    back = dict(x=t, w_in=meta(8, 16), w_out=w, pre=meta(4, 16), dy=t, dpre=meta(4, 16), hidden=t)
    for n in ("x", "pre"):
        refused(ARG, evk.gated_ffn_backward, **{**back, n: None})
    q = meta(1, 2, 16)
    for n in ("q", "q_out", "k_out"):
        refused(ARG, evk.qk_norm_rope, **{**dict(q=q, k=q, q_out=q, k_out=q, heads=2), n: None})
    refused(ARG, evk.qk_norm_rope, q, q, q, None, 2, cache=True)
    for n in ("q", "dq_out", "dq", "dk_out", "dk"):
        refused(ARG, evk.qk_norm_rope_backward,
                **{**dict(q=q, k=q, dq_out=q, dk_out=q, dq=q, dk=q, heads=2), n: None})


REFUSALS = os.path.join(ROOT, "evk_b200", "reftests", "layer_refusals")


@pytest.mark.skipif(not os.path.exists(REFUSALS), reason="layer_refusals not built")
@pytest.mark.parametrize("case", ["linear of nothing", "linear_backward of nothing", "gated_ffn of nothing",
                                  "gated_ffn_backward of nothing", "linear past 32 bits",
                                  "linear_backward past 32 bits", "gated_ffn past 32 bits",
                                  "gated_ffn_backward past 32 bits", "qk_norm_rope past 32 bits",
                                  "qk_norm_rope_backward past 32 bits"])
def test_cpp_layer_refuses(case):
    """The C++ layer's refusal: its message with EVKCU_BAD_SHAPE, then abort."""
    r = subprocess.run([REFUSALS, case], capture_output=True, text=True, timeout=120)
    assert r.returncode == -signal.SIGABRT, (r.returncode, r.stdout, r.stderr)
    assert f"evk::ai::{case.split()[0]}" in r.stderr and "failed (status 1)" in r.stderr
