"""evk_b200 — B200 (sm_100a) backend for the evk::ai inference operators.

The product is the C ABI in ``include/evkcu.h`` (``libevkcu.so``) and the
C++20 ``evk::ai`` layer above it (``libevk_ai.so``).  This module binds the C
ABI with ctypes so Python callers (tests, ``bench.py``) can drive the kernels
on torch-allocated device memory.  It is a thin binding: no kernel runs
anywhere but in ``libevkcu.so``, and importing it fails loudly when the
library has not been built.

Function names follow the reference's operators (carloshgsilva/evk
``evk_ai.h:489-615``); argument meaning follows ``include/evkcu.h``.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libevkcu.so")
AI_LIB_PATH = os.path.join(_HERE, "libevk_ai.so")

F16 = 0
BF16 = 1
MM_TRANSPOSE_A = 1
MM_TRANSPOSE_B = 2
MM_ACC_C = 4
ATTN_CAUSAL = 1
ATTN_BWD_NORMALIZED = 2
ACT_NONE = 0
ACT_RELU = 1
ACT_GELU = 2
ACT_SILU = 3
QK_HALF_SPLIT = 1
QK_CACHE = 2
QK_ACC_GAIN = 4

STATUS = {
    0: "OK",
    1: "BAD_SHAPE",
    2: "BAD_ALIGN",
    3: "CUDA_ERROR",
    4: "COMM_ERROR",
    5: "TIMEOUT",
    6: "UNSUPPORTED",
    7: "BAD_ARG",
}


class EvkcuError(RuntimeError):
    def __init__(self, op: str, status: int, msg: str):
        super().__init__(f"{op} failed: {STATUS.get(status, status)}: {msg}")
        self.status = status


_u32, _u64, _f32, _int, _vp = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float, ctypes.c_int, ctypes.c_void_p

# name -> argtypes (all return int status unless listed in _RET)
SIGNATURES = {
    "evkcu_init": [_int],
    "evkcu_shutdown": [],
    "evkcu_last_error": [],
    "evkcu_version": [],
    "evkcu_check_device_error": [],
    "evkcu_launch_count": [],
    "evkcu_reset_launch_count": [],
    "evkcu_matmul": [_vp, _vp, _vp, _u32, _u32, _u32, _u32, _u64, _u64, _u64, _u32, _int, _vp],
    "evkcu_flash_attention": [_vp, _vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _f32, _u32, _int, _vp],
    "evkcu_single_query_attention": [_vp, _vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _u32, _f32, _int, _vp],
    "evkcu_rms_norm": [_vp, _vp, _vp, _u32, _u32, _f32, _int, _vp],
    "evkcu_rope": [_vp, _vp, _u32, _u32, _u32, _u32, _u32, _f32, _int, _vp],
    "evkcu_gelu": [_vp, _vp, _u64, _int, _vp],
    "evkcu_softmax": [_vp, _vp, _u32, _u32, _f32, _int, _vp],
    "evkcu_add": [_vp, _vp, _vp, _u64, _int, _vp],
    "evkcu_scale": [_vp, _u64, _f32, _int, _vp],
    "evkcu_zero": [_vp, _u64, _int, _vp],
    "evkcu_causal_mask": [_vp, _u32, _u32, _int, _vp],
    "evkcu_embed": [_vp, _vp, _vp, _u32, _u32, _u32, _u32, _int, _vp],
    "evkcu_greedy_sample": [_vp, _vp, _u32, _u32, _u32, _u32, _u32, _u32, _u32, _int, _vp],
    "evkcu_greedy_sample_noalloc": [_vp, _vp, _u32, _u32, _u32, _u32, _u32, _u32, _u32, _int, _vp],
    "evkcu_rms_norm_rope": [_vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _f32, _f32, _int, _vp],
    # training side
    "evkcu_relu": [_vp, _vp, _u64, _int, _vp],
    "evkcu_relu_backward": [_vp, _vp, _vp, _u64, _int, _vp],
    "evkcu_gelu_backward": [_vp, _vp, _vp, _u64, _int, _vp],
    "evkcu_softmax_backward": [_vp, _vp, _vp, _u32, _u32, _f32, _int, _vp],
    "evkcu_rms_norm_backward": [_vp, _vp, _vp, _u32, _u32, _f32, _int, _vp],
    "evkcu_rope_backward": [_vp, _vp, _u32, _u32, _u32, _f32, _int, _vp],
    "evkcu_embed_backward": [_vp, _vp, _vp, _u32, _u32, _u32, _u32, _int, _vp],
    "evkcu_position_add": [_vp, _vp, _vp, _u32, _u32, _u32, _int, _vp],
    "evkcu_position_add_backward": [_vp, _vp, _vp, _u32, _u32, _u32, _int, _vp],
    "evkcu_sum_batch": [_vp, _vp, _u32, _u64, _int, _vp],
    "evkcu_sgd": [_vp, _vp, _u64, _f32, _int, _vp],
    "evkcu_adam": [_vp, _vp, _vp, _vp, _u64, _u32, _f32, _f32, _f32, _f32, _int, _vp],
    "evkcu_mse_loss": [_vp, _vp, _vp, _vp, _u64, _int, _vp],
    "evkcu_cross_entropy_loss": [_vp, _vp, _vp, _vp, _u32, _u32, _u32, _int, _vp],
    "evkcu_flash_attention_bwd": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _f32, _u32,
                                  _int, _vp],
}
_RET = {
    "evkcu_last_error": ctypes.c_char_p,
    "evkcu_version": ctypes.c_char_p,
    "evkcu_launch_count": ctypes.c_uint64,
    "evkcu_reset_launch_count": None,
}


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    """Loads libevkcu.so and declares every C-ABI entry point."""
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `make -C evk_b200` (or __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    for name, args in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = _RET.get(name, ctypes.c_int)
    return lib


_lib: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def _check(op: str, status: int) -> None:
    if status != 0:
        raise EvkcuError(op, status, lib().evkcu_last_error().decode())


_torch = None


def _get_torch():
    """torch, imported on first use (an import statement in every call costs
    more than a look at a global)."""
    global _torch
    if _torch is None:
        import torch

        _torch = torch
    return _torch


def _dtype_code(t) -> int:
    torch = _torch or _get_torch()
    if t.dtype is torch.float16:
        return F16
    if t.dtype is torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {t.dtype}: evk tensors are 2-byte fp16 (or bf16)")


def _ptr(t) -> int:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("evk_b200 ops take CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("evk_b200 ops take contiguous (row-major) tensors")
    return t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        # the raw handle, without building a Stream object (3 us a call)
        torch = _torch or _get_torch()
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    return getattr(stream, "cuda_stream", stream)


def init(device: int = -1) -> None:
    _check("evkcu_init", lib().evkcu_init(device))


def launch_count() -> int:
    return int(lib().evkcu_launch_count())


def reset_launch_count() -> None:
    lib().evkcu_reset_launch_count()


def check_device_error() -> None:
    _check("evkcu_check_device_error", lib().evkcu_check_device_error())


# ------------------------------------------------------------------ operators
def matmul(a, b, c, transpose_a=False, transpose_b=False, acc_c=False, stream=None):
    """evk::ai::matmul (evk_ai.cpp:254-330): c = op(a) @ op(b) (+ c).

    Shapes follow the reference: (..., M, K) x (..., K, N) -> (..., M, N); an
    operand whose leading dims multiply to 1 is broadcast over the batch.
    """
    def lead(t):
        n = 1
        for d in t.shape[:-2]:
            n *= d
        return n

    ba, bb, bc = lead(a), lead(b), lead(c)
    batch = max(ba, bb, bc)
    M = a.shape[-1] if transpose_a else a.shape[-2]
    K = a.shape[-2] if transpose_a else a.shape[-1]
    N = b.shape[-2] if transpose_b else b.shape[-1]
    Kb = b.shape[-1] if transpose_b else b.shape[-2]
    if Kb != K or c.shape[-2] != M or c.shape[-1] != N or bc != batch or ba not in (1, batch) or bb not in (1, batch):
        raise EvkcuError("matmul", 1, f"incompatible shapes {tuple(a.shape)} {tuple(b.shape)} {tuple(c.shape)}")
    ea, eb, ec = a.shape[-2] * a.shape[-1], b.shape[-2] * b.shape[-1], c.shape[-2] * c.shape[-1]
    sa = 0 if (ba == 1 and batch > 1) else ea
    sb = 0 if (bb == 1 and batch > 1) else eb
    flags = (MM_TRANSPOSE_A if transpose_a else 0) | (MM_TRANSPOSE_B if transpose_b else 0) | (MM_ACC_C if acc_c else 0)
    _check("evkcu_matmul", lib().evkcu_matmul(_ptr(a), _ptr(b), _ptr(c), batch, M, K, N, sa, sb, ec, flags,
                                              _dtype_code(a), _stream(stream)))
    return c


def flash_attention(q, k, v, o, heads: Optional[int] = None, causal=False, scale: float = 0.0, stream=None):
    """evk::ai::flash_attention (evk_ai.cpp:332-369) plus extensions.

    q, o: (B, N, H*Dh); k, v: (B, N, Hkv*Dh).  Without `heads` the reference's
    multi-query call is assumed (Hkv = 1, Dh = k.shape[-1]).  `heads` gives H
    (Dh = q.shape[-1] // H, Hkv = k.shape[-1] // Dh).
    """
    B, N, D = q.shape
    if heads is None:
        Dh = k.shape[-1]
        H, Hkv = D // Dh, 1
    else:
        H = heads
        Dh = D // H
        Hkv = k.shape[-1] // Dh
    _check("evkcu_flash_attention", lib().evkcu_flash_attention(
        _ptr(q), _ptr(k), _ptr(v), _ptr(o), B, N, H, Hkv, Dh, scale, ATTN_CAUSAL if causal else 0,
        _dtype_code(q), _stream(stream)))
    return o


def single_query_attention(q, kcache, vcache, out, heads: int, cur_len: int, scale: float = 0.0, stream=None):
    """Decode attention over a KV cache (shaders/single_query_attention.comp).

    q, out: (B, H*Dh); kcache, vcache: (B, max_len, Hkv*Dh).
    """
    B = q.shape[0]
    Dh = q.shape[-1] // heads
    max_len = kcache.shape[1]
    Hkv = kcache.shape[-1] // Dh
    _check("evkcu_single_query_attention", lib().evkcu_single_query_attention(
        _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(out), B, heads, Hkv, Dh, max_len, cur_len, scale,
        _dtype_code(q), _stream(stream)))
    return out


def rms_norm(x, out, eps=1e-4, gamma=None, stream=None):
    D = x.shape[-1]
    _check("evkcu_rms_norm", lib().evkcu_rms_norm(_ptr(x), _ptr(out), _ptr(gamma), x.numel() // D, D, eps,
                                                  _dtype_code(x), _stream(stream)))
    return out


def rope(x, out, batch, seq_len, dim, base=10000.0, head_dim=0, pos_offset=0, stream=None):
    _check("evkcu_rope", lib().evkcu_rope(_ptr(x), _ptr(out), batch, seq_len, dim, head_dim, pos_offset, base,
                                          _dtype_code(x), _stream(stream)))
    return out


def rms_norm_rope(x, out, seq_len, eps=1e-5, base=10000.0, head_dim=0, pos_offset=0, gamma=None, stream=None):
    """Fused rms_norm + rope over rows of the last dimension (evkcu_rms_norm_rope)."""
    D = x.shape[-1]
    _check("evkcu_rms_norm_rope", lib().evkcu_rms_norm_rope(
        _ptr(x), _ptr(out), _ptr(gamma), x.numel() // D, seq_len, D, head_dim, pos_offset, eps, base,
        _dtype_code(x), _stream(stream)))
    return out


def gelu(x, out, stream=None):
    _check("evkcu_gelu", lib().evkcu_gelu(_ptr(x), _ptr(out), x.numel(), _dtype_code(x), _stream(stream)))
    return out


def softmax(x, out, scale=1.0, stream=None):
    L = x.shape[-1]
    _check("evkcu_softmax", lib().evkcu_softmax(_ptr(x), _ptr(out), x.numel() // L, L, scale, _dtype_code(x),
                                                _stream(stream)))
    return out


def add(a, b, c, stream=None):
    _check("evkcu_add", lib().evkcu_add(_ptr(a), _ptr(b), _ptr(c), a.numel(), _dtype_code(a), _stream(stream)))
    return c


def scale(x, s, stream=None):
    _check("evkcu_scale", lib().evkcu_scale(_ptr(x), x.numel(), s, _dtype_code(x), _stream(stream)))
    return x


def zero(x, stream=None):
    _check("evkcu_zero", lib().evkcu_zero(_ptr(x), x.numel(), _dtype_code(x), _stream(stream)))
    return x


def apply_causal_mask(s, stream=None):
    N = s.shape[-1]
    _check("evkcu_causal_mask", lib().evkcu_causal_mask(_ptr(s), s.numel() // (N * N), N, _dtype_code(s),
                                                        _stream(stream)))
    return s


def embed(E, idx, out, stream=None):
    """idx: int16/uint16 (reference) or int32 ids, any shape."""
    import torch

    ib = 2 if idx.element_size() == 2 else 4
    _check("evkcu_embed", lib().evkcu_embed(_ptr(E), _ptr(idx), _ptr(out), E.shape[0], E.shape[1], idx.numel(), ib,
                                            _dtype_code(E), _stream(stream)))
    return out


def greedy_sample(logits, out, position, token_base, token_count, stream=None):
    """logits (B, S, V); out (B,) int16/uint16 (reference) or int32 ids."""
    B, S, V = logits.shape
    ob = 2 if out.element_size() == 2 else 4
    _check("evkcu_greedy_sample", lib().evkcu_greedy_sample(
        _ptr(logits), _ptr(out), B, S, V, position, token_base, token_count, ob, _dtype_code(logits),
        _stream(stream)))
    return out


# ------------------------------------------------------------ training side --
def relu(x, out, stream=None):
    _check("evkcu_relu", lib().evkcu_relu(_ptr(x), _ptr(out), x.numel(), _dtype_code(x), _stream(stream)))
    return out


def relu_backward(grad_out, x, grad_in, stream=None):
    _check("evkcu_relu_backward", lib().evkcu_relu_backward(_ptr(grad_out), _ptr(x), _ptr(grad_in), x.numel(),
                                                            _dtype_code(x), _stream(stream)))
    return grad_in


def gelu_backward(grad_out, x, grad_in, stream=None):
    _check("evkcu_gelu_backward", lib().evkcu_gelu_backward(_ptr(grad_out), _ptr(x), _ptr(grad_in), x.numel(),
                                                            _dtype_code(x), _stream(stream)))
    return grad_in


def softmax_backward(probs, grad_out, grad_in, scale=1.0, stream=None):
    L = probs.shape[-1]
    _check("evkcu_softmax_backward", lib().evkcu_softmax_backward(
        _ptr(probs), _ptr(grad_out), _ptr(grad_in), probs.numel() // L, L, scale, _dtype_code(probs),
        _stream(stream)))
    return grad_in


def rms_norm_backward(x, grad_out, grad_in, eps=1e-4, stream=None):
    D = x.shape[-1]
    _check("evkcu_rms_norm_backward", lib().evkcu_rms_norm_backward(
        _ptr(x), _ptr(grad_out), _ptr(grad_in), x.numel() // D, D, eps, _dtype_code(x), _stream(stream)))
    return grad_in


def rope_backward(grad_out, grad_in, batch, seq_len, dim, base=10000.0, stream=None):
    _check("evkcu_rope_backward", lib().evkcu_rope_backward(_ptr(grad_out), _ptr(grad_in), batch, seq_len, dim,
                                                            base, _dtype_code(grad_out), _stream(stream)))
    return grad_in


def embed_backward(grad_out, idx, grad_E, stream=None):
    ib = 2 if idx.element_size() == 2 else 4
    _check("evkcu_embed_backward", lib().evkcu_embed_backward(
        _ptr(grad_out), _ptr(idx), _ptr(grad_E), grad_E.shape[0], grad_E.shape[1], idx.numel(), ib,
        _dtype_code(grad_E), _stream(stream)))
    return grad_E


def position_add(x, pos, out, batch, seq_len, dim, stream=None):
    _check("evkcu_position_add", lib().evkcu_position_add(_ptr(x), _ptr(pos), _ptr(out), batch, seq_len, dim,
                                                          _dtype_code(x), _stream(stream)))
    return out


def position_add_backward(grad_out, grad_in, grad_pos, batch, seq_len, dim, stream=None):
    _check("evkcu_position_add_backward", lib().evkcu_position_add_backward(
        _ptr(grad_out), _ptr(grad_in), _ptr(grad_pos), batch, seq_len, dim, _dtype_code(grad_out),
        _stream(stream)))
    return grad_in, grad_pos


def sum_batch(x, out, batch, size, stream=None):
    _check("evkcu_sum_batch", lib().evkcu_sum_batch(_ptr(x), _ptr(out), batch, size, _dtype_code(x),
                                                    _stream(stream)))
    return out


def sgd(param, grad, lr, stream=None):
    _check("evkcu_sgd", lib().evkcu_sgd(_ptr(param), _ptr(grad), param.numel(), lr, _dtype_code(param),
                                        _stream(stream)))
    return param


def adam(param, grad, m, v, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-4, stream=None):
    """m, v: the AdamState buffers (zero-initialised, same dtype/size as param);
    step: the state's timestep after increment (1 on the first call)."""
    _check("evkcu_adam", lib().evkcu_adam(_ptr(param), _ptr(grad), _ptr(m), _ptr(v), param.numel(), step, lr, beta1,
                                          beta2, eps, _dtype_code(param), _stream(stream)))
    return param


def mse_loss(pred, target, grad, result, stream=None):
    _check("evkcu_mse_loss", lib().evkcu_mse_loss(_ptr(pred), _ptr(target), _ptr(grad), _ptr(result), pred.numel(),
                                                  _dtype_code(pred), _stream(stream)))
    return result


def cross_entropy_loss(logits, targets, grad, result, stream=None):
    """logits (rows, V); targets (rows,) int16/uint16 (reference) or int32."""
    V = logits.shape[-1]
    tb = 2 if targets.element_size() == 2 else 4
    _check("evkcu_cross_entropy_loss", lib().evkcu_cross_entropy_loss(
        _ptr(logits), _ptr(targets), _ptr(grad), _ptr(result), logits.numel() // V, V, tb, _dtype_code(logits),
        _stream(stream)))
    return result


def flash_attention_bwd(q, k, v, o, dO, dQ, dK, dV, heads: Optional[int] = None, causal=False, normalized=False,
                        scale: float = 0.0, stream=None):
    """Gradients of flash_attention (evk_ai.cpp:371-473).  Layouts as
    flash_attention; without `heads` the reference's multi-query call."""
    B, N, D = q.shape
    if heads is None:
        Dh = k.shape[-1]
        H, Hkv = D // Dh, 1
    else:
        H = heads
        Dh = D // H
        Hkv = k.shape[-1] // Dh
    flags = (ATTN_CAUSAL if causal else 0) | (ATTN_BWD_NORMALIZED if normalized else 0)
    _check("evkcu_flash_attention_bwd", lib().evkcu_flash_attention_bwd(
        _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(dO), _ptr(dQ), _ptr(dK), _ptr(dV), B, N, H, Hkv, Dh, scale, flags,
        _dtype_code(q), _stream(stream)))
    return dQ, dK, dV


# ------------------------------------- decoder-layer operators (extension) --
class QkNormRopeDesc(ctypes.Structure):
    """evkcu_qk_norm_rope_desc (include/evkcu.h)."""

    _fields_ = [(n, ctypes.c_uint32) for n in ("batch", "seq_len", "heads", "kv_heads", "head_dim", "rot_dim", "flags",
                                                "pos_offset", "cache_len")] + \
               [("eps", ctypes.c_float), ("base", ctypes.c_float), ("positions", ctypes.c_void_p)] + \
               [(n, ctypes.c_uint64) for n in ("q_pitch", "k_pitch", "v_pitch", "q_out_pitch", "k_out_pitch",
                                                "dq_pitch", "dk_pitch")]


SIGNATURES.update({
    "evkcu_linear": [_vp] * 6 + [_u32, _u32, _u32, _int, _u32, _int, _vp],
    "evkcu_linear_backward": [_vp] * 8 + [_u32, _u32, _u32, _int, _u32, _int, _vp],
    "evkcu_gated_ffn": [_vp] * 7 + [_u32, _u32, _u32, _int, _u32, _int, _vp],
    "evkcu_gated_ffn_backward": [_vp] * 10 + [_u32, _u32, _u32, _int, _u32, _int, _vp],
    "evkcu_qk_norm_rope": [ctypes.POINTER(QkNormRopeDesc)] + [_vp] * 8 + [_int, _vp],
    "evkcu_qk_norm_rope_backward": [ctypes.POINTER(QkNormRopeDesc)] + [_vp] * 11 + [_u64, _int, _vp],
    "evkcu_qk_norm_rope_workspace": [_u32],
})
_RET["evkcu_qk_norm_rope_workspace"] = _u64


def _same(op, like, want):
    """Checks (name, tensor or None, shape) triples against `like`'s dtype and
    device, which has to be the current one."""
    dt, dev = like.dtype, like.get_device()
    for name, t, shape in want:
        if t is None:
            continue
        if t.dtype is not dt or t.get_device() != dev:
            raise EvkcuError(op, 7, f"{name} is {t.dtype} on {t.device}, expected {dt} on {like.device}")
        if t.shape != shape:
            raise EvkcuError(op, 1, f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if dev < 0:
        raise ValueError("evk_b200 ops take CUDA tensors")
    torch = _torch or _get_torch()
    if dev != torch.cuda.current_device():
        raise EvkcuError(op, 7, f"tensors are on cuda:{dev}, the current device is "
                                f"cuda:{torch.cuda.current_device()}")


def _same_ptrs(op, like, want):
    """_same, and the pointers of the tensors (None for none), which have to be
    contiguous."""
    _same(op, like, want)
    out = []
    for name, t, _ in want:
        if t is None:
            out.append(None)
        elif t.is_contiguous():
            out.append(t.data_ptr())
        else:
            raise ValueError(f"evk_b200 ops take contiguous (row-major) tensors: {name}")
    return out


def _missing(op, **tensors):
    """The error of a call that lacks one of these tensors, from which the
    binding takes shapes and strides (the C ABI checks the others)."""
    names = ", ".join(n for n, t in tensors.items() if t is None)
    return EvkcuError(op, 7, f"{names} must be given")


def _row_count(op, x, a, b):
    """Rows of x's last dimension a.  The C ABI takes 32-bit sizes, and ctypes
    would cut larger ones to their low bits."""
    rows = x.numel() // a if a else 0
    if (rows | a | b) >> 32:
        raise EvkcuError(op, 1, f"{rows} rows of {a} and {b} columns: sizes above 2^32 - 1")
    return rows


def linear(x, w, y, bias=None, residual=None, act=ACT_NONE, pre=None, transpose_w=False, stream=None):
    """y = act(x @ w + bias) + residual (evkcu_linear).

    x (..., K); w (K, N), or (N, K) with transpose_w; bias (N,); residual, y
    and pre (..., N), pre receiving x @ w + bias for linear_backward.  residual
    may be y."""
    if x is None or y is None:
        raise _missing("linear", x=x, y=y)
    *lead, K = x.shape
    N = y.shape[-1]
    out = (*lead, N)
    rows = _row_count("linear", x, K, N)
    p = _same_ptrs("linear", x, (("x", x, x.shape), ("w", w, (N, K) if transpose_w else (K, N)), ("bias", bias, (N,)),
                                 ("residual", residual, out), ("y", y, out), ("pre", pre, out)))
    _check("evkcu_linear", lib().evkcu_linear(
        *p, rows, K, N, act, MM_TRANSPOSE_B if transpose_w else 0, _dtype_code(x),
        _stream(stream)))
    return y


def linear_backward(x, w, dy, dx=None, dw=None, dbias=None, act=ACT_NONE, pre=None, dpre=None, transpose_w=False,
                    acc=False, stream=None):
    """Gradients of linear from dy (evkcu_linear_backward) into those of dx, dw
    and dbias that are given; acc adds to them.  With an activation, pre is
    linear's and dpre (like pre; pre or dy itself is allowed) receives the
    gradient of x @ w + bias."""
    if x is None or dy is None:
        raise _missing("linear_backward", x=x, dy=dy)
    K, N = x.shape[-1], dy.shape[-1]
    out = (*x.shape[:-1], N)
    wshape = (N, K) if transpose_w else (K, N)
    rows = _row_count("linear_backward", x, K, N)
    p = _same_ptrs("linear_backward", x, (("x", x, x.shape), ("w", w, wshape), ("pre", pre, out), ("dy", dy, out),
                                          ("dpre", dpre, out), ("dx", dx, x.shape), ("dw", dw, wshape),
                                          ("dbias", dbias, (N,))))
    flags = (MM_TRANSPOSE_B if transpose_w else 0) | (MM_ACC_C if acc else 0)
    _check("evkcu_linear_backward", lib().evkcu_linear_backward(
        *p, rows, K, N, act, flags, _dtype_code(x), _stream(stream)))
    return dx, dw, dbias


def gated_ffn(x, w_in, w_out, y, hidden, act=ACT_SILU, residual=None, pre=None, transpose_w=False, stream=None):
    """Gated feed-forward block (evkcu_gated_ffn): with [g | u] = x @ w_in,
    hidden = act(g) * u and y = hidden @ w_out + residual.

    x, y, residual (..., D); w_in (D, 2 F), w_out (F, D), or both transposed
    with transpose_w; hidden (..., F); pre (..., 2 F) receives [g | u] for
    gated_ffn_backward.  y = None (then w_out may be None) stops at hidden."""
    if x is None or hidden is None:
        raise _missing("gated_ffn", x=x, hidden=hidden)
    D, F = x.shape[-1], hidden.shape[-1]
    lead = x.shape[:-1]
    rows = _row_count("gated_ffn", x, D, F)
    p = _same_ptrs("gated_ffn", x, (("x", x, x.shape), ("w_in", w_in, (2 * F, D) if transpose_w else (D, 2 * F)),
                                    ("w_out", w_out, (D, F) if transpose_w else (F, D)),
                                    ("residual", residual, x.shape), ("y", y, x.shape), ("hidden", hidden, (*lead, F)),
                                    ("pre", pre, (*lead, 2 * F))))
    _check("evkcu_gated_ffn", lib().evkcu_gated_ffn(
        *p, rows, D, F, act, MM_TRANSPOSE_B if transpose_w else 0, _dtype_code(x),
        _stream(stream)))
    return y if y is not None else hidden


def gated_ffn_backward(x, w_in, w_out, pre, dy, dpre, hidden, dx=None, dw_in=None, dw_out=None, act=ACT_SILU,
                       transpose_w=False, acc=False, stream=None):
    """Gradients of gated_ffn from dy (evkcu_gated_ffn_backward) into those of
    dx, dw_in and dw_out that are given; acc adds to them.  pre is gated_ffn's;
    dpre (like pre; pre itself is allowed) receives its gradient; hidden
    (..., F) is recomputed and needed only for dw_out."""
    if x is None or pre is None:
        raise _missing("gated_ffn_backward", x=x, pre=pre)
    D, F = x.shape[-1], pre.shape[-1] // 2
    lead = x.shape[:-1]
    rows = _row_count("gated_ffn_backward", x, D, F)
    si, so = ((2 * F, D), (D, F)) if transpose_w else ((D, 2 * F), (F, D))
    p = _same_ptrs("gated_ffn_backward", x, (("x", x, x.shape), ("w_in", w_in, si), ("w_out", w_out, so),
                                             ("pre", pre, (*lead, 2 * F)), ("dy", dy, x.shape),
                                             ("dpre", dpre, (*lead, 2 * F)), ("hidden", hidden, (*lead, F)),
                                             ("dx", dx, x.shape), ("dw_in", dw_in, si), ("dw_out", dw_out, so)))
    flags = (MM_TRANSPOSE_B if transpose_w else 0) | (MM_ACC_C if acc else 0)
    _check("evkcu_gated_ffn_backward", lib().evkcu_gated_ffn_backward(
        *p, rows, D, F, act, flags, _dtype_code(x), _stream(stream)))
    return dx, dw_in, dw_out


def _rows(op, name, t, B, S):
    """(pointer, row pitch) of a (B, S, cols) tensor whose rows are evenly
    spaced (a slice of the last dimension of a contiguous tensor is)."""
    sb, st, sc = t.stride()
    if (sc != 1 and t.shape[2] > 1) or (B > 1 and S > 1 and sb != S * st):
        raise EvkcuError(op, 1, f"{name}: strides {t.stride()} are not evenly spaced rows")
    return t.data_ptr(), st if S > 1 else sb if B > 1 else max(t.shape[2], 1)


def _qk_shape(op, q, k, heads, positions, rot_dim, pos_offset):
    """(B, S, head_dim, key columns, positions pointer) from q and k."""
    if q.dim() != 3 or heads <= 0 or q.shape[2] % heads:
        raise EvkcuError(op, 1, f"q is {tuple(q.shape)}, expected (B, S, {heads} heads * head_dim)")
    B, S, cols = q.shape
    dh = cols // heads
    kc = 0
    if k is not None:
        if dh == 0 or k.dim() != 3 or k.shape[2] % dh:
            raise EvkcuError(op, 1, f"k is {tuple(k.shape)}, expected (B, S, kv_heads * {dh})")
        kc = k.shape[2]
    if (B | S | cols | kc) >> 32:  # as in _row_count
        raise EvkcuError(op, 1, f"q is {tuple(q.shape)}, with {kc} columns of keys: sizes above 2^32 - 1")
    pos = None
    if positions is not None:
        torch = _torch or _get_torch()
        if positions.dtype is not torch.int32 or positions.numel() != B * S or positions.get_device() != q.get_device():
            raise EvkcuError(op, 1, f"positions must be {B * S} int32 values on {q.device}")
        pos = _ptr(positions)
    if not 0 <= rot_dim <= 0xFFFFFFFF or not 0 <= pos_offset <= 0xFFFFFFFF:
        raise EvkcuError(op, 1, "rot_dim and pos_offset must be non-negative")
    return B, S, dh, kc, pos


def qk_norm_rope(q, k, q_out, k_out, heads: int, gain_q=None, gain_k=None, v=None, v_out=None, cache=False,
                 positions=None, rot_dim=0, half_split=False, eps=1e-5, base=10000.0, pos_offset=0, stream=None):
    """Per-head RMSNorm and rotation of queries and keys in one pass
    (evkcu_qk_norm_rope).

    q, q_out (B, S, heads * Dh); k, k_out (B, S, Hkv * Dh), or None for queries
    only; rows may be slices of a fused QKV tensor.  gain_q, gain_k (Dh,).
    rot_dim: the rotated part of a head, even, 0 for all of it; pairs are
    (2 i, 2 i + 1), or (i, i + rot_dim / 2) with half_split, where the rotated
    part (Dh, if rot_dim is 0) has to be a multiple of 16.  positions: B * S
    int32 values, else pos_offset + t.  With cache=True, k_out is a contiguous
    KV cache (B, cache_len, Hkv * Dh) and keys go to the rows of their
    positions.  v, where given, is copied along to v_out, which is laid out as
    k_out."""
    op = "qk_norm_rope"
    if q is None or q_out is None or (k is not None and k_out is None):
        raise _missing(op, q=q, q_out=q_out, **(dict(k_out=k_out) if k is not None else {}))
    B, S, dh, kc, pos = _qk_shape(op, q, k, heads, positions, rot_dim, pos_offset)
    cache_len = 0
    if k is None:
        if v is not None or v_out is not None or cache:
            raise EvkcuError(op, 7, "v, v_out and cache need k")
    elif cache:
        if k_out.dim() != 3:
            raise EvkcuError(op, 1, f"k_out is {tuple(k_out.shape)}, expected (B, cache_len, {kc})")
        cache_len = k_out.shape[1]
        if cache_len >> 32:
            raise EvkcuError(op, 1, f"a cache of {cache_len} rows: sizes above 2^32 - 1")
    ks = (B, S, kc)
    os = (B, cache_len, kc) if cache else ks
    _same(op, q, (("q_out", q_out, q.shape), ("gain_q", gain_q, (dh,)), ("gain_k", gain_k, (dh,)), ("k", k, ks),
                  ("k_out", k_out if k is not None else None, os), ("v", v, ks), ("v_out", v_out, os)))
    qp, q_pitch = _rows(op, "q", q, B, S)
    qo, qo_pitch = _rows(op, "q_out", q_out, B, S)
    kp = ko = vp = vo = None
    k_pitch = ko_pitch = v_pitch = 0
    if k is not None:
        kp, k_pitch = _rows(op, "k", k, B, S)
        if cache:
            ko, vo, ko_pitch = _ptr(k_out), _ptr(v_out), kc
        else:
            ko, ko_pitch = _rows(op, "k_out", k_out, B, S)
            if v_out is not None:
                vo, vo_pitch = _rows(op, "v_out", v_out, B, S)
                if vo_pitch != ko_pitch:
                    raise EvkcuError(op, 1, "v_out must have the row pitch of k_out")
        if v is not None:
            vp, v_pitch = _rows(op, "v", v, B, S)
    d = QkNormRopeDesc(B, S, heads, kc // dh if kc else 0, dh, rot_dim,
                       (QK_HALF_SPLIT if half_split else 0) | (QK_CACHE if cache else 0), pos_offset, cache_len, eps,
                       base, pos, q_pitch, k_pitch, v_pitch, qo_pitch, ko_pitch)
    _check("evkcu_qk_norm_rope", lib().evkcu_qk_norm_rope(
        d, qp, kp, vp, _ptr(gain_q), _ptr(gain_k), qo, ko, vo, _dtype_code(q), _stream(stream)))
    return q_out, k_out


def qk_norm_rope_workspace(head_dim: int) -> int:
    """Bytes of workspace that qk_norm_rope_backward needs for gain gradients."""
    return int(lib().evkcu_qk_norm_rope_workspace(head_dim))


def qk_norm_rope_backward(q, k, dq_out, dk_out, dq, dk, heads: int, gain_q=None, gain_k=None, dgain_q=None,
                          dgain_k=None, workspace=None, positions=None, rot_dim=0, half_split=False, eps=1e-5,
                          base=10000.0, pos_offset=0, acc_gain=False, stream=None):
    """Gradients of qk_norm_rope (evkcu_qk_norm_rope_backward): from those of
    its outputs and its saved inputs q, k into dq, dk (dq may be dq_out, dk may
    be dk_out) and, where given, dgain_q, dgain_k (Dh,), which need a
    `workspace` tensor of qk_norm_rope_workspace(Dh) bytes and are added to with
    acc_gain."""
    op = "qk_norm_rope_backward"
    if q is None or dq_out is None or dq is None or (k is not None and (dk_out is None or dk is None)):
        raise _missing(op, q=q, dq_out=dq_out, dq=dq, **(dict(dk_out=dk_out, dk=dk) if k is not None else {}))
    B, S, dh, kc, pos = _qk_shape(op, q, k, heads, positions, rot_dim, pos_offset)
    ks = (B, S, kc)
    if k is None:
        dk_out = dk = None
    _same(op, q, (("dq_out", dq_out, q.shape), ("dq", dq, q.shape), ("gain_q", gain_q, (dh,)),
                  ("gain_k", gain_k, (dh,)), ("dgain_q", dgain_q, (dh,)), ("dgain_k", dgain_k, (dh,)), ("k", k, ks),
                  ("dk_out", dk_out, ks), ("dk", dk, ks)))
    qp, q_pitch = _rows(op, "q", q, B, S)
    gq, gq_pitch = _rows(op, "dq_out", dq_out, B, S)
    dqp, dq_pitch = _rows(op, "dq", dq, B, S)
    kp = gk = dkp = None
    k_pitch = gk_pitch = dk_pitch = 0
    if k is not None:
        kp, k_pitch = _rows(op, "k", k, B, S)
        gk, gk_pitch = _rows(op, "dk_out", dk_out, B, S)
        dkp, dk_pitch = _rows(op, "dk", dk, B, S)
    wbytes = 0
    if workspace is not None:
        if workspace.get_device() != q.get_device():
            raise EvkcuError(op, 7, f"workspace is on {workspace.device}, expected {q.device}")
        wbytes = workspace.numel() * workspace.element_size()
    d = QkNormRopeDesc(B, S, heads, kc // dh if kc else 0, dh, rot_dim,
                       (QK_HALF_SPLIT if half_split else 0) | (QK_ACC_GAIN if acc_gain else 0), pos_offset, 0, eps,
                       base, pos, q_pitch, k_pitch, 0, gq_pitch, gk_pitch, dq_pitch, dk_pitch)
    _check("evkcu_qk_norm_rope_backward", lib().evkcu_qk_norm_rope_backward(
        d, qp, kp, _ptr(gain_q), _ptr(gain_k), gq, gk, dqp, dkp, _ptr(dgain_q), _ptr(dgain_k), _ptr(workspace), wbytes,
        _dtype_code(q), _stream(stream)))
    return dq, dk


# ------------------------------------------------------------- LLM driver --
class LlmConfig(ctypes.Structure):
    """evkcu_llm_config (include/evkcu.h)."""

    _fields_ = [(n, ctypes.c_uint32) for n in ("layers", "d_model", "heads", "kv_heads", "hidden", "vocab",
                                                "max_batch", "max_seq")] + \
               [("rope_base", ctypes.c_float), ("eps", ctypes.c_float), ("dtype", ctypes.c_int),
                ("tied_embeddings", ctypes.c_uint32), ("tp_rank", ctypes.c_uint32), ("tp_size", ctypes.c_uint32)]


_pp = ctypes.POINTER(ctypes.c_void_p)
SIGNATURES.update({
    "evkcu_single_query_attention_devlen": [_vp, _vp, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _vp, _f32, _int, _vp],
    "evkcu_comm_unique_id": [_vp],
    "evkcu_comm_init": [_vp, _int, _int, _pp],
    "evkcu_comm_destroy": [_vp],
    "evkcu_llm_create": [ctypes.POINTER(LlmConfig), _vp, _pp],
    "evkcu_llm_destroy": [_vp],
    "evkcu_llm_init_random": [_vp, _u64, _f32, _vp],
    "evkcu_llm_set_weight": [_vp, ctypes.c_char_p, _u32, _vp, _vp],
    "evkcu_llm_prefill": [_vp, _vp, _u32, _u32, _vp, _vp, _vp],
    "evkcu_llm_decode": [_vp, _vp, _vp, _vp, _vp],
    "evkcu_llm_length": [_vp],
    "evkcu_llm_fused_allreduce": [_vp],
    "evkcu_llm_load": [_vp, ctypes.c_char_p, _vp],
    "evkcu_llm_save": [_vp, ctypes.c_char_p, _vp],
})
_RET["evkcu_llm_length"] = ctypes.c_uint32
_RET["evkcu_llm_fused_allreduce"] = ctypes.c_uint32


class Comm:
    """NCCL communicator for tensor parallelism (one process per GPU)."""

    def __init__(self, unique_id: bytes, rank: int, world: int):
        self.handle = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(unique_id, 128)
        _check("evkcu_comm_init", lib().evkcu_comm_init(buf, rank, world, ctypes.byref(self.handle)))

    @staticmethod
    def unique_id() -> bytes:
        buf = ctypes.create_string_buffer(128)
        _check("evkcu_comm_unique_id", lib().evkcu_comm_unique_id(buf))
        return buf.raw

    def close(self):
        if self.handle:
            _check("evkcu_comm_destroy", lib().evkcu_comm_destroy(self.handle))
            self.handle = ctypes.c_void_p()


class Llm:
    """Device-resident decoder (evkcu_llm_*): prefill, CUDA-graph decode,
    optional tensor parallelism.  Token ids are int32 CUDA tensors."""

    def __init__(self, layers, d_model, heads, hidden, vocab, max_batch, max_seq, kv_heads=None, rope_base=10000.0,
                 eps=1e-5, dtype=F16, tied_embeddings=True, tp_rank=0, tp_size=1, comm: Optional[Comm] = None):
        self.cfg = LlmConfig(layers, d_model, heads, kv_heads or heads, hidden, vocab, max_batch, max_seq, rope_base,
                             eps, dtype, int(tied_embeddings), tp_rank, tp_size)
        self.handle = ctypes.c_void_p()
        _check("evkcu_llm_create", lib().evkcu_llm_create(ctypes.byref(self.cfg), comm.handle if comm else None,
                                                          ctypes.byref(self.handle)))

    def close(self):
        if self.handle:
            lib().evkcu_llm_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def init_random(self, seed=42, std=0.02, stream=None):
        _check("evkcu_llm_init_random", lib().evkcu_llm_init_random(self.handle, seed, std, _stream(stream)))

    def set_weight(self, name: str, tensor, layer: int = 0, stream=None):
        _check("evkcu_llm_set_weight", lib().evkcu_llm_set_weight(self.handle, name.encode(), layer, _ptr(tensor),
                                                                  _stream(stream)))

    def load(self, path: str, stream=None):
        """Loads every weight from a weight blob (see write_weight_blob)."""
        _check("evkcu_llm_load", lib().evkcu_llm_load(self.handle, os.fsencode(path), _stream(stream)))

    def save(self, path: str, stream=None):
        """Writes every weight to a weight blob (single-GPU models)."""
        _check("evkcu_llm_save", lib().evkcu_llm_save(self.handle, os.fsencode(path), _stream(stream)))

    def prefill(self, tokens, next_ids, logits=None, stream=None):
        B, S = tokens.shape
        _check("evkcu_llm_prefill", lib().evkcu_llm_prefill(self.handle, _ptr(tokens), B, S, _ptr(next_ids),
                                                            _ptr(logits), _stream(stream)))
        return next_ids

    def decode(self, ids, next_ids, logits=None, stream=None):
        _check("evkcu_llm_decode", lib().evkcu_llm_decode(self.handle, _ptr(ids), _ptr(next_ids), _ptr(logits),
                                                          _stream(stream)))
        return next_ids

    @property
    def fused_allreduce(self) -> bool:
        """Whether decode all-reduces run fused over peer memory (tensor parallel)."""
        return bool(lib().evkcu_llm_fused_allreduce(self.handle))

    @property
    def length(self) -> int:
        return int(lib().evkcu_llm_length(self.handle))


# ------------------------------------------------------------- weight blob --
BLOB_MAGIC = b"EVKWBLOB"


def blob_layout(layers, d_model, heads, hidden, vocab, kv_heads=None, tied_embeddings=True):
    """(name, layer, shape) of every tensor of a weight blob, in file order
    (include/evkcu.h, evkcu_llm_load)."""
    kv = kv_heads or heads
    dh = d_model // heads
    out = [("embedding", 0, (vocab, d_model))]
    if not tied_embeddings:
        out.append(("lm_head", 0, (d_model, vocab)))
    for l in range(layers):
        out += [("wqkv", l, (d_model, (heads + 2 * kv) * dh)), ("wo", l, (heads * dh, d_model)),
                ("w1", l, (d_model, hidden)), ("w2", l, (hidden, d_model))]
    return out


def write_weight_blob(path, weights, layers, d_model, heads, hidden, vocab, kv_heads=None, tied_embeddings=True,
                      dtype=F16):
    """Writes a weight blob from host arrays of 2-byte storage values.

    weights maps (name, layer) to an array with the blob_layout shape (any
    2-byte dtype: numpy uint16/float16, or torch half/bfloat16 on the CPU)."""
    import numpy as np

    kv = kv_heads or heads
    header = np.zeros(16, np.uint32)
    header[:2] = np.frombuffer(BLOB_MAGIC, np.uint32)
    header[2:11] = [1, dtype, layers, d_model, heads, kv, hidden, vocab, 1 if tied_embeddings else 0]
    with open(path, "wb") as f:
        f.write(header.tobytes())
        for name, layer, shape in blob_layout(layers, d_model, heads, hidden, vocab, kv, tied_embeddings):
            a = weights[(name, layer)]
            if hasattr(a, "numpy"):
                import torch

                a = a.detach().contiguous().cpu().view(torch.int16).numpy()
            a = np.ascontiguousarray(a)
            if a.dtype.itemsize != 2 or a.size != shape[0] * shape[1]:
                raise ValueError(f"{name}[{layer}]: expected {shape} of 2-byte values, got {a.shape} {a.dtype}")
            f.write(a.view(np.uint16).tobytes())
