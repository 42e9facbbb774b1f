"""Python host driver of the operators on rows of channels (ctypes over include/fhc_seq.h in libfhconv.so): a gated
linear recurrence (``glr``), the norms around a block with its gate and the scaled residual (``norm_block``) and a
gated feed-forward block (``ffn``), each with its backward pass.

Inputs are torch tensors on the current GPU in f16, bf16 or (not ``ffn``) f32, all of one call in the same type; states
and the gradients of the recurrence's and norms' weights are f32. Each function returns new tensors. ``stream`` (a torch stream) is where the call runs,
the current stream if None; what it allocates belongs to that stream. The module only passes device pointers: when the
library is missing, loading it raises, and nothing is computed on the host.
"""
from __future__ import annotations

import contextlib
import ctypes

import fhconv
from fhconv import FhcError

F16, BF16, F32 = 0, 1, 2

_P, _U, _I64, _F, _SZ = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class FhcSeq(ctypes.Structure):
    _fields_ = [("p", _P), ("bs", _I64), ("ts", _I64)]


class GlrDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("b", _U), ("t", _U), ("d", _U), ("rate", _F), ("lam", _P), ("lengths", _P)]


class NormDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("rows", _U), ("c", _U), ("rows_per_group", _U), ("alpha", _F), ("eps", _F),
                ("w_post", _P), ("w_pre", _P), ("gate", _P)]


class FhcRows(ctypes.Structure):
    _fields_ = [("p", _P), ("ld", _I64)]


class FfnDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("act", _U), ("rows", _U), ("c", _U), ("f", _U)]


_typed = None


def _lib():
    global _typed
    if _typed is None:
        L = fhconv.load()
        G, S, N, R, D = (ctypes.POINTER(t) for t in (GlrDesc, FhcSeq, NormDesc, FhcRows, FfnDesc))
        sig = {
            "fhc_glr_states_bytes": ([G], _SZ),
            "fhc_glr_workspace_bytes": ([G, ctypes.c_int], _SZ),
            "fhc_glr_forward": ([G, S, S, S, _P, S, _P, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_glr_backward": ([G, S, S, S, _P, S, _P, S, S, S, _P, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_norm_block": ([N, R, R, R, R, _P], ctypes.c_int),
            "fhc_norm_block_workspace_bytes": ([N], _SZ),
            "fhc_norm_block_backward": ([N, R, R, R, R, R, R, _P, _P, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_ffn_saved_bytes": ([D], _SZ),
            "fhc_ffn_workspace_bytes": ([D, ctypes.c_int], _SZ),
            "fhc_ffn_forward": ([D, R, _P, _P, _P, R, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_ffn_backward": ([D, R, _P, _P, _P, _P, R, R, _P, _P, _P, _P, _SZ, _P], ctypes.c_int),
        }
        for name, (args, res) in sig.items():
            f = getattr(L, name)
            f.argtypes, f.restype = args, res
        _typed = L
    return _typed


def _torch():
    import torch
    return torch


_types = {}


def _dtype(t):
    if not _types:
        torch = _torch()
        _types.update({torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32})
    if t.dtype not in _types:
        raise FhcError(f"tensors of {t.dtype}: f16, bf16 or f32 is wanted")
    return _types[t.dtype]


def _run(name, rc):
    if rc < 0:
        raise FhcError(f"{name}: {fhconv.last_error()}")


def _on(stream):
    """What the call allocates is the stream's: freed memory is then not handed to another stream's work too early."""
    return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)


def _handle(stream):
    return (stream or _torch().cuda.current_stream()).cuda_stream


def _same(name, ref, **tensors):
    """Tensors of a call: ref's device (the current one), and the given (shape, dtype)."""
    torch = _torch()
    if not ref.is_cuda or ref.device.index != torch.cuda.current_device():
        raise FhcError(f"{name}: tensors have to be on the current GPU (got {ref.device})")
    for k, (t, shape, dtype) in tensors.items():
        if t is None:
            continue
        if t.device != ref.device or t.dtype != dtype or tuple(t.shape) != tuple(shape):
            raise FhcError(f"{name}: {k} is {tuple(t.shape)} {t.dtype} on {t.device}, wanted {tuple(shape)} {dtype} "
                           f"on {ref.device}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense(name, **tensors):
    for k, t in tensors.items():
        if t is not None and not t.is_contiguous():
            raise FhcError(f"{name}: {k} has to be contiguous")


def _seq(name, what, t):
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise FhcError(f"{name}: the channels of {what} have to be adjacent (strides {t.stride()})")
    return FhcSeq(t.data_ptr(), t.stride(0), t.stride(1))


def _like(x):
    """A new tensor in x's order of dimensions in memory (time-major inputs give time-major outputs)."""
    if x.shape[1] > 1 and x.shape[0] > 1 and x.stride(0) < x.stride(1):
        return x.new_empty((x.shape[1], x.shape[0], x.shape[2])).transpose(0, 1)
    return x.new_empty(x.shape)


def _bytes(x, n):
    return x.new_empty((n,), dtype=_torch().uint8) if n else None


def _glr_desc(name, x, r, i, lam, rate, lengths):
    torch = _torch()
    if x.dim() != 3:
        raise FhcError(f"{name}: x is [sequences, steps, channels], got {tuple(x.shape)}")
    dtype = _dtype(x)
    b, t, d = x.shape
    _same(name, x, r=(r, x.shape, x.dtype), i=(i, x.shape, x.dtype), lam=(lam, (d,), torch.float32),
          lengths=(lengths, (b,), torch.int32))
    _dense(name, lam=lam, lengths=lengths)
    return GlrDesc(dtype, b, t, d, rate, lam.data_ptr(), _ptr(lengths))


def glr(x, r, i, lam, rate=8.0, h0=None, lengths=None, train=False, stream=None):
    """The gated linear recurrence over x, r, i [sequences, steps, channels] (any order of the first two in memory):
    log a = -rate softplus(lam) sigmoid(r), h = a h + sqrt(1 - a^2) sigmoid(i) x from h0 ([sequences, channels] f32,
    or zeros). Returns (y, the last state), with train also the states that ``glr_backward`` takes. lengths: int32
    [sequences]; y past a sequence's length is 0 and its state stays."""
    L, torch = _lib(), _torch()
    g = _glr_desc("glr", x, r, i, lam, rate, lengths)
    _same("glr", x, h0=(h0, (g.b, g.d), torch.float32))
    _dense("glr", h0=h0)
    with _on(stream):
        y = _like(x)
        ht = x.new_empty((g.b, g.d), dtype=torch.float32)
        states = _bytes(x, L.fhc_glr_states_bytes(g)) if train else None
        n = L.fhc_glr_workspace_bytes(g, 0)
        ws = _bytes(x, n)
        _run("glr", L.fhc_glr_forward(g, _seq("glr", "x", x), _seq("glr", "r", r), _seq("glr", "i", i), _ptr(h0),
                                      _seq("glr", "y", y), ht.data_ptr(), _ptr(states), _ptr(ws), n, _handle(stream)))
    return (y, ht, states) if train else (y, ht)


def glr_backward(x, r, i, lam, states, dy, rate=8.0, dht=None, lengths=None, stream=None):
    """(dx, dr, di, dlam, dh0) of a loss with dy and dht ([sequences, channels] f32, or zeros); ``states`` from the
    training ``glr`` call of the same inputs."""
    L, torch, op = _lib(), _torch(), "glr_backward"
    g = _glr_desc(op, x, r, i, lam, rate, lengths)
    _same(op, x, dy=(dy, x.shape, x.dtype), dht=(dht, (g.b, g.d), torch.float32),
          states=(states, (L.fhc_glr_states_bytes(g),), torch.uint8))
    _dense(op, dht=dht)
    with _on(stream):
        dx, dr, di = _like(x), _like(r), _like(i)
        dlam = x.new_empty((g.d,), dtype=torch.float32)
        dh0 = x.new_empty((g.b, g.d), dtype=torch.float32)
        n = L.fhc_glr_workspace_bytes(g, 1)
        ws = _bytes(x, n)
        _run(op, L.fhc_glr_backward(g, _seq(op, "x", x), _seq(op, "r", r), _seq(op, "i", i), _ptr(states),
                                    _seq(op, "dy", dy), _ptr(dht), _seq(op, "dx", dx), _seq(op, "dr", dr),
                                    _seq(op, "di", di), dlam.data_ptr(), dh0.data_ptr(), _ptr(ws), n, _handle(stream)))
    return dx, dr, di, dlam, dh0


def _rows(name, what, t):
    if t is None:
        return None
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise FhcError(f"{name}: the channels of {what} have to be adjacent (strides {t.stride()})")
    return FhcRows(t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _norm_desc(name, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group):
    if x.dim() != 2:
        raise FhcError(f"{name}: x is [rows, channels], got {tuple(x.shape)}")
    rows, c = x.shape
    dtype = _dtype(x)
    groups = -(-rows // max(rows_per_group, 1))
    _same(name, x, o=(o, x.shape, x.dtype), w_post=(w_post, (c,), x.dtype), w_pre=(w_pre, (c,), x.dtype),
          gate=(gate, (groups, c), x.dtype))
    _dense(name, w_post=w_post, w_pre=w_pre, gate=gate)
    return NormDesc(dtype, rows, c, rows_per_group, alpha, eps, _ptr(w_post), _ptr(w_pre), _ptr(gate))


def norm_block(x, o, w_post, gate, w_pre, alpha=1.0, eps=1e-6, rows_per_group=1, stream=None):
    """y = alpha x + gate w_post o / rms(o) and u = w_pre y / rms(y) of rows x, o [rows, channels]; gate [groups,
    channels], one for each rows_per_group rows. o, w_post, gate and w_pre may be None. Returns (y, u)."""
    L, op = _lib(), "norm_block"
    n = _norm_desc(op, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group)
    with _on(stream):
        y, u = x.new_empty(x.shape), x.new_empty(x.shape)
        _run(op, L.fhc_norm_block(n, _rows(op, "x", x), _rows(op, "o", o), _rows(op, "y", y), _rows(op, "u", u),
                                  _handle(stream)))
    return y, u


def norm_block_backward(x, o, w_post, gate, w_pre, dy, du, alpha=1.0, eps=1e-6, rows_per_group=1, stream=None):
    """(dx, do, dw_post, dgate, dw_pre) for dy and du (either may be None); the sums of weights and gate are f32, and
    None where there is no weight, gate or block output."""
    L, torch, op = _lib(), _torch(), "norm_block_backward"
    n = _norm_desc(op, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group)
    _same(op, x, dy=(dy, x.shape, x.dtype), du=(du, x.shape, x.dtype))
    with _on(stream):
        dx = x.new_empty(x.shape)
        do = x.new_empty(x.shape) if o is not None else None
        dw_post, dgate, dw_pre = (None if w is None else w.new_empty(w.shape, dtype=torch.float32)
                                  for w in (w_post, gate, w_pre))
        size = L.fhc_norm_block_workspace_bytes(n)
        ws = _bytes(x, size)
        _run(op, L.fhc_norm_block_backward(n, _rows(op, "x", x), _rows(op, "o", o), _rows(op, "dy", dy),
                                           _rows(op, "du", du), _rows(op, "dx", dx), _rows(op, "do", do),
                                           _ptr(dw_post), _ptr(dgate), _ptr(dw_pre), _ptr(ws), size, _handle(stream)))
    return dx, do, dw_post, dgate, dw_pre


ACTS = {"silu": 0, "gelu": 1}


def _ffn_desc(name, x, wg, wu, wd, act):
    if x.dim() != 2 or wg.dim() != 2:
        raise FhcError(f"{name}: x is [rows, channels] and wg [features, channels], got {tuple(x.shape)}, "
                       f"{tuple(wg.shape)}")
    if act not in ACTS:
        raise FhcError(f"{name}: act {act!r} is none of {', '.join(ACTS)}")
    rows, c = x.shape
    f = wg.shape[0]
    dtype = _dtype(x)
    _same(name, x, wg=(wg, (f, c), x.dtype), wu=(wu, (f, c), x.dtype), wd=(wd, (c, f), x.dtype))
    _dense(name, wg=wg, wu=wu, wd=wd)
    return FfnDesc(dtype, ACTS[act], rows, c, f)


def ffn(x, wg, wu, wd, act="silu", train=False, stream=None):
    """(act(x wg^T) * (x wu^T)) wd^T of rows x [rows, c] with wg, wu [f, c] and wd [c, f], act "silu" or "gelu" (tanh
    form), in f16 or bf16. With train: (y, what ``ffn_backward`` takes)."""
    L, op = _lib(), "ffn"
    d = _ffn_desc(op, x, wg, wu, wd, act)
    with _on(stream):
        y = x.new_empty(x.shape)
        saved = _bytes(x, L.fhc_ffn_saved_bytes(d)) if train else None
        n = L.fhc_ffn_workspace_bytes(d, 0)
        ws = _bytes(x, n)
        _run(op, L.fhc_ffn_forward(d, _rows(op, "x", x), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(),
                                   _rows(op, "y", y), _ptr(saved), _ptr(ws), n, _handle(stream)))
    return (y, saved) if train else y


def ffn_backward(x, wg, wu, wd, saved, dy, act="silu", stream=None):
    """(dx, dwg, dwu, dwd), in the inputs' type, for dy; ``saved`` from the training ``ffn`` call of the same inputs."""
    L, torch, op = _lib(), _torch(), "ffn_backward"
    d = _ffn_desc(op, x, wg, wu, wd, act)
    size = L.fhc_ffn_saved_bytes(d)
    _same(op, x, dy=(dy, x.shape, x.dtype), saved=(saved, (size,), torch.uint8) if size else (None, (), None))
    with _on(stream):
        dx, dwg, dwu, dwd = (t.new_empty(t.shape) for t in (x, wg, wu, wd))
        n = L.fhc_ffn_workspace_bytes(d, 1)
        ws = _bytes(x, n)
        _run(op, L.fhc_ffn_backward(d, _rows(op, "x", x), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), _ptr(saved),
                                    _rows(op, "dy", dy), _rows(op, "dx", dx), dwg.data_ptr(), dwu.data_ptr(),
                                    dwd.data_ptr(), _ptr(ws), n, _handle(stream)))
    return dx, dwg, dwu, dwd
