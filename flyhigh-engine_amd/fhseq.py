"""Python host driver of the operators on rows of channels (ctypes over include/fhc_seq.h in libfhconv.so): a gated
linear recurrence (``glr``), the norms around a block with its gate and the scaled residual (``norm_block``), a gated
feed-forward block (``ffn``), a short causal convolution (``short_conv``), a selective state space scan (``ssm``) and a
matrix product with bias, activation and residual (``linear``), each with its backward pass.

Inputs are torch tensors on the current GPU in f16, bf16 or (not ``ffn`` and ``linear``) f32, all of one call in the same
type; the recurrences' states and the gradients of the weights of the recurrences, the norms and the convolution are f32.
Each function returns new tensors, which autograd does not know: a call with tensors that require gradients is refused while
autograd records (``torch.no_grad()``, and the ``*_backward`` functions, are the way). ``stream`` (a torch stream) is where
the call runs, the current stream if None; what it allocates belongs to that stream. The module only passes device pointers:
when the library is missing, loading it raises, and nothing is computed on the host.
"""
from __future__ import annotations

import ctypes
import functools
import struct

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


class ShortConvDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("act", _U), ("b", _U), ("t", _U), ("d", _U), ("k", _U), ("w", _P), ("bias", _P),
                ("lengths", _P)]


class SsmDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("b", _U), ("t", _U), ("d", _U), ("n", _U), ("groups", _U), ("a", _P), ("dt_bias", _P),
                ("skip", _P), ("lengths", _P)]


class LinearDesc(ctypes.Structure):
    _fields_ = [("dtype", _U), ("act", _U), ("rows", _U), ("c", _U), ("f", _U)]


class _Desc:
    """A structure's argument: the structure, a reference to it, or its packed bytes."""

    @staticmethod
    def from_param(v):
        if isinstance(v, bytes):
            return ctypes.c_char_p(v)
        return ctypes.byref(v) if isinstance(v, ctypes.Structure) else v


_typed = None


def _lib():
    global _typed
    if _typed is None:
        L = fhconv.load()
        G = S = N = R = D = _Desc
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
            "fhc_short_conv_forward": ([D, S, _P, S, _P, _P], ctypes.c_int),
            "fhc_short_conv_workspace_bytes": ([D], _SZ),
            "fhc_short_conv_backward": ([D, S, _P, S, _P, S, _P, _P, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_ssm_states_bytes": ([D], _SZ),
            "fhc_ssm_workspace_bytes": ([D, ctypes.c_int], _SZ),
            "fhc_ssm_forward": ([D, S, S, S, S, S, _P, S, _P, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_ssm_backward": ([D] + [S] * 5 + [_P, S, _P] + [S] * 5 + [_P] * 5 + [_SZ, _P], ctypes.c_int),
            "fhc_linear_saved_bytes": ([D], _SZ),
            "fhc_linear_workspace_bytes": ([D, ctypes.c_int], _SZ),
            "fhc_linear_forward": ([D, R, _P, _P, R, R, _P, _P, _SZ, _P], ctypes.c_int),
            "fhc_linear_backward": ([D, R, _P, _P, R, R, _P, _P, _P, _SZ, _P], ctypes.c_int),
        }
        for name, (args, res) in sig.items():
            f = getattr(L, name)
            f.argtypes, f.restype = args, res
        _typed = L
    return _typed


# A call for one token takes a few microseconds on the GPU, so the host's side is kept short: descriptors go as packed
# bytes (ctypes structures cost several times as much to fill), sizes of workspaces are asked once a shape, and the
# stream's handle is read without a Stream object.
_GLR, _SEQ = struct.Struct("@IIIIfPP").pack, struct.Struct("@Pqq").pack
_NORM, _ROWS, _FFN = struct.Struct("@IIIIffPPP").pack, struct.Struct("@Pq").pack, struct.Struct("@IIIII").pack
_CONV, _SSM, _LINEAR = struct.Struct("@IIIIIIPPP").pack, struct.Struct("@IIIIIIPPPP").pack, _FFN


class _Fast:
    """The entry points taking descriptors as bytes and pointers as integers, and what torch is asked at every call."""

    def __init__(self):
        import torch
        L = _lib()
        for name in ("fhc_glr_forward", "fhc_glr_backward", "fhc_norm_block", "fhc_norm_block_backward",
                     "fhc_ffn_forward", "fhc_ffn_backward", "fhc_short_conv_forward", "fhc_short_conv_backward",
                     "fhc_ssm_forward", "fhc_ssm_backward", "fhc_linear_forward", "fhc_linear_backward"):
            types = [_SZ if t is _SZ else _P for t in getattr(L, name).argtypes]
            setattr(self, name[4:], ctypes.CFUNCTYPE(ctypes.c_int, *types)((name, L)))
        self.torch, self.empty_like, self.empty = torch, torch.empty_like, torch.empty
        self.new = functools.partial(torch.empty_like, memory_format=torch.contiguous_format)
        self.f32, self.i32, self.u8 = torch.float32, torch.int32, torch.uint8
        self.types = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
        self.recording = torch.is_grad_enabled
        self.device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda _: torch.cuda.current_stream().cuda_stream)


_fast_calls = None


def _fast():
    global _fast_calls
    if _fast_calls is None:
        _fast_calls = _Fast()
    return _fast_calls


@functools.lru_cache(4096)
def _glr_sizes(dtype, b, t, d):
    """Bytes of the states, and of the workspace forward and backward."""
    L, g = _lib(), GlrDesc(dtype, b, t, d, 1.0, 256, None)
    return L.fhc_glr_states_bytes(g), L.fhc_glr_workspace_bytes(g, 0), L.fhc_glr_workspace_bytes(g, 1)


@functools.lru_cache(4096)
def _norm_size(dtype, rows, c, rows_per_group, has_gate):
    return _lib().fhc_norm_block_workspace_bytes(
        NormDesc(dtype, rows, c, rows_per_group, 1.0, 1.0, None, None, 256 if has_gate else None))


@functools.lru_cache(4096)
def _ffn_sizes(dtype, act, rows, c, f):
    """Bytes of what a training forward keeps, and of the workspace forward and backward."""
    L, d = _lib(), FfnDesc(dtype, act, rows, c, f)
    return L.fhc_ffn_saved_bytes(d), L.fhc_ffn_workspace_bytes(d, 0), L.fhc_ffn_workspace_bytes(d, 1)


@functools.lru_cache(4096)
def _conv_size(dtype, b, t, d, taps):
    return _lib().fhc_short_conv_workspace_bytes(ShortConvDesc(dtype, 0, b, t, d, taps, 256, None, None))


@functools.lru_cache(4096)
def _ssm_sizes(dtype, b, t, d, n, groups):
    """Bytes of the states, and of the workspace forward and backward."""
    L, g = _lib(), SsmDesc(dtype, b, t, d, n, groups, 256, None, None, None)
    return L.fhc_ssm_states_bytes(g), L.fhc_ssm_workspace_bytes(g, 0), L.fhc_ssm_workspace_bytes(g, 1)


@functools.lru_cache(4096)
def _linear_sizes(dtype, act, rows, c, f):
    """Bytes of what a training forward keeps, and of the workspace forward and backward."""
    L, d = _lib(), LinearDesc(dtype, act, rows, c, f)
    return L.fhc_linear_saved_bytes(d), L.fhc_linear_workspace_bytes(d, 0), L.fhc_linear_workspace_bytes(d, 1)


def _on(stream):
    """Runs a call on its stream: what it allocates is then the stream's, and freed memory is not handed to another
    stream's work too early."""
    return _fast().torch.cuda.stream(stream)


def _pack(name, pack, *fields):
    try:
        return pack(*fields)
    except (struct.error, OverflowError) as e:  # a negative count, a float beyond f32
        raise FhcError(f"{name}: {e}") from None


def _refuse(name):
    raise FhcError(f"{name}: {fhconv.last_error()}")


def _unrecorded(k, name, *tensors):
    """The results would lose their gradients without a word."""
    if k.recording():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise FhcError(f"{name}: a tensor requires gradients, which this call does not record: call it under "
                               f"torch.no_grad() or with detached tensors, and take them from the *_backward function")


def _first(k, name, x):
    """(its type's number, its device) of a call's first tensor, which has to be on the current GPU."""
    dtype = k.types.get(x.dtype)
    if dtype is None:
        raise FhcError(f"{name}: tensors of {x.dtype}: f16, bf16 or f32 is wanted")
    at = x.get_device()
    if at < 0 or at != k.device():
        raise FhcError(f"{name}: tensors have to be on the current GPU (got {x.device})")
    return dtype, at


def _match(name, what, t, shape, dtype, at):
    if t.dtype is not dtype or t.shape != shape or t.get_device() != at:
        raise FhcError(f"{name}: {what} is {tuple(t.shape)} {t.dtype} on {t.device}, wanted {tuple(shape)} {dtype} "
                       f"on the current GPU")


def _dense(name, what, t, shape, dtype, at):
    """The pointer of a dense tensor, None for None."""
    if t is None:
        return None
    _match(name, what, t, shape, dtype, at)
    if not t.is_contiguous():
        raise FhcError(f"{name}: {what} has to be contiguous")
    return t.data_ptr()


def _seq(name, what, t):
    bs, ts, cs = t.stride()
    if cs != 1 and t.shape[2] > 1:
        raise FhcError(f"{name}: the channels of {what} have to be adjacent (strides {t.stride()})")
    return _SEQ(t.data_ptr(), bs, ts)


def _new_seq(k, x):
    """An output of x's shape, in x's order in memory (time-major inputs give time-major outputs) where it has one with
    the channels adjacent: sequences or steps that overlap by all but one element have none."""
    y = k.empty_like(x)
    return y if y.stride(2) == 1 or y.shape[2] <= 1 else k.new(x)


def _like_seq(name, what, t, x, at):
    if t.dtype is not x.dtype or t.shape != x.shape or t.get_device() != at:
        _match(name, what, t, x.shape, x.dtype, at)
    return _seq(name, what, t)


def _bytes(k, n, at):
    return k.empty((n,), dtype=k.u8, device=at) if n else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _glr_desc(k, name, x, r, i, lam, rate, lengths):
    if x.dim() != 3:
        raise FhcError(f"{name}: x is [sequences, steps, channels], got {tuple(x.shape)}")
    dtype, at = _first(k, name, x)
    b, t, d = x.shape
    g = _pack(name, _GLR, dtype, b, t, d, rate, _dense(name, "lam", lam, (d,), k.f32, at),
              _dense(name, "lengths", lengths, (b,), k.i32, at) or 0)
    return (g, _glr_sizes(dtype, b, t, d), at, _seq(name, "x", x),
            _like_seq(name, "r", r, x, at), _like_seq(name, "i", i, x, at))


def glr(x, r, i, lam, rate=8.0, h0=None, lengths=None, train=False, stream=None):
    """The gated linear recurrence over x, r, i [sequences, steps, channels] (any order of the first two in memory):
    log a = -rate softplus(lam) sigmoid(r), h = a h + sqrt(1 - a^2) sigmoid(i) x from h0 ([sequences, channels] f32,
    or zeros). Returns (y, the last state), with train also the states that ``glr_backward`` takes. lengths: int32
    [sequences]; y past a sequence's length is 0 and its state stays."""
    if stream is not None:
        with _on(stream):
            return glr(x, r, i, lam, rate, h0, lengths, train)
    k, op = _fast(), "glr"
    _unrecorded(k, op, x, r, i, lam, h0)
    g, sizes, at, sx, sr, si = _glr_desc(k, op, x, r, i, lam, rate, lengths)
    b, _, d = x.shape
    start = _dense(op, "h0", h0, (b, d), k.f32, at)
    y = _new_seq(k, x)
    ht = k.empty((b, d), dtype=k.f32, device=at) if h0 is None else k.empty_like(h0)
    states = k.empty((sizes[0],), dtype=k.u8, device=at) if train else None
    n = sizes[1]
    ws = _bytes(k, n, at)
    if k.glr_forward(g, sx, sr, si, start, _seq(op, "y", y), ht.data_ptr(), _ptr(states), _ptr(ws), n,
                     k.raw_stream(at)) < 0:
        _refuse(op)
    return (y, ht, states) if train else (y, ht)


def glr_backward(x, r, i, lam, states, dy, rate=8.0, dht=None, lengths=None, stream=None):
    """(dx, dr, di, dlam, dh0) of a loss with dy and dht ([sequences, channels] f32, or zeros); ``states`` from the
    training ``glr`` call of the same inputs."""
    if stream is not None:
        with _on(stream):
            return glr_backward(x, r, i, lam, states, dy, rate, dht, lengths)
    k, op = _fast(), "glr_backward"
    _unrecorded(k, op, x, r, i, lam, dy, dht)
    g, sizes, at, sx, sr, si = _glr_desc(k, op, x, r, i, lam, rate, lengths)
    b, _, d = x.shape
    end = _dense(op, "dht", dht, (b, d), k.f32, at)
    kept = _dense(op, "states", states, (sizes[0],), k.u8, at)
    sdy = _like_seq(op, "dy", dy, x, at)
    dx, dr, di = _new_seq(k, x), _new_seq(k, r), _new_seq(k, i)
    dlam = k.empty((d,), dtype=k.f32, device=at)
    dh0 = k.empty((b, d), dtype=k.f32, device=at)
    n = sizes[2]
    ws = _bytes(k, n, at)
    if k.glr_backward(g, sx, sr, si, kept, sdy, end, _seq(op, "dx", dx), _seq(op, "dr", dr), _seq(op, "di", di),
                      dlam.data_ptr(), dh0.data_ptr(), _ptr(ws), n, k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, dr, di, dlam, dh0


def _rows(name, what, t):
    if t is None:
        return None
    rows, c = t.shape
    ld, cs = t.stride()
    if cs != 1 and c > 1:
        raise FhcError(f"{name}: the channels of {what} have to be adjacent (strides {t.stride()})")
    return _ROWS(t.data_ptr(), ld if rows > 1 else c)


def _like_rows(name, what, t, x, at):
    if t is None:
        return None
    _match(name, what, t, x.shape, x.dtype, at)
    return _rows(name, what, t)


def _norm_desc(k, name, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group):
    if x.dim() != 2:
        raise FhcError(f"{name}: x is [rows, channels], got {tuple(x.shape)}")
    dtype, at = _first(k, name, x)
    rows, c = x.shape
    ty = x.dtype
    groups = -(-rows // rows_per_group) if rows_per_group > 1 else rows
    n = _pack(name, _NORM, dtype, rows, c, rows_per_group, alpha, eps, _dense(name, "w_post", w_post, (c,), ty, at) or 0,
              _dense(name, "w_pre", w_pre, (c,), ty, at) or 0, _dense(name, "gate", gate, (groups, c), ty, at) or 0)
    return n, at, dtype, _rows(name, "x", x), _like_rows(name, "o", o, x, at)


def norm_block(x, o, w_post, gate, w_pre, alpha=1.0, eps=1e-6, rows_per_group=1, stream=None):
    """y = alpha x + gate w_post o / rms(o) and u = w_pre y / rms(y) of rows x, o [rows, channels]; gate [groups,
    channels], one for each rows_per_group rows. o, w_post, gate and w_pre may be None. Returns (y, u)."""
    if stream is not None:
        with _on(stream):
            return norm_block(x, o, w_post, gate, w_pre, alpha, eps, rows_per_group)
    k, op = _fast(), "norm_block"
    _unrecorded(k, op, x, o, w_post, gate, w_pre)
    n, at, _, rx, ro = _norm_desc(k, op, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group)
    y, u = k.new(x), k.new(x)
    c = x.shape[1]
    if k.norm_block(n, rx, ro, _ROWS(y.data_ptr(), c), _ROWS(u.data_ptr(), c), k.raw_stream(at)) < 0:
        _refuse(op)
    return y, u


def norm_block_backward(x, o, w_post, gate, w_pre, dy, du, alpha=1.0, eps=1e-6, rows_per_group=1, stream=None):
    """(dx, do, dw_post, dgate, dw_pre) for dy and du (either may be None); the sums of weights and gate are f32, and
    None where there is no weight, gate or block output."""
    if stream is not None:
        with _on(stream):
            return norm_block_backward(x, o, w_post, gate, w_pre, dy, du, alpha, eps, rows_per_group)
    k, op = _fast(), "norm_block_backward"
    _unrecorded(k, op, x, o, w_post, gate, w_pre, dy, du)
    n, at, dtype, rx, ro = _norm_desc(k, op, x, o, w_post, gate, w_pre, alpha, eps, rows_per_group)
    rdy, rdu = _like_rows(op, "dy", dy, x, at), _like_rows(op, "du", du, x, at)
    rows, c = x.shape
    dx = k.new(x)
    do = k.new(x) if o is not None else None
    dw_post, dgate, dw_pre = (None if w is None else k.empty(w.shape, dtype=k.f32, device=at)
                              for w in (w_post, gate, w_pre))
    size = _norm_size(dtype, rows, c, rows_per_group, gate is not None)
    ws = _bytes(k, size, at)
    if k.norm_block_backward(n, rx, ro, rdy, rdu, _ROWS(dx.data_ptr(), c), None if do is None else _rows(op, "do", do),
                             _ptr(dw_post), _ptr(dgate), _ptr(dw_pre), _ptr(ws), size, k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, do, dw_post, dgate, dw_pre


ACTS = {"silu": 0, "gelu": 1}


def _ffn_desc(k, name, x, wg, wu, wd, act):
    if x.dim() != 2 or wg.dim() != 2:
        raise FhcError(f"{name}: x is [rows, channels] and wg [features, channels], got {tuple(x.shape)}, "
                       f"{tuple(wg.shape)}")
    if act not in ACTS:
        raise FhcError(f"{name}: act {act!r} is none of {', '.join(ACTS)}")
    dtype, at = _first(k, name, x)
    rows, c = x.shape
    f = wg.shape[0]
    act, ty = ACTS[act], x.dtype
    return (_FFN(dtype, act, rows, c, f), at, _ffn_sizes(dtype, act, rows, c, f), _rows(name, "x", x),
            _dense(name, "wg", wg, (f, c), ty, at), _dense(name, "wu", wu, (f, c), ty, at),
            _dense(name, "wd", wd, (c, f), ty, at))


def ffn(x, wg, wu, wd, act="silu", train=False, stream=None):
    """(act(x wg^T) * (x wu^T)) wd^T of rows x [rows, c] with wg, wu [f, c] and wd [c, f], act "silu" or "gelu" (tanh
    form), in f16 or bf16. With train: (y, what ``ffn_backward`` takes)."""
    if stream is not None:
        with _on(stream):
            return ffn(x, wg, wu, wd, act, train)
    k, op = _fast(), "ffn"
    _unrecorded(k, op, x, wg, wu, wd)
    d, at, sizes, rx, pg, pu, pd = _ffn_desc(k, op, x, wg, wu, wd, act)
    y = k.new(x)
    saved = _bytes(k, sizes[0], at) if train else None
    n = sizes[1]
    ws = _bytes(k, n, at)
    if k.ffn_forward(d, rx, pg, pu, pd, _ROWS(y.data_ptr(), x.shape[1]), _ptr(saved), _ptr(ws), n,
                     k.raw_stream(at)) < 0:
        _refuse(op)
    return (y, saved) if train else y


def ffn_backward(x, wg, wu, wd, saved, dy, act="silu", stream=None):
    """(dx, dwg, dwu, dwd), in the inputs' type, for dy; ``saved`` from the training ``ffn`` call of the same inputs."""
    if stream is not None:
        with _on(stream):
            return ffn_backward(x, wg, wu, wd, saved, dy, act)
    k, op = _fast(), "ffn_backward"
    _unrecorded(k, op, x, wg, wu, wd, dy)
    d, at, sizes, rx, pg, pu, pd = _ffn_desc(k, op, x, wg, wu, wd, act)
    kept = _dense(op, "saved", saved, (sizes[0],), k.u8, at) if sizes[0] else None
    rdy = _like_rows(op, "dy", dy, x, at)
    dx, dwg, dwu, dwd = (k.new(t) for t in (x, wg, wu, wd))
    n = sizes[2]
    ws = _bytes(k, n, at)
    if k.ffn_backward(d, rx, pg, pu, pd, kept, rdy, _ROWS(dx.data_ptr(), x.shape[1]), dwg.data_ptr(), dwu.data_ptr(),
                      dwd.data_ptr(), _ptr(ws), n, k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, dwg, dwu, dwd


CONV_ACTS = {"silu": 0, "none": 2}


def _conv_desc(k, name, x, w, bias, act, state, lengths):
    if x.dim() != 3 or w.dim() != 2:
        raise FhcError(f"{name}: x is [sequences, steps, channels] and w [channels, taps], got {tuple(x.shape)}, "
                       f"{tuple(w.shape)}")
    if act not in CONV_ACTS:
        raise FhcError(f"{name}: act {act!r} is none of {', '.join(CONV_ACTS)}")
    dtype, at = _first(k, name, x)
    b, t, d = x.shape
    ty, taps = x.dtype, w.shape[1]
    g = _pack(name, _CONV, dtype, CONV_ACTS[act], b, t, d, taps, _dense(name, "w", w, (d, taps), ty, at) or 0,
              _dense(name, "bias", bias, (d,), ty, at) or 0, _dense(name, "lengths", lengths, (b,), k.i32, at) or 0)
    return g, at, dtype, taps, _seq(name, "x", x), _dense(name, "state", state, (b, taps - 1, d), ty, at)


def short_conv(x, w, bias=None, act="silu", state=None, lengths=None, stream=None):
    """The causal convolution of x [sequences, steps, channels] along its steps with w [channels, taps] (2 to 4 taps, the
    last one meets a step's own input): y_t = act(bias + sum_j w[j] x_(t - taps + 1 + j)), act "silu" or "none", behind
    ``state`` [sequences, taps - 1, channels] (or zeros), the inputs before the first, the oldest first. Returns (y, the
    state that the next call takes). lengths: int32 [sequences]; y past a sequence's length is 0."""
    if stream is not None:
        with _on(stream):
            return short_conv(x, w, bias, act, state, lengths)
    k, op = _fast(), "short_conv"
    _unrecorded(k, op, x, w, bias, state)
    g, at, _, taps, sx, before = _conv_desc(k, op, x, w, bias, act, state, lengths)
    y = _new_seq(k, x)
    end = k.empty((x.shape[0], max(taps - 1, 0), x.shape[2]), dtype=x.dtype, device=at)
    if k.short_conv_forward(g, sx, before, _seq(op, "y", y), end.data_ptr(), k.raw_stream(at)) < 0:
        _refuse(op)
    return y, end


def short_conv_backward(x, w, bias, dy, act="silu", state=None, dstate=None, lengths=None, stream=None):
    """(dx, dw, dbias, the gradient of ``state``) of a loss with dy and dstate (that of the state that was returned, or
    zeros); dw and dbias are f32."""
    if stream is not None:
        with _on(stream):
            return short_conv_backward(x, w, bias, dy, act, state, dstate, lengths)
    k, op = _fast(), "short_conv_backward"
    _unrecorded(k, op, x, w, bias, dy, state, dstate)
    g, at, dtype, taps, sx, before = _conv_desc(k, op, x, w, bias, act, state, lengths)
    b, t, d = x.shape
    sdy = _like_seq(op, "dy", dy, x, at)
    dend = _dense(op, "dstate", dstate, (b, taps - 1, d), x.dtype, at)
    dx = _new_seq(k, x)
    dw, dbias = k.empty((d, taps), dtype=k.f32, device=at), k.empty((d,), dtype=k.f32, device=at)
    dbefore = k.empty((b, max(taps - 1, 0), d), dtype=x.dtype, device=at)
    n = _conv_size(dtype, b, t, d, taps)
    ws = _bytes(k, n, at)
    if k.short_conv_backward(g, sx, before, sdy, dend, _seq(op, "dx", dx), dw.data_ptr(), dbias.data_ptr(),
                             dbefore.data_ptr(), _ptr(ws), n, k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, dw, dbias, dbefore


def _ssm_desc(k, name, x, dt, a, bm, cm, skip, z, dt_bias, lengths):
    if x.dim() != 3 or a.dim() != 2 or bm.dim() != 3:
        raise FhcError(f"{name}: x is [sequences, steps, channels], a [channels, states] and bm [sequences, steps, groups "
                       f"* states], got {tuple(x.shape)}, {tuple(a.shape)}, {tuple(bm.shape)}")
    dtype, at = _first(k, name, x)
    b, t, d = x.shape
    n, wide = a.shape[1], bm.shape[2]
    groups = wide // n if n and wide % n == 0 else 0
    if groups < 1:
        raise FhcError(f"{name}: bm has {wide} values a step, not a multiple of the {n} states of a")
    g = _pack(name, _SSM, dtype, b, t, d, n, groups, _dense(name, "a", a, (d, n), k.f32, at) or 0,
              _dense(name, "dt_bias", dt_bias, (d,), k.f32, at) or 0, _dense(name, "skip", skip, (d,), k.f32, at) or 0,
              _dense(name, "lengths", lengths, (b,), k.i32, at) or 0)
    for what, m in (("bm", bm), ("cm", cm)):
        if m.dtype is not x.dtype or m.shape != (b, t, wide) or m.get_device() != at:
            _match(name, what, m, (b, t, wide), x.dtype, at)
    seqs = (_seq(name, "x", x), _like_seq(name, "dt", dt, x, at), _seq(name, "bm", bm), _seq(name, "cm", cm),
            None if z is None else _like_seq(name, "z", z, x, at))
    return g, at, _ssm_sizes(dtype, b, t, d, n, groups), n, seqs


def ssm(x, dt, a, bm, cm, skip=None, z=None, dt_bias=None, h0=None, lengths=None, train=False, stream=None):
    """The selective state space scan over x, dt, z [sequences, steps, channels] and bm, cm [sequences, steps, groups *
    states] with a [channels, states], skip and dt_bias [channels] in f32: D = softplus(dt + dt_bias),
    h = exp(D a) h + D x B from h0 ([sequences, channels, states] f32, or zeros), y = (sum C h + skip x) silu(z).
    Returns (y, the last states), with train also the states that ``ssm_backward`` takes. lengths: int32 [sequences]; y
    past a sequence's length is 0 and its states stay."""
    if stream is not None:
        with _on(stream):
            return ssm(x, dt, a, bm, cm, skip, z, dt_bias, h0, lengths, train)
    k, op = _fast(), "ssm"
    _unrecorded(k, op, x, dt, a, bm, cm, skip, z, dt_bias, h0)
    g, at, sizes, n, seqs = _ssm_desc(k, op, x, dt, a, bm, cm, skip, z, dt_bias, lengths)
    b, _, d = x.shape
    start = _dense(op, "h0", h0, (b, d, n), k.f32, at)
    y = _new_seq(k, x)
    ht = k.empty((b, d, n), dtype=k.f32, device=at)
    states = k.empty((sizes[0],), dtype=k.u8, device=at) if train else None
    ws = _bytes(k, sizes[1], at)
    if k.ssm_forward(g, *seqs, start, _seq(op, "y", y), ht.data_ptr(), _ptr(states), _ptr(ws), sizes[1],
                     k.raw_stream(at)) < 0:
        _refuse(op)
    return (y, ht, states) if train else (y, ht)


def ssm_backward(x, dt, a, bm, cm, states, dy, skip=None, z=None, dt_bias=None, dht=None, lengths=None, stream=None):
    """(dx, ddt, da, dbm, dcm, dskip, dz, ddt_bias, dh0) of a loss with dy and dht ([sequences, channels, states] f32, or
    zeros); ``states`` from the training ``ssm`` call of the same inputs. da, dskip, ddt_bias and dh0 are f32; dskip and
    ddt_bias also where there was no weight, dz is None without z."""
    if stream is not None:
        with _on(stream):
            return ssm_backward(x, dt, a, bm, cm, states, dy, skip, z, dt_bias, dht, lengths)
    k, op = _fast(), "ssm_backward"
    _unrecorded(k, op, x, dt, a, bm, cm, dy, skip, z, dt_bias, dht)
    g, at, sizes, n, seqs = _ssm_desc(k, op, x, dt, a, bm, cm, skip, z, dt_bias, lengths)
    b, _, d = x.shape
    end = _dense(op, "dht", dht, (b, d, n), k.f32, at)
    kept = _dense(op, "states", states, (sizes[0],), k.u8, at)
    sdy = _like_seq(op, "dy", dy, x, at)
    dx, ddt, dbm, dcm = _new_seq(k, x), _new_seq(k, dt), _new_seq(k, bm), _new_seq(k, cm)
    dz = None if z is None else _new_seq(k, z)
    da, dskip, ddt_bias, dh0 = (k.empty(s, dtype=k.f32, device=at) for s in ((d, n), (d,), (d,), (b, d, n)))
    ws = _bytes(k, sizes[2], at)
    if k.ssm_backward(g, *seqs, kept, sdy, end, _seq(op, "dx", dx), _seq(op, "ddt", ddt), _seq(op, "dbm", dbm),
                      _seq(op, "dcm", dcm), None if dz is None else _seq(op, "dz", dz), da.data_ptr(),
                      ddt_bias.data_ptr(), dskip.data_ptr(), dh0.data_ptr(), _ptr(ws), sizes[2], k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, ddt, da, dbm, dcm, dskip, dz, ddt_bias, dh0


LINEAR_ACTS, ROUND_DV = {"silu": 0, "gelu": 1, "none": 2}, 0x100


def _linear_desc(k, name, x, w, act, flag=0):
    if x.dim() != 2 or w.dim() != 2:
        raise FhcError(f"{name}: x is [rows, channels] and w [features, channels], got {tuple(x.shape)}, "
                       f"{tuple(w.shape)}")
    if act not in LINEAR_ACTS:
        raise FhcError(f"{name}: act {act!r} is none of {', '.join(LINEAR_ACTS)}")
    dtype, at = _first(k, name, x)
    rows, c = x.shape
    f, act = w.shape[0], LINEAR_ACTS[act] + flag
    return (_pack(name, _LINEAR, dtype, act, rows, c, f), at, _linear_sizes(dtype, act, rows, c, f),
            _rows(name, "x", x), _dense(name, "w", w, (f, c), x.dtype, at))


def linear(x, w, bias=None, residual=None, act="none", train=False, stream=None):
    """act(x w^T + bias) + residual of rows x [rows, c] with w [f, c], bias [f] and residual [rows, f], act "none", "silu"
    or "gelu" (tanh form), in f16 or bf16. With train: (y, what ``linear_backward`` takes)."""
    if stream is not None:
        with _on(stream):
            return linear(x, w, bias, residual, act, train)
    k, op = _fast(), "linear"
    _unrecorded(k, op, x, w, bias, residual)
    d, at, sizes, rx, pw = _linear_desc(k, op, x, w, act)
    rows, f = x.shape[0], w.shape[0]
    pb = _dense(op, "bias", bias, (f,), x.dtype, at)
    y = k.empty((rows, f), dtype=x.dtype, device=at)
    res = _like_rows(op, "residual", residual, y, at)
    saved = _bytes(k, sizes[0], at) if train else None
    n = sizes[1]
    ws = _bytes(k, n, at)
    if k.linear_forward(d, rx, pw, pb, res, _ROWS(y.data_ptr(), f), _ptr(saved), _ptr(ws), n, k.raw_stream(at)) < 0:
        _refuse(op)
    return (y, saved) if train else y


def linear_backward(x, w, saved, dy, act="none", bias=True, stream=None, round_dv=False):
    """(dx, dw, dbias) for dy, dx and dw in the inputs' type and dbias in f32 (None where bias is false); ``saved`` from the
    training ``linear`` call of the same inputs (None where it kept nothing). The residual's gradient is dy. ``round_dv``:
    with an activation, the gradient behind it is rounded to the inputs' type before the products for dx and dw, which
    halves their work."""
    if stream is not None:
        with _on(stream):
            return linear_backward(x, w, saved, dy, act, bias, None, round_dv)
    k, op = _fast(), "linear_backward"
    _unrecorded(k, op, x, w, dy)
    d, at, sizes, rx, pw = _linear_desc(k, op, x, w, act, ROUND_DV if round_dv else 0)
    rows, f = x.shape[0], w.shape[0]
    kept = _dense(op, "saved", saved, (sizes[0],), k.u8, at) if sizes[0] else None
    _match(op, "dy", dy, (rows, f), x.dtype, at)
    dx, dw = k.new(x), k.new(w)
    dbias = k.empty((f,), dtype=k.f32, device=at) if bias else None
    n = sizes[2]
    ws = _bytes(k, n, at)
    if k.linear_backward(d, rx, pw, kept, _rows(op, "dy", dy), _ROWS(dx.data_ptr(), x.shape[1]), dw.data_ptr(),
                         _ptr(dbias), _ptr(ws), n, k.raw_stream(at)) < 0:
        _refuse(op)
    return dx, dw, dbias
