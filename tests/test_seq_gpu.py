"""The operators on rows of channels (through fhseq.py and the C ABI, include/fhc_seq.h) against plain 64-bit forms,
on the GPU. The tolerances are the forms' own error bounds (tests/seqref.py) plus half a step of each output's type."""
import math

import pytest

import fhtest  # noqa: F401  (puts the package on sys.path)
import seqref

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def mod():
    import fhseq
    return fhseq


def types():
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


class Rand:
    def __init__(self, seed):
        import torch
        self.torch, self.g = torch, torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0, dtype=None):
        v = self.torch.randn(*shape, generator=self.g, device="cuda") * scale
        return v.to(dtype) if dtype is not None else v

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return self.torch.rand(*shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def ints(self, lo, hi, n):
        return self.torch.randint(lo, hi, (n,), generator=self.g, device="cuda", dtype=self.torch.int32)


# ---- the gated linear recurrence --------------------------------------------------------------------------------

GLR = [  # b, t, d: one step; less and more than a wave's stretch, a chunk; odd widths; each way of walking the chunks
    (1, 1, 1), (5, 1, 64), (3, 2, 7), (2, 8, 130), (2, 16, 66), (2, 17, 66), (1, 64, 33), (3, 65, 34), (2, 200, 128),
    (1, 1000, 130), (1, 1537, 3), (2, 700, 250), (40, 70, 2048), (70, 130, 1001), (300, 20, 2048), (1030, 9, 512),
]


def glr_inputs(q, b, t, d, dtype, time_major=False, ragged=False):
    def seq():
        return q.normal(t, b, d, dtype=dtype).transpose(0, 1) if time_major else q.normal(b, t, d, dtype=dtype)

    lengths = None
    if ragged:
        lengths = q.ints(0, t + 1, b)
        lengths[-1] = 0
        lengths[0] = t
    return dict(x=seq(), r=seq(), i=seq(), lam=q.normal(d, scale=1.5) - 4, h0=q.normal(b, d), dy=seq(),
                dht=q.normal(b, d), lengths=lengths)


def glr_check(v, rate=8.0):
    m = mod()
    y, ht, states = m.glr(v["x"], v["r"], v["i"], v["lam"], rate, h0=v["h0"], lengths=v["lengths"], train=True)
    grads = m.glr_backward(v["x"], v["r"], v["i"], v["lam"], states, v["dy"], rate, dht=v["dht"],
                           lengths=v["lengths"])
    ref, err = seqref.glr(v["x"], v["r"], v["i"], v["lam"], rate, v["h0"], v["lengths"], v["dy"], v["dht"])
    for name, got, want, tol in zip(("y", "ht", "dx", "dr", "di", "dlam", "dh0"), (y, ht) + grads, ref, err):
        seqref.close(got, want, tol, name)
    return (y, ht) + grads


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", GLR, ids=str)
def test_glr(shape, dtype):
    say("glr", shape, dtype)
    q = Rand(sum(shape))
    glr_check(glr_inputs(q, *shape, types()[dtype], time_major=shape[2] % 3 == 0, ragged=shape[1] % 2 == 1))


@pytest.mark.parametrize("shape", [(4, 9, 10), (3, 131, 64), (40, 140, 2048)], ids=str)
def test_glr_masked_places_are_not_read(shape):
    """NaN and infinities past the lengths, empty sequences, lengths outside [0, t]."""
    say("glr masked", shape)
    import torch
    q = Rand(7)
    v = glr_inputs(q, *shape, torch.float16, ragged=True)
    v["lengths"][1], v["lengths"][2] = shape[1] + 1000, -3
    past = torch.arange(shape[1], device="cuda")[None] >= v["lengths"][:, None]
    clean = glr_check(v)
    for k, bad in (("x", math.nan), ("r", math.inf), ("i", math.nan), ("dy", -math.inf)):
        v[k] = v[k].masked_fill(past[:, :, None], bad)
    m = mod()
    y, ht, st = m.glr(v["x"], v["r"], v["i"], v["lam"], h0=v["h0"], lengths=v["lengths"], train=True)
    got = (y, ht) + m.glr_backward(v["x"], v["r"], v["i"], v["lam"], st, v["dy"], dht=v["dht"], lengths=v["lengths"])
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert not y[past].any() and not got[2][past].any()
    assert torch.equal(ht[2], v["h0"][2])  # an empty sequence's state


@pytest.mark.parametrize("t", [0, 1, 40, 300])
def test_glr_gates_at_their_ends(t):
    """Gates shut and open beyond f32's exponent range: the state stays, or is replaced; no gradient is NaN."""
    say("glr ends", t)
    import torch
    q = Rand(3)
    v = glr_inputs(q, 2, t, 48, torch.float32)
    v["r"][:, :, :8], v["r"][:, :, 8:16] = -200.0, 200.0
    v["i"][:, :, 16:24], v["i"][:, :, 24:32] = -200.0, 200.0
    v["r"][:, :, 32:36] = -math.inf
    v["lam"][36:40], v["lam"][40:44] = -120.0, 40.0
    m = mod()
    y, ht, st = m.glr(v["x"], v["r"], v["i"], v["lam"], h0=v["h0"], train=True)
    grads = m.glr_backward(v["x"], v["r"], v["i"], v["lam"], st, v["dy"], dht=v["dht"])
    assert all(torch.isfinite(k).all() for k in (y, ht) + grads)
    assert torch.equal(ht[:, :8], v["h0"][:, :8]) and torch.equal(ht[:, 32:36], v["h0"][:, 32:36])
    if t:
        ref, _ = seqref.glr(v["x"], v["r"], v["i"], v["lam"], 8.0, v["h0"])
        assert torch.allclose(y.double(), ref[0], rtol=1e-4, atol=1e-5)


def test_glr_views_strides_and_states_in_place():
    """Views into wider buffers, at odd offsets, equal the dense call; the state may be updated in place."""
    say("glr views")
    import torch
    q = Rand(11)
    b, t, d = 3, 150, 40
    m = mod()
    for off in (0, 1, 2):
        wide = [q.normal(t, b, 3 * d + 5, dtype=torch.bfloat16) for _ in range(3)]
        x, r, i = (w[:, :, off:off + d].transpose(0, 1) for w in wide)
        lam, h0 = q.normal(d) - 4, q.normal(b, d)
        y, ht = m.glr(x, r, i, lam, h0=h0)
        y2, ht2 = m.glr(x.contiguous(), r.contiguous(), i.contiguous(), lam, h0=h0)
        assert torch.equal(y, y2) and torch.equal(ht, ht2)
    # step by step over the same tokens, the state in place
    L = m._lib()
    import ctypes
    state = h0.clone()
    for k in range(t):
        step = [v[:, k:k + 1] for v in (x, r, i)]
        g = m.GlrDesc(1, b, 1, d, 8.0, lam.data_ptr(), None)
        out = torch.empty((b, 1, d), dtype=torch.bfloat16, device="cuda")
        s = [ctypes.byref(m.FhcSeq(v.data_ptr(), v.stride(0), v.stride(1))) for v in step + [out]]
        assert L.fhc_glr_forward(ctypes.byref(g), s[0], s[1], s[2], state.data_ptr(), s[3], state.data_ptr(), None,
                                 None, 0, torch.cuda.current_stream().cuda_stream) == 0
    ref, err = seqref.glr(x, r, i, lam, 8.0, h0)
    seqref.close(state, ref[1], err[1], "state after single steps")


def test_glr_gradient_against_differences():
    """The kernels' gradients along random directions against central differences of the 64-bit loss."""
    say("glr differences")
    import torch
    q = Rand(5)
    v = glr_inputs(q, 2, 90, 20, torch.float32, ragged=True)
    got = dict(zip(("x", "r", "i", "lam", "h0"), glr_check(v)[2:]))

    def loss(**change):
        w = {k: (v[k].double() + change[k] if k in change else v[k].double()) for k in ("x", "r", "i", "lam", "h0")}
        (y, ht), _ = seqref.glr(w["x"], w["r"], w["i"], w["lam"], 8.0, w["h0"], v["lengths"])
        return float((y * v["dy"].double()).sum() + (ht * v["dht"].double()).sum())

    for k, grad in got.items():
        u = q.normal(*v[k].shape).double()
        s = 1e-5
        slope = (loss(**{k: s * u}) - loss(**{k: -s * u})) / (2 * s)
        want = float((grad.double() * u).sum())
        # f32 gradients, and the third difference's s^2
        assert abs(slope - want) <= 1e-4 * float((grad.double() * u).abs().sum()), (k, slope, want)


def test_glr_long_offsets():
    """A tensor whose last rows lie past 2^31 elements."""
    say("glr long offsets")
    import torch
    b, t, d = 2, 8, 64
    far = (1 << 30) + 64
    buf = torch.zeros(2 * far + 4096, dtype=torch.float16, device="cuda")
    q = Rand(2)
    dense = q.normal(b, t, d, dtype=torch.float16)
    x = torch.as_strided(buf, (b, t, d), (2 * far, d, 1))
    x.copy_(dense)
    m = mod()
    lam = q.normal(d) - 4
    assert torch.equal(m.glr(x, dense, dense, lam)[0], m.glr(dense, dense, dense, lam)[0])
    xt = torch.as_strided(buf, (1, 3, d), (0, far, 1))
    xt.copy_(dense[:1, :3])
    assert torch.equal(m.glr(xt, dense[:1, :3], dense[:1, :3], lam)[0], m.glr(*(dense[:1, :3],) * 3, lam)[0])


@pytest.mark.parametrize("shape", [(2, 1, 64), (2, 300, 64), (40, 70, 2048)], ids=str)
def test_glr_in_a_graph_and_on_another_stream(shape):
    """Captured and replayed with other work between, every replay equals the eager call; so does a side stream."""
    say("glr graph", shape)
    import torch
    v = glr_inputs(Rand(9), *shape, torch.bfloat16)
    m = mod()

    def call(stream=None):
        y, ht, st = m.glr(v["x"], v["r"], v["i"], v["lam"], h0=v["h0"], train=True, stream=stream)
        return (y, ht) + m.glr_backward(v["x"], v["r"], v["i"], v["lam"], st, v["dy"], dht=v["dht"], stream=stream)

    want = [k.clone() for k in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = call(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        for o in out:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        call()


# ---- the norms around a block -----------------------------------------------------------------------------------

NORM = [  # rows, channels, rows per group (0: no gate)
    (1, 1, 1), (3, 5, 2), (7, 32, 7), (50, 128, 11), (33, 129, 33), (64, 257, 1), (20, 512, 20), (9, 1000, 4),
    (300, 1024, 100), (40, 1931, 40), (5, 4096, 5), (17, 8192, 3), (6, 8200, 0), (3, 16384, 2), (5000, 64, 1250),
    (2100, 40, 1), (1, 2048, 0),
]


def norm_inputs(q, rows, c, rpg, dtype):
    g = -(-rows // rpg) if rpg else 0
    return dict(x=q.normal(rows, c, dtype=dtype), o=q.normal(rows, c, scale=3.0, dtype=dtype),
                w_post=(1 + 0.1 * q.normal(c)).to(dtype), w_pre=(1 + 0.1 * q.normal(c)).to(dtype),
                gate=q.normal(g, c, scale=0.5, dtype=dtype) if rpg else None,
                dy=q.normal(rows, c, dtype=dtype), du=q.normal(rows, c, dtype=dtype))


NORM_OUT = ("y", "u", "dx", "do", "dw_post", "dgate", "dw_pre")


def norm_check(v, alpha, eps, rpg):
    m = mod()
    w = [v[k] for k in ("x", "o", "w_post", "gate", "w_pre")]
    got = m.norm_block(*w, alpha, eps, max(rpg, 1)) + m.norm_block_backward(*w, v["dy"], v["du"], alpha, eps,
                                                                          max(rpg, 1))
    ref, err = seqref.norm_block(*w, alpha, eps, max(rpg, 1), v["dy"], v["du"])
    for name, g, want, tol in zip(NORM_OUT, got, ref, err):
        if g is not None:
            seqref.close(g, want, tol, name)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", NORM, ids=str)
def test_norm_block(shape, dtype):
    say("norm", shape, dtype)
    norm_check(norm_inputs(Rand(sum(shape)), *shape, types()[dtype]), math.sqrt(0.5), 1e-6, shape[2])


def test_norm_block_parts_left_out():
    """Without the block (the first norm of a stack), without either weight, the gate, dy or du."""
    say("norm parts")
    import torch
    for gone in (("o", "w_post", "gate"), ("w_post",), ("w_pre",), ("gate",), ("dy",), ("du",), ("w_post", "w_pre", "gate")):
        v = norm_inputs(Rand(4), 37, 200, 10, torch.bfloat16)
        v.update({k: None for k in gone})
        got = dict(zip(NORM_OUT, norm_check(v, 1.0, 1e-5, 10)))
        assert all((got["d" + k] is None) == (k in gone) for k in ("w_post", "gate", "w_pre"))


def test_norm_block_zero_rows_and_empty_tensors():
    say("norm zeros")
    import torch
    m = mod()
    v = norm_inputs(Rand(6), 12, 64, 4, torch.float32)
    v["x"][3], v["o"][3], v["o"][5] = 0, 0, 0  # rms of the eps alone
    norm_check(v, 0.5, 1e-6, 4)
    e = norm_inputs(Rand(6), 0, 64, 4, torch.float32)
    w = [e[k] for k in ("x", "o", "w_post", "gate", "w_pre")]
    y, u = m.norm_block(*w, rows_per_group=4)
    assert y.shape == u.shape == (0, 64)
    back = m.norm_block_backward(*w, e["dy"], e["du"], rows_per_group=4)
    torch.cuda.synchronize()
    assert not back[2].any() and not back[4].any() and back[3].shape == (0, 64)


@pytest.mark.parametrize("c", [64, 65, 600])
def test_norm_block_views_and_in_place(c):
    """Row views of wider buffers at odd offsets; y over x, u over o; dx over dy, do over du."""
    say("norm views", c)
    import ctypes
    import torch
    m, rows = mod(), 30
    v = norm_inputs(Rand(8), rows, c, 10, torch.float16)
    w = [v[k] for k in ("x", "o", "w_post", "gate", "w_pre")]
    y, u = m.norm_block(*w, rows_per_group=10)
    grads = m.norm_block_backward(*w, v["dy"], v["du"], rows_per_group=10)
    wide = {k: torch.full((rows, c + 19), 7.0, dtype=torch.float16, device="cuda") for k in ("x", "o", "dy", "du")}
    views = {k: b[:, 3:3 + c] for k, b in wide.items()}
    for k, b in views.items():
        b.copy_(v[k])
    n = m.NormDesc(0, rows, c, 10, 1.0, 1e-6, v["w_post"].data_ptr(), v["w_pre"].data_ptr(), v["gate"].data_ptr())
    at = {k: ctypes.byref(m.FhcRows(b.data_ptr(), b.stride(0))) for k, b in views.items()}
    L, s = m._lib(), torch.cuda.current_stream().cuda_stream
    size = L.fhc_norm_block_workspace_bytes(ctypes.byref(n))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert L.fhc_norm_block_backward(ctypes.byref(n), at["x"], at["o"], at["dy"], at["du"], at["dy"], at["du"], None,
                                     None, None, ws.data_ptr(), size, s) == 0
    assert L.fhc_norm_block(ctypes.byref(n), at["x"], at["o"], at["x"], at["o"], s) == 0
    torch.cuda.synchronize()
    for got, want in ((views["x"], y), (views["o"], u), (views["dy"], grads[0]), (views["du"], grads[1])):
        assert torch.equal(got, want)
    for b in wide.values():
        assert (b[:, :3] == 7).all() and (b[:, 3 + c:] == 7).all()


def test_norm_block_gradient_against_differences():
    say("norm differences")
    import torch
    q = Rand(12)
    v = norm_inputs(q, 24, 48, 7, torch.float32)
    got = dict(zip(("x", "o", "w_post", "gate", "w_pre"), norm_check(v, 0.7, 1e-6, 7)[2:]))

    def loss(**change):
        w = [v[k].double() + change.get(k, 0) for k in ("x", "o", "w_post", "gate", "w_pre")]
        (y, u), _ = seqref.norm_block(*w, 0.7, 1e-6, 7)
        return float((y * v["dy"].double()).sum() + (u * v["du"].double()).sum())

    for k, grad in got.items():
        d = q.normal(*v[k].shape).double()
        s = 1e-5
        slope = (loss(**{k: s * d}) - loss(**{k: -s * d})) / (2 * s)
        want = float((grad.double() * d).sum())
        assert abs(slope - want) <= 1e-4 * float((grad.double() * d).abs().sum()), (k, slope, want)


def test_norm_block_in_a_graph():
    say("norm graph")
    import torch
    m = mod()
    v = norm_inputs(Rand(13), 500, 300, 125, torch.bfloat16)
    w = [v[k] for k in ("x", "o", "w_post", "gate", "w_pre")]

    def call():
        return m.norm_block(*w, rows_per_group=125) + m.norm_block_backward(*w, v["dy"], v["du"], rows_per_group=125)

    want = [k.clone() for k in call()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        for o in out:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        call()


# ---- the gated feed-forward block -------------------------------------------------------------------------------

FFN = [  # rows, c, f: few rows (each width of the streaming product) and tiles; widths odd, even, cut in a group of 8
    (1, 1, 1), (1, 64, 128), (3, 40, 72), (16, 128, 100), (17, 96, 130), (33, 256, 512), (64, 130, 62), (65, 64, 64),
    (128, 128, 128), (130, 257, 129), (200, 100, 300), (257, 72, 514), (1000, 128, 512), (300, 512, 1030),
    (700, 33, 65), (5000, 64, 96), (4100, 512, 1024), (2049, 1024, 2050),
]


def ffn_inputs(q, rows, c, f, dtype):
    return dict(x=q.normal(rows, c, dtype=dtype), wg=q.normal(f, c, scale=c ** -0.5, dtype=dtype),
                wu=q.normal(f, c, scale=c ** -0.5, dtype=dtype), wd=q.normal(c, f, scale=f ** -0.5, dtype=dtype),
                dy=q.normal(rows, c, dtype=dtype))


FFN_OUT = ("y", "dx", "dwg", "dwu", "dwd")


def ffn_check(v, act):
    m = mod()
    w = [v[k] for k in ("x", "wg", "wu", "wd")]
    serve = m.ffn(*w, act)
    y, saved = m.ffn(*w, act, train=True)
    got = (y,) + m.ffn_backward(*w, saved, v["dy"], act)
    ref, err = seqref.ffn(*w, act, v["dy"])
    seqref.close(serve, ref[0], err[0], "y without states kept")
    for name, g, want, tol in zip(FFN_OUT, got, ref, err):
        seqref.close(g, want, tol, name)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", FFN, ids=str)
def test_ffn(shape, dtype):
    say("ffn", shape, dtype)
    ffn_check(ffn_inputs(Rand(sum(shape)), *shape, types()[dtype]), "silu" if shape[0] % 2 else "gelu")


def test_ffn_what_lies_beside_a_row_is_not_read():
    """Row views whose neighbours are NaN, widths cut inside a group of 8, outputs in wider buffers."""
    say("ffn views")
    import ctypes
    import torch
    m = mod()
    for rows, c, f, off in ((40, 36, 44, 8), (40, 36, 44, 1), (150, 36, 44, 2), (150, 35, 43, 3), (300, 100, 92, 4)):
        v = ffn_inputs(Rand(rows + off), rows, c, f, torch.bfloat16)
        want = m.ffn(v["x"], v["wg"], v["wu"], v["wd"])
        y, saved = m.ffn(v["x"], v["wg"], v["wu"], v["wd"], train=True)
        grads = m.ffn_backward(v["x"], v["wg"], v["wu"], v["wd"], saved, v["dy"])
        wide = {k: torch.full((rows, c + 20), math.nan, dtype=torch.bfloat16, device="cuda") for k in ("x", "dy")}
        views = {k: b[:, off:off + c] for k, b in wide.items()}
        for k, b in views.items():
            b.copy_(v[k])
        # weights with NaN right behind them
        pool = {k: torch.full((v[k].numel() + 64,), math.nan, dtype=torch.bfloat16, device="cuda")
                for k in ("wg", "wu", "wd")}
        w = []
        for k, b in pool.items():
            b[:v[k].numel()] = v[k].flatten()
            w.append(b[:v[k].numel()].view(v[k].shape))
        assert torch.equal(m.ffn(views["x"], *w), want)
        y2, saved2 = m.ffn(views["x"], *w, train=True)
        assert torch.equal(y2, y)
        got = m.ffn_backward(views["x"], *w, saved2, views["dy"])
        for name, a, b in zip(FFN_OUT[1:], got, grads):
            assert torch.equal(a, b), (rows, c, f, off, name)
        out = torch.full((rows, c + 20), 7.0, dtype=torch.bfloat16, device="cuda")
        d = m.FfnDesc(1, 0, rows, c, f)
        L = m._lib()
        n = L.fhc_ffn_workspace_bytes(ctypes.byref(d), 0)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        o = out[:, off:off + c]
        assert L.fhc_ffn_forward(ctypes.byref(d), m._rows("", "", views["x"]), w[0].data_ptr(), w[1].data_ptr(),
                                 w[2].data_ptr(), m._rows("", "", o), None, ws.data_ptr(), n,
                                 torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(o, want) and (out[:, :off] == 7).all() and (out[:, off + c:] == 7).all()


def test_ffn_empty_sides():
    say("ffn empty")
    import torch
    m = mod()
    for rows, c, f in ((0, 8, 16), (5, 8, 0), (200, 8, 0), (0, 8, 0)):
        v = ffn_inputs(Rand(1), rows, max(c, 1), max(f, 1), torch.float16)
        w = [v["wg"][:f].contiguous(), v["wu"][:f].contiguous(), v["wd"][:, :f].contiguous()]
        y, saved = m.ffn(v["x"], *w, train=True)
        grads = m.ffn_backward(v["x"], *w, saved, v["dy"])
        torch.cuda.synchronize()
        assert y.shape == (rows, c) and not y.any() and not any(g.any() for g in grads)


def test_ffn_values_that_are_not_finite_stay_in_their_rows():
    say("ffn not finite")
    import torch
    m = mod()
    for rows in (20, 300):
        v = ffn_inputs(Rand(3), rows, 72, 136, torch.bfloat16)
        clean = m.ffn(v["x"], v["wg"], v["wu"], v["wd"])
        v["x"][7, 3], v["x"][11, 70] = math.nan, math.inf
        got = m.ffn(v["x"], v["wg"], v["wu"], v["wd"])
        assert not torch.isfinite(got[7]).any() and not torch.isfinite(got[11]).all()
        keep = [r for r in range(rows) if r not in (7, 11)]
        assert torch.equal(got[keep], clean[keep])


def test_ffn_activation_at_its_ends():
    """Pre-activations far outside exp's range: act is 0 on one side and the identity on the other."""
    say("ffn ends")
    import torch
    m = mod()
    for act in ("silu", "gelu"):
        x = torch.tensor([[1.0], [-1.0]], dtype=torch.bfloat16, device="cuda").repeat(70, 1)
        wg = torch.tensor([[300.0], [2.0 ** 30]], dtype=torch.bfloat16, device="cuda")
        one = torch.ones_like(wg)
        y, saved = m.ffn(x, wg, one, one.t().contiguous(), act, train=True)
        grads = m.ffn_backward(x, wg, one, one.t().contiguous(), saved, torch.ones_like(x), act)
        assert torch.equal(y[0], (wg.float().sum()).to(torch.bfloat16)[None]) and not y[1].any()
        assert all(torch.isfinite(g).all() for g in grads)


def test_ffn_gradient_against_differences():
    say("ffn differences")
    import torch
    q = Rand(14)
    for act in ("silu", "gelu"):
        v = ffn_inputs(q, 90, 40, 56, torch.float16)
        got = dict(zip(("x", "wg", "wu", "wd"), ffn_check(v, act)[1:]))

        def loss(**change):
            w = [v[k].double() + change.get(k, 0) for k in ("x", "wg", "wu", "wd")]
            h = seqref._act(w[0] @ w[1].t(), act)[0] * (w[0] @ w[2].t())
            return float(((h @ w[3].t()) * v["dy"].double()).sum())

        for k, grad in got.items():
            d = q.normal(*v[k].shape).double()
            s = 1e-5
            slope = (loss(**{k: s * d}) - loss(**{k: -s * d})) / (2 * s)
            want = float((grad.double() * d).sum())
            # f16 gradients: two roundings each
            assert abs(slope - want) <= 2 ** -10 * float((grad.double() * d).abs().sum()), (act, k, slope, want)


@pytest.mark.parametrize("shape", [(8, 128, 256), (300, 128, 256)], ids=str)
def test_ffn_in_a_graph_and_on_another_stream(shape):
    say("ffn graph", shape)
    import torch
    m = mod()
    v = ffn_inputs(Rand(15), *shape, torch.bfloat16)
    w = [v[k] for k in ("x", "wg", "wu", "wd")]

    def call(stream=None):
        serve = m.ffn(*w, stream=stream)
        y, saved = m.ffn(*w, train=True, stream=stream)
        return (serve, y) + m.ffn_backward(*w, saved, v["dy"], stream=stream)

    want = [k.clone() for k in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = call(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        for o in out:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        call()


# few channels and many rows: the one-kernel form; widths short of and past each of its sizes, tails of rows and features
FFN_FUSED = [(8192, 64, 128), (8200, 128, 512), (8193, 256, 100), (9000, 100, 90), (8192, 65, 129), (8500, 200, 264),
             (8192, 7, 33), (20001, 129, 31)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", FFN_FUSED, ids=str)
def test_ffn_many_rows_of_few_channels(shape, dtype):
    say("ffn fused", shape, dtype)
    ffn_check(ffn_inputs(Rand(sum(shape)), *shape, types()[dtype]), "silu" if shape[0] % 2 else "gelu")


def test_ffn_many_rows_some_gradients_only_views_and_rows_not_finite():
    """dx or the weights' gradients alone are those of the whole call; row views with NaN beside them; a row of NaN."""
    say("ffn fused parts")
    import ctypes
    import torch
    m, (rows, c, f) = mod(), (8195, 72, 136)
    v = ffn_inputs(Rand(21), rows, c, f, torch.bfloat16)
    w = [v[k] for k in ("wg", "wu", "wd")]
    y, saved = m.ffn(v["x"], *w, train=True)
    grads = m.ffn_backward(v["x"], *w, saved, v["dy"])
    wide = {k: torch.full((rows, c + 20), math.nan, dtype=torch.bfloat16, device="cuda") for k in ("x", "dy")}
    for off in (1, 2, 8):
        views = {k: b[:, off:off + c] for k, b in wide.items()}
        for k, b in views.items():
            b.copy_(v[k])
        assert torch.equal(m.ffn(views["x"], *w), y)
        assert all(torch.equal(a, b) for a, b in zip(m.ffn_backward(views["x"], *w, saved, views["dy"]), grads))
        for b in wide.values():
            b.fill_(math.nan)
    L, d = m._lib(), m.FfnDesc(1, 0, rows, c, f)
    n = L.fhc_ffn_workspace_bytes(ctypes.byref(d), 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    for only in range(4):
        out = [torch.full_like(g, 7) for g in grads]
        at = [o.data_ptr() if k == only else None for k, o in enumerate(out)]
        assert L.fhc_ffn_backward(ctypes.byref(d), m._rows("", "", v["x"]), w[0].data_ptr(), w[1].data_ptr(),
                                  w[2].data_ptr(), saved.data_ptr(), m._rows("", "", v["dy"]),
                                  m._rows("", "", out[0]) if only == 0 else None, at[1], at[2], at[3], ws.data_ptr(), n,
                                  torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[only], grads[only]), only
        assert all((o == 7).all() for k, o in enumerate(out) if k != only)
    v["x"][100, 3] = math.nan
    got = m.ffn(v["x"], *w)
    keep = torch.arange(rows, device="cuda") != 100
    assert torch.equal(got[keep], y[keep]) and not torch.isfinite(got[100]).any()


def test_ffn_many_rows_in_a_graph():
    say("ffn fused graph")
    import torch
    m = mod()
    v = ffn_inputs(Rand(22), 8192, 128, 96, torch.float16)
    w = [v[k] for k in ("x", "wg", "wu", "wd")]

    def call():
        y, saved = m.ffn(*w, train=True)
        return (y,) + m.ffn_backward(*w, saved, v["dy"])

    want = [k.clone() for k in call()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        for o in out:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        call()


# on either side of where the one-kernel form is taken, with and without states kept
@pytest.mark.parametrize("shape", [(5999, 64, 96), (6000, 64, 96), (11499, 128, 70), (11500, 128, 72), (12003, 100, 520),
                                   (19501, 200, 136), (23003, 72, 40), (22001, 256, 65)], ids=str)
def test_ffn_where_the_form_changes(shape):
    say("ffn forms", shape)
    for k, dtype in enumerate(("f16", "bf16")):
        ffn_check(ffn_inputs(Rand(sum(shape)), *shape, types()[dtype]), "gelu" if k else "silu")


def test_ffn_in_one_kernel_some_gradients_only_views_and_graph():
    """As for fewer rows: dx or the weights' gradients alone, row views with NaN beside them, replays of a graph."""
    say("ffn one kernel parts")
    import ctypes
    import torch
    m, (rows, c, f) = mod(), (11523, 72, 136)
    v = ffn_inputs(Rand(31), rows, c, f, torch.bfloat16)
    w = [v[k] for k in ("wg", "wu", "wd")]

    def call():
        y, saved = m.ffn(v["x"], *w, train=True)
        return (y,) + m.ffn_backward(v["x"], *w, saved, v["dy"])

    y, saved = m.ffn(v["x"], *w, train=True)
    want = [k.clone() for k in call()]
    wide = {k: torch.full((rows, c + 20), math.nan, dtype=torch.bfloat16, device="cuda") for k in ("x", "dy")}
    for off in (1, 2, 8):
        views = {k: b[:, off:off + c] for k, b in wide.items()}
        for k, b in views.items():
            b.copy_(v[k])
        y2, saved2 = m.ffn(views["x"], *w, train=True)
        got = (y2,) + m.ffn_backward(views["x"], *w, saved2, views["dy"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for b in wide.values():
            b.fill_(math.nan)
    L, d = m._lib(), m.FfnDesc(1, 0, rows, c, f)
    n = L.fhc_ffn_workspace_bytes(ctypes.byref(d), 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    for only in range(4):
        out = [torch.full_like(g, 7) for g in want[1:]]
        at = [o.data_ptr() if k == only else None for k, o in enumerate(out)]
        assert L.fhc_ffn_backward(ctypes.byref(d), m._rows("", "", v["x"]), w[0].data_ptr(), w[1].data_ptr(),
                                  w[2].data_ptr(), saved.data_ptr(), m._rows("", "", v["dy"]),
                                  m._rows("", "", out[0]) if only == 0 else None, at[1], at[2], at[3], ws.data_ptr(), n,
                                  torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[only], want[1 + only]), only
        assert all((o == 7).all() for k, o in enumerate(out) if k != only)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        for o in out:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        call()


@pytest.mark.parametrize("shape", [(40, 20, 52), (300, 132, 78), (33, 1020, 34), (129, 6, 10), (70, 35, 51)])
def test_ffn_views_that_end_with_their_buffer(shape):
    """x and dy are the last columns of rows of up8(c) elements, so the last row's last element is their buffer's last:
    every gradient equals the dense call's."""
    rows, c, f = shape
    say("ffn views to the end", shape)
    import torch
    m = mod()
    v = ffn_inputs(Rand(11), rows, c, f, torch.bfloat16)
    w = [v[k] for k in ("wg", "wu", "wd")]

    def call(x, dy):
        y, saved = m.ffn(x, *w, train=True)
        return (y,) + m.ffn_backward(x, *w, saved, dy)

    want = call(v["x"], v["dy"])
    ld = (c + 7) // 8 * 8
    views = []
    for k in ("x", "dy"):
        b = torch.full((rows, ld), math.nan, dtype=torch.bfloat16, device="cuda")
        b[:, ld - c:].copy_(v[k])
        views.append(b[:, ld - c:])
    assert all(torch.equal(a, b) for a, b in zip(call(*views), want))


@pytest.mark.parametrize("c", [13, 131, 261, 523, 1931])
def test_norm_block_infinite_gate_stays_in_its_channel(c):
    """An infinite gate on one of the last 8 channels, which at odd widths are read twice: y is infinite there alone, u
    there not a number and 0 elsewhere (a finite y over an infinite mean)."""
    say("norm infinite gate", c)
    import torch
    m, q = mod(), Rand(c)
    x, o = q.normal(5, c, dtype=torch.float16), q.normal(5, c, dtype=torch.float16)
    one = torch.ones(c, dtype=torch.float16, device="cuda")
    for at in range(c - 8, c):
        gate = torch.ones(1, c, dtype=torch.float16, device="cuda")
        gate[0, at] = math.inf
        y, u = m.norm_block(x, o.abs() + 1, one, gate, one, rows_per_group=5)
        others = torch.arange(c, device="cuda") != at
        assert torch.isinf(y[:, at]).all() and torch.isfinite(y[:, others]).all(), at
        assert torch.isnan(u[:, at]).all() and (u[:, others] == 0).all(), at


def test_norm_block_more_rows_than_a_launch_has():
    """2^28 rows of one channel are three launches: each row still finds its group's gate. o / rms(o) is 1 for o = 1."""
    say("norm many rows")
    import torch
    m, rows, rpg = mod(), (1 << 28) + 37, (1 << 26) + 5
    o = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    x = torch.zeros_like(o)
    gate = torch.tensor([[2.0], [-3.0], [4.0], [-5.0], [6.0]], dtype=torch.float16, device="cuda")
    y, u = m.norm_block(x, o, None, gate, None, rows_per_group=rpg)
    for k in range(5):
        part = slice(k * rpg, min((k + 1) * rpg, rows))
        # f32 statistics: off by a few 1e-7, and 1e-6 / 2 for eps, then rounded to f16 (the values are whole: no change)
        assert (y[part] == gate[k]).all(), k
        assert (u[part] == gate[k].sign()).all(), k


@pytest.mark.parametrize("shape", [(4, 1, 48), (3, 9, 1532), (5, 40, 100), (3, 300, 48), (70, 130, 100), (7, 20, 33)],
                         ids=str)
def test_glr_sequences_that_share_their_elements(shape):
    """Inputs that are one and the same for every sequence, or overlap from one to the next, give what their copies
    give: forward, one step and backward, in each argument by itself and in all of them."""
    say("glr shared", shape)
    import torch
    b, t, d = shape
    q, m = Rand(sum(shape)), mod()
    for dtype in (torch.bfloat16, torch.float32):
        lam, h0, dht = q.normal(d) - 4, q.normal(b, d), q.normal(b, d)
        dense = [q.normal(b, t, d, dtype=dtype) for _ in range(4)]
        half = d // 2
        width = (b - 1) * half + d
        for form in ("one", "overlapping"):
            if form == "one":
                shared = [q.normal(1, t, d, dtype=dtype).expand(b, t, d) for _ in range(4)]
            else:
                shared = [torch.as_strided(q.normal(t, width, dtype=dtype), (b, t, d), (half, width, 1)) for _ in range(4)]
            for which in ((0,), (1,), (2,), (3,), (0, 1, 2, 3)):
                say(dtype, form, which)
                v = [shared[k] if k in which else dense[k] for k in range(4)]
                got, want = [], []
                for out, (x, r, i, dy) in ((got, v), (want, [k.contiguous() for k in v])):
                    y, ht, states = m.glr(x, r, i, lam, h0=h0, train=True)
                    out += [y, ht, *m.glr_backward(x, r, i, lam, states, dy, dht=dht)]
                assert all(torch.equal(a, w) for a, w in zip(got, want)), (form, which)


@pytest.mark.parametrize("rows", [20, 140, 8192])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_ffn_slope_far_from_zero(act, rows):
    """Pre-activations whose cube leaves f32's range: act's slope is 1 on one side and 0 on the other. Every value is a
    power of two, or a number of rows times one, so the results are the formula's exactly."""
    say("ffn slope", act, rows)
    import torch
    m, n = mod(), rows // 2
    x = torch.tensor([[1.0], [-1.0]], dtype=torch.bfloat16, device="cuda").repeat(n, 1)
    wg = torch.tensor([[2.0 ** 44], [2.0 ** 70]], dtype=torch.bfloat16, device="cuda")
    one = torch.ones_like(wg)
    y, saved = m.ffn(x, wg, one, one.t().contiguous(), act, train=True)
    dx, dwg, dwu, dwd = m.ffn_backward(x, wg, one, one.t().contiguous(), saved, torch.ones_like(x), act)
    total = wg.double().sum()
    for got, want in ((y, total), (dx, 2 * total)):  # dL/dgate = slope, dL/dup = act = wg; of x = -1 both are 0
        assert (got[::2] == want.to(torch.bfloat16)).all() and not got[1::2].any()
    assert (dwg == n).all()
    assert torch.equal(dwu, (wg.double() * n).to(torch.bfloat16)) and torch.equal(dwd, dwu.t())


@pytest.mark.parametrize("c,f", [(300, 520), (1024, 2048)])
def test_ffn_of_an_empty_batch_and_a_wide_hidden_layer(c, f):
    say("ffn empty batch", c, f)
    import torch
    m = mod()
    v = ffn_inputs(Rand(1), 0, c, f, torch.bfloat16)
    w = [v[k] for k in ("x", "wg", "wu", "wd")]
    y, saved = m.ffn(*w, train=True)
    dx, *grads = m.ffn_backward(*w, saved, v["dy"])
    torch.cuda.synchronize()
    assert m.ffn(*w).shape == y.shape == dx.shape == (0, c) and not any(g.any() for g in grads)


@pytest.mark.parametrize("c,f", [(16, 24), (33, 17), (300, 520)])
def test_ffn_backward_without_rows(c, f):
    """The weights' gradients of no rows are 0, whatever the descriptors of x and dy hold."""
    say("ffn no rows", c, f)
    import ctypes
    import torch
    m = mod()
    L, d = m._lib(), m.FfnDesc(1, 0, 0, c, f)
    n = L.fhc_ffn_workspace_bytes(ctypes.byref(d), 1)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    v = ffn_inputs(Rand(1), 1, c, f, torch.bfloat16)
    w = [v[k].data_ptr() for k in ("wg", "wu", "wd")]
    for rows in (None, m.FhcRows(None, 0), m.FhcRows(None, c)):
        out = [torch.full_like(v[k], 7) for k in ("wg", "wu", "wd")]
        assert L.fhc_ffn_backward(ctypes.byref(d), rows, *w, None, rows, rows, *(o.data_ptr() for o in out),
                                  ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert not any(o.any() for o in out), rows


def test_glr_outputs_of_overlapping_windows():
    """Inputs that overlap have no order in memory of their own to give to the outputs: windows that move by one element
    from step to step or from sequence to sequence give what their copies give."""
    say("glr windows")
    import torch
    q, m = Rand(17), mod()
    b, t, d = 3, 5, 12
    lam, dy = q.normal(d) - 4, q.normal(b, t, d)
    r, i = q.normal(b, t, d), q.normal(b, t, d)
    for strides in ((t + d - 1, 1, 1), (1, d + b - 1, 1), (1, 1, 1)):
        say(strides)
        win = torch.as_strided(q.normal(200), (b, t, d), strides)
        for x, rr, ii in ((win, r, i), (r, win, win)):
            got, want = [], []
            for out, (a, e, f) in ((got, (x, rr, ii)), (want, [v.contiguous() for v in (x, rr, ii)])):
                y, ht, states = m.glr(a, e, f, lam, train=True)
                out += [y, ht, *m.glr_backward(a, e, f, lam, states, dy)]
            assert all(torch.equal(a, w) for a, w in zip(got, want)), strides


@pytest.mark.parametrize("eps", [2.0 ** -126, 2.0 ** -127, 2.0 ** -130, 2.0 ** -140])
@pytest.mark.parametrize("c", [40, 300])
def test_norm_block_of_zeros_under_a_subnormal_eps(c, eps):
    """Rows of zeros: of the block's output, or of the residual stream without one. 1 / rms is 2^63 to 2^70 there."""
    say("norm subnormal eps", c, eps)
    import torch
    v = norm_inputs(Rand(c), 12, c, 4, torch.float32)
    v["o"][3], v["o"][8] = 0, 0
    norm_check(v, 0.5, eps, 4)
    v.update(o=None, w_post=None, gate=None)
    v["x"][5], v["x"][11] = 0, 0
    norm_check(v, 0.5, eps, 4)


def test_glr_backward_over_more_channels_than_a_launch_of_sums_takes():
    """dlam of sequences that are one and the same is that of one times their number (the sum is in f64)."""
    say("glr wide sums")
    import torch
    m, q = mod(), Rand(29)
    for b, d in ((520, (1 << 20) + 48), (1, (1 << 26) + 24)):
        say(b, d)
        x, r, i, dy = (q.normal(1, 1, d, dtype=torch.float16) for _ in range(4))
        lam = q.normal(d) - 4
        one = [v.expand(b, 1, d) for v in (x, r, i, dy)]
        y, _, states = m.glr(*one[:3], lam, train=True)
        dlam = m.glr_backward(*one[:3], lam, states, one[3])[3]
        del y, states
        for part in (slice(0, 500), slice(d // 2, d // 2 + 500), slice(d - 500, d)):
            ref, err = seqref.glr(*(v[:, :, part] for v in (x, r, i)), lam[part], 8.0, dy=dy[:, :, part])
            seqref.close(dlam[part], b * ref[5], b * err[5], "dlam")


@pytest.mark.parametrize("shape", [(20, 37, 51), (300, 37, 51), (700, 132, 1030), (6003, 37, 51), (11501, 101, 70),
                                   (19501, 131, 33)], ids=str)
def test_ffn_stays_in_its_workspace(shape):
    """Widths and addresses that make a call copy every operand: what lies behind the workspace, the kept states and the
    outputs stays as it was."""
    rows, c, f = shape
    say("ffn workspace", shape)
    import ctypes
    import torch
    m = mod()
    L, d = m._lib(), m.FfnDesc(1, 1, rows, c, f)
    v = ffn_inputs(Rand(33), rows, c, f, torch.bfloat16)
    at = {}
    for k in ("x", "wg", "wu", "wd", "dy"):  # at odd elements
        b = torch.empty(v[k].numel() + 1, dtype=torch.bfloat16, device="cuda")
        b[1:] = v[k].flatten()
        at[k] = b[1:].view(v[k].shape)
    stream = torch.cuda.current_stream().cuda_stream

    def room(n):
        return torch.full((n + 8192,), 0x5A, dtype=torch.uint8, device="cuda")

    sizes = (L.fhc_ffn_saved_bytes(ctypes.byref(d)), L.fhc_ffn_workspace_bytes(ctypes.byref(d), 0),
             L.fhc_ffn_workspace_bytes(ctypes.byref(d), 1), rows * c * 2, rows * c * 2, f * c * 2, f * c * 2, f * c * 2)
    bufs = [room(n) for n in sizes]
    saved, ws, wsb, y, dx, dwg, dwu, dwd = (b.data_ptr() for b in bufs)
    w = [at[k].data_ptr() for k in ("wg", "wu", "wd")]
    x, dy, yr, dxr = (m._ROWS(p, c) for p in (at["x"].data_ptr(), at["dy"].data_ptr(), y, dx))
    assert L.fhc_ffn_forward(ctypes.byref(d), x, *w, yr, saved, ws, sizes[1], stream) == 0
    assert L.fhc_ffn_backward(ctypes.byref(d), x, *w, saved, dy, dxr, dwg, dwu, dwd, wsb, sizes[2], stream) == 0
    torch.cuda.synchronize()
    for b, n in zip(bufs, sizes):
        assert (b[n:] == 0x5A).all()
    want, err = seqref.ffn(*(at[k] for k in ("x", "wg", "wu", "wd")), "gelu", at["dy"])
    for name, b, n, r, e in zip(FFN_OUT, bufs[3:], sizes[3:], want, err):
        seqref.close(b[:n].view(torch.bfloat16).view(r.shape), r, e, name)


# ---- paths that only larger calls take --------------------------------------------------------------------------

# one run of chained chunks is 8192 steps forward and 4096 backward: into the second run, the third and the fifth
@pytest.mark.parametrize("shape", [(1, 8400, 34), (2, 8193, 3), (2, 16500, 3)], ids=str)
def test_glr_of_several_runs(shape):
    say("glr runs", shape)
    for dtype, ragged in (("f16", False), ("f32", True)):
        glr_check(glr_inputs(Rand(sum(shape)), *shape, types()[dtype], ragged=ragged))


# a workgroup that takes several short groups one after the other: one row a group, two, three; wide rows and narrow ones
@pytest.mark.parametrize("shape", [(600, 8192, 1), (2500, 2048, 2), (3100, 2040, 3), (13000, 40, 1), (26000, 24, 2)],
                         ids=str)
def test_norm_block_of_many_short_groups(shape):
    say("norm short groups", shape)
    for dtype in ("bf16", "f32"):
        norm_check(norm_inputs(Rand(sum(shape)), *shape, types()[dtype]), math.sqrt(0.5), 1e-6, shape[2])


def ffn_tile(m, n, pairs=1, glu=False):
    """The tile that a product of many slabs takes: 0 narrow, 1 medium, 2 large (the rule of ffn_kernels.hip)."""
    def rounds(bm, bn):
        return -(-(-(-m // bm) * -(-n // (bn // (2 if glu else 1))) * pairs) // 256)

    time = [rounds(128, 64) * 75, rounds(128, 128) * 100, rounds(256, 256) * 270]
    return time.index(min(time))


@pytest.mark.parametrize("shape", [(3301, 3275, 3283), (3298, 3276, 3282)], ids=str)
def test_ffn_large_tiles_with_remainders(shape):
    """Every product of a step in the largest tile: rows and columns of either operand, cut in a tile and in a slab."""
    rows, c, f = shape
    say("ffn large tiles", shape)
    tiles = (ffn_tile(rows, f, glu=True), ffn_tile(rows, c), ffn_tile(rows, f), ffn_tile(rows, c), ffn_tile(f, c, 2),
             ffn_tile(c, f))
    assert all(t == 2 for t in tiles), tiles
    for k, dtype in enumerate(("f16", "bf16")):
        ffn_check(ffn_inputs(Rand(sum(shape)), *shape, types()[dtype]), "gelu" if k else "silu")


# the one-kernel form at each of its register sizes, short of them and full, with tails of rows and features
@pytest.mark.parametrize("shape", [(6001, 7, 33), (6130, 64, 31), (11600, 65, 129), (11777, 128, 100), (19600, 129, 31),
                                   (20001, 256, 100)], ids=str)
def test_ffn_in_one_kernel_at_its_edges(shape):
    say("ffn one kernel", shape)
    for k, dtype in enumerate(("f16", "bf16")):
        ffn_check(ffn_inputs(Rand(sum(shape)), *shape, types()[dtype]), "silu" if k else "gelu")


@pytest.mark.parametrize("shape", [(6003, 40, 64), (11523, 72, 136), (19523, 200, 70)], ids=str)
def test_ffn_in_one_kernel_values_that_are_not_finite_stay_in_their_rows(shape):
    """Forward and dx: a row of x that holds a NaN or an infinity, and one of dy, reach their own rows only."""
    rows, c, f = shape
    say("ffn one kernel not finite", shape)
    import torch
    m = mod()
    v = ffn_inputs(Rand(23), rows, c, f, torch.bfloat16)
    w = [v[k] for k in ("wg", "wu", "wd")]
    y, saved = m.ffn(v["x"], *w, train=True)
    dx = m.ffn_backward(v["x"], *w, saved, v["dy"])[0]
    v["x"][100, 3], v["x"][5000, c - 1], v["dy"][4321, 0] = math.nan, math.inf, math.nan
    y2, saved2 = m.ffn(v["x"], *w, train=True)
    dx2 = m.ffn_backward(v["x"], *w, saved2, v["dy"])[0]
    at = torch.arange(rows, device="cuda")
    whole = (at != 100) & (at != 5000)
    assert torch.equal(y2[whole], y[whole]) and not torch.isfinite(y2[100]).any()
    whole &= at != 4321
    assert torch.equal(dx2[whole], dx[whole]) and not torch.isfinite(dx2[100]).any()
    assert not torch.isfinite(dx2[4321]).any() and torch.equal(y2[4321], y[4321])
