"""The short convolution, the selective state space scan and the product with its epilogue (through fhseq.py and the C
ABI, include/fhc_seq.h) against plain 64-bit forms, on the GPU. The tolerances are the forms' own error bounds
(tests/ssmref.py) plus half a step of each output's type."""
import ctypes
import math

import pytest

import fhtest  # noqa: F401  (puts the package on sys.path)
import seqref
import ssmref
from test_seq_gpu import Rand, mod, say, types

pytestmark = pytest.mark.gpu


def seqs(q, time_major):
    """Draws sequence tensors, in either order of batch and time in memory."""
    def seq(b, t, d, dtype, scale=1.0):
        if time_major:
            return q.normal(t, b, d, scale=scale, dtype=dtype).transpose(0, 1)
        return q.normal(b, t, d, scale=scale, dtype=dtype)
    return seq


def lengths_of(q, b, t, ragged):
    if not ragged:
        return None
    n = q.ints(0, t + 1, b)
    n[-1] = 0
    n[0] = t
    return n


def compare(names, got, ref, err):
    assert len(got) == len(ref) == len(names)
    for name, g, r, e in zip(names, got, ref, err):
        assert (g is None) == (r is None), name
        if g is not None:
            assert g.shape == r.shape, (name, g.shape, r.shape)
            seqref.close(g, r, e, name)


# ---- the short convolution ----------------------------------------------------------------------------------------

CONV = [  # b, t, d, k: one step; fewer steps than taps; less and more than a chunk; odd and narrow widths; many sequences
    (1, 1, 1, 2), (64, 1, 96, 4), (3, 2, 7, 4), (2, 3, 8, 4), (2, 8, 130, 3), (1, 33, 33, 2), (3, 65, 34, 4),
    (2, 200, 1931, 3), (70, 130, 40, 4), (300, 24, 128, 4), (4, 1000, 513, 2), (1, 5000, 3, 4),
]
CONV_NAMES = ("y", "state", "dx", "dw", "dbias", "dstate")


def conv_inputs(q, b, t, d, k, dtype, time_major=False, ragged=False):
    seq = seqs(q, time_major)
    return dict(x=seq(b, t, d, dtype), w=q.normal(d, k, scale=k ** -0.5, dtype=dtype), bias=q.normal(d, dtype=dtype),
                state=q.normal(b, k - 1, d, dtype=dtype), lengths=lengths_of(q, b, t, ragged), dy=seq(b, t, d, dtype),
                dstate=q.normal(b, k - 1, d, dtype=dtype))


def conv_run(v, act="silu"):
    m = mod()
    out = m.short_conv(v["x"], v["w"], v["bias"], act, state=v["state"], lengths=v["lengths"])
    return out + m.short_conv_backward(v["x"], v["w"], v["bias"], v["dy"], act, state=v["state"], dstate=v["dstate"],
                                       lengths=v["lengths"])


def conv_check(v, act="silu"):
    got = conv_run(v, act)
    ref, err = ssmref.short_conv(v["x"], v["w"], v["bias"], act, v["state"], v["lengths"], v["dy"], v["dstate"])
    compare(CONV_NAMES, got, ref, err)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", CONV, ids=str)
def test_short_conv(shape, dtype):
    say("short_conv", shape, dtype)
    q = Rand(sum(shape))
    conv_check(conv_inputs(q, *shape, types()[dtype], time_major=shape[2] % 3 == 0, ragged=shape[1] % 2 == 1),
               "none" if shape[3] == 2 else "silu")


def test_short_conv_parts_left_out():
    say("short_conv parts left out")
    import torch
    q = Rand(5)
    v = conv_inputs(q, 3, 21, 40, 4, torch.bfloat16)
    for gone in (("bias",), ("state",), ("dstate",), ("bias", "state", "dstate")):
        conv_check({k: None if k in gone else x for k, x in v.items()})


@pytest.mark.parametrize("shape", [(4, 9, 10, 4), (3, 131, 64, 3)], ids=str)
def test_short_conv_masked_places_are_not_read(shape):
    """NaN and infinities past the lengths, empty sequences, lengths outside [0, t]."""
    say("short_conv masked", shape)
    import torch
    q = Rand(7)
    v = conv_inputs(q, *shape, torch.float16, ragged=True)
    v["lengths"][1], v["lengths"][2] = shape[1] + 1000, -3
    past = torch.arange(shape[1], device="cuda")[None] >= v["lengths"][:, None]
    clean = conv_check(v)
    v["x"], v["dy"] = (v[k].masked_fill(past[:, :, None], bad) for k, bad in (("x", math.nan), ("dy", -math.inf)))
    got = conv_run(v)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert not got[0][past].any() and not got[2][past].any()
    assert torch.equal(got[1][2], v["state"][2])  # an empty sequence's state


def test_short_conv_stream_of_calls_is_the_whole():
    """The state that a call leaves is what the next one takes, in place too: cut anywhere, a sequence gives the same bits."""
    say("short_conv stream")
    import torch
    q, m = Rand(9), mod()
    v = conv_inputs(q, 5, 41, 72, 4, torch.bfloat16)
    whole = m.short_conv(v["x"], v["w"], v["bias"], state=v["state"])
    state, at = v["state"].clone(), 0
    for n in (1, 1, 2, 1, 20, 0, 3, 13):
        y, state = m.short_conv(v["x"][:, at:at + n], v["w"], v["bias"], state=state)
        assert torch.equal(y, whole[0][:, at:at + n]), at
        at += n
    assert at == 41 and torch.equal(state, whole[1])
    L, S = m._lib(), m.FhcSeq
    for n, d in ((0, 72), (1, 72), (2, 72), (41, 72), (1, 5), (2, 37), (3, 515), (1, 515), (2, 1031)):
        v = conv_inputs(q, 5, n, d, 4, torch.bfloat16)  # through the C ABI, the new state over the old one
        x, y, st = v["x"], torch.empty_like(v["x"]), v["state"].clone()
        g = m.ShortConvDesc(1, 0, 5, n, d, 4, v["w"].data_ptr(), v["bias"].data_ptr(), None)
        rc = L.fhc_short_conv_forward(g, S(x.data_ptr(), n * d, d), st.data_ptr(), S(y.data_ptr(), n * d, d),
                                      st.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0, m.fhconv.last_error()
        want = m.short_conv(x, v["w"], v["bias"], state=v["state"])
        assert torch.equal(st, want[1]) and torch.equal(y, want[0])


def test_short_conv_views():
    """Channels out of wider rows, an element off every alignment; what lies beside stays."""
    say("short_conv views")
    import torch
    q, m = Rand(11), mod()
    for dtype in (torch.float16, torch.float32):
        for d, off in ((37, 1), (64, 3), (9, 0)):
            wide = q.normal(3, 50, d + 11, dtype=dtype)
            v = conv_inputs(q, 3, 50, d, 4, dtype)
            v["x"] = wide[:, :, off:off + d]
            v["dy"] = q.normal(50, 3, d + 7, dtype=dtype)[:, :, off:off + d].transpose(0, 1)
            conv_check(v)
            out = torch.full_like(wide, 7.0)
            g = m.ShortConvDesc({torch.float16: 0, torch.float32: 2}[dtype], 0, 3, 50, d, 4, v["w"].data_ptr(),
                                v["bias"].data_ptr(), None)
            view = out[:, :, off:off + d]
            to, of = (m.FhcSeq(p.data_ptr(), p.stride(0), p.stride(1)) for p in (view, v["x"]))
            assert m._lib().fhc_short_conv_forward(g, of, None, to, None, torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(view, m.short_conv(v["x"], v["w"], v["bias"])[0])
            view.fill_(7.0)
            assert (out == 7.0).all()


def test_short_conv_sequences_that_share_their_elements():
    say("short_conv shared")
    import torch
    q, m = Rand(13), mod()
    v = conv_inputs(q, 6, 30, 40, 3, torch.float16)
    one = q.normal(1, 30, 40, dtype=torch.float16)
    windows = q.normal(1, 60, 40, dtype=torch.float16).as_strided((6, 30, 40), (80, 40, 1))
    for x in (one.expand(6, 30, 40), windows):
        a, b = (conv_run({**v, "x": p}) for p in (x, x.contiguous()))
        assert all(torch.equal(p, r) for p, r in zip(a, b))


def test_short_conv_values_that_are_not_finite_stay_where_they_are():
    say("short_conv not finite")
    import torch
    q, m = Rand(15), mod()
    v = conv_inputs(q, 2, 70, 21, 4, torch.float32)
    clean = m.short_conv(v["x"], v["w"], v["bias"], state=v["state"])[0]
    v["x"][1, 40, 5], v["x"][0, 3, 20] = math.inf, math.nan
    y = m.short_conv(v["x"], v["w"], v["bias"], state=v["state"])[0]
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[1, 40:44, 5] = touched[0, 3:7, 20] = True
    assert torch.equal(y[~touched], clean[~touched]) and not torch.isfinite(y[0, 3:7, 20]).any()


def test_short_conv_gradient_against_differences():
    say("short_conv differences")
    import torch
    q = Rand(17)
    v = conv_inputs(q, 3, 40, 24, 4, torch.float32, ragged=True)
    grads = dict(zip(("x", "w", "bias", "state"), conv_run(v)[2:]))

    def loss(name, d):
        a = {k: v[k].double() for k in ("x", "w", "bias", "state")}
        a[name] = a[name] + d
        (y, end), _ = ssmref.short_conv(a["x"], a["w"], a["bias"], "silu", a["state"], v["lengths"])
        return float((y * v["dy"].double()).sum() + (end * v["dstate"].double()).sum())

    for k, grad in grads.items():
        d, s = q.normal(*grad.shape).double(), 1e-5
        slope, want = (loss(k, s * d) - loss(k, -s * d)) / (2 * s), float((grad.double() * d).sum())
        assert abs(slope - want) <= 1e-5 * float((grad.double() * d).abs().sum()) + 1e-7, (k, slope, want)


def replays(run, inputs, outputs):
    """A captured call against eager ones, over several replays with other inputs, eager work between them."""
    import torch
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run()
    for k in range(4):
        for x in inputs:
            x.copy_(torch.roll(x, 1, 0) if k else x)
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want) if a is not None and a.dtype is not torch.uint8), k
        with torch.cuda.stream(stream):  # the same on another stream
            stream.wait_stream(torch.cuda.default_stream())
            other = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want) if a is not None and a.dtype is not torch.uint8), k
    assert len(kept) == outputs


@pytest.mark.parametrize("shape", [(4, 1, 64, 4), (3, 300, 100, 4)], ids=str)
def test_short_conv_in_a_graph_and_on_another_stream(shape):
    say("short_conv graph", shape)
    import torch
    v = conv_inputs(Rand(19), *shape, torch.bfloat16)
    replays(lambda: conv_run(v), [v["x"], v["dy"], v["state"]], 6)


def test_short_conv_empty_sides():
    say("short_conv empty")
    import torch
    m = mod()
    for b, t, d in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        v = conv_inputs(Rand(21), b, t, d, 3, torch.float16)
        got = conv_run(v)
        assert got[0].shape == got[2].shape == (b, t, d) and got[1].shape == (b, 2, d)
        if t == 0:
            assert torch.equal(got[1], v["state"]) and torch.equal(got[5], v["dstate"])
        assert not got[3].any() and not got[4].any() if min(b, t) == 0 else True
    assert m is mod()


# ---- the selective scan -------------------------------------------------------------------------------------------

SSM = [  # b, t, d, n, groups: few steps; part of a tile, whole ones; each number of waves; odd states; groups; segments
    (1, 1, 1, 1, 1), (5, 1, 64, 16, 1), (3, 2, 7, 5, 1), (2, 4, 130, 16, 2), (3, 3, 34, 64, 2), (2, 5, 66, 4, 1),
    (2, 16, 66, 8, 1), (2, 17, 66, 16, 1), (1, 64, 33, 33, 1), (3, 65, 34, 64, 2), (2, 31, 200, 13, 4),
    (2, 200, 128, 16, 1), (1, 1000, 130, 16, 2), (2, 700, 250, 12, 1), (40, 70, 256, 16, 1), (300, 20, 96, 16, 3),
    (1, 2100, 64, 30, 1), (1030, 9, 128, 4, 1),
]
SSM_NAMES = ("y", "ht", "dx", "ddt", "da", "dbm", "dcm", "dskip", "dz", "ddt_bias", "dh0")


def ssm_inputs(q, b, t, d, n, groups, dtype, time_major=False, ragged=False):
    import torch
    seq = seqs(q, time_major)
    return dict(x=seq(b, t, d, dtype), dt=seq(b, t, d, dtype, 0.5), z=seq(b, t, d, dtype), bm=seq(b, t, groups * n, dtype),
                cm=seq(b, t, groups * n, dtype), a=-torch.arange(1, n + 1, device="cuda") * q.uniform(d, n, lo=0.9, hi=1.1),
                dt_bias=q.uniform(d, lo=-6.0, hi=1.0), skip=q.normal(d), h0=q.normal(b, d, n, scale=0.3),
                lengths=lengths_of(q, b, t, ragged), dy=seq(b, t, d, dtype), dht=q.normal(b, d, n))


def ssm_run(v, serving=True):
    m = mod()
    kw = {k: v[k] for k in ("skip", "z", "dt_bias", "lengths")}
    y, ht, states = m.ssm(v["x"], v["dt"], v["a"], v["bm"], v["cm"], h0=v["h0"], train=True, **kw)
    if serving:  # it gives a training forward's bits
        plain = m.ssm(v["x"], v["dt"], v["a"], v["bm"], v["cm"], h0=v["h0"], **kw)
        assert all(_same(a, b) for a, b in zip(plain, (y, ht)))
    return (y, ht) + m.ssm_backward(v["x"], v["dt"], v["a"], v["bm"], v["cm"], states, v["dy"], dht=v["dht"], **kw)


def _same(a, b):
    import torch
    if a is None or b is None:
        return a is b
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


def ssm_check(v):
    got = ssm_run(v)
    ref, err = ssmref.ssm(v["x"], v["dt"], v["a"], v["bm"], v["cm"], v["skip"], v["z"], v["dt_bias"], v["h0"],
                          v["lengths"], v["dy"], v["dht"])
    compare(SSM_NAMES, got, ref, err)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SSM, ids=str)
def test_ssm(shape, dtype):
    say("ssm", shape, dtype)
    q = Rand(sum(shape))
    ssm_check(ssm_inputs(q, *shape, types()[dtype], time_major=shape[2] % 4 == 2, ragged=shape[1] % 2 == 1))


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", [(3, 4, 70, 16, 1), (3, 6, 70, 6, 1), (2, 8, 40, 64, 1), (9, 512, 256, 16, 1),
                                   (2, 1030, 128, 64, 1), (5, 333, 192, 8, 3), (600, 40, 64, 16, 1)], ids=str)
def test_ssm_sides_of_the_rules(shape, ragged):
    """The last step kernels and the first tiles; segments by rounds of workgroups and, with lengths, by their number."""
    say("ssm rules", shape, ragged)
    ssm_check(ssm_inputs(Rand(sum(shape) + 1), *shape, types()["bf16"], ragged=ragged))


def test_ssm_lengths_at_the_ends_of_tiles_and_segments():
    say("ssm lengths at ends")
    import torch
    v = ssm_inputs(Rand(29), 8, 640, 72, 16, 1, torch.float16)
    v["lengths"] = torch.tensor([640, 0, 16, 15, 17, 64, 320, 639], dtype=torch.int32, device="cuda")
    ssm_check(v)


def test_ssm_two_streams_at_once():
    """Calls of their own workspaces that overlap give the bits of calls one after the other."""
    say("ssm two streams")
    import torch
    vs = [ssm_inputs(Rand(31 + i), 2, 900, 128, 16, 1, torch.bfloat16) for i in range(2)]
    want = [ssm_run(v, False) for v in vs]
    streams = [torch.cuda.Stream() for _ in vs]
    for _ in range(3):
        got = []
        for v, s in zip(vs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(ssm_run(v, False))
        torch.cuda.synchronize()
        assert all(_same(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_ssm_parts_left_out():
    say("ssm parts left out")
    import torch
    for shape in ((3, 2, 40, 8, 1), (3, 40, 70, 16, 2), (1, 400, 64, 4, 1)):
        v = ssm_inputs(Rand(23), *shape, torch.float16)
        for gone in (("skip",), ("z",), ("dt_bias",), ("h0",), ("dht",), ("skip", "z", "dt_bias", "h0", "dht")):
            ssm_check({k: None if k in gone else x for k, x in v.items()})


@pytest.mark.parametrize("shape", [(4, 3, 10, 16, 1), (4, 37, 70, 16, 2), (3, 600, 64, 5, 1)], ids=str)
def test_ssm_masked_places_are_not_read(shape):
    """NaN and infinities past the lengths, empty sequences, lengths outside [0, t]."""
    say("ssm masked", shape)
    import torch
    v = ssm_inputs(Rand(25), *shape, torch.float16, ragged=True)
    v["lengths"][1], v["lengths"][2] = shape[1] + 1000, -3
    past = torch.arange(shape[1], device="cuda")[None] >= v["lengths"][:, None]
    clean = ssm_check(v)
    for k, bad in (("x", math.nan), ("dt", math.inf), ("z", math.nan), ("bm", -math.inf), ("cm", math.nan), ("dy", math.inf)):
        v[k] = v[k].masked_fill(past[:, :, None], bad)
    got = ssm_run(v)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    for i in (0, 2, 3, 5, 6, 8):
        assert not got[i][past].any()
    assert torch.equal(got[1][2], v["h0"][2]) and torch.equal(got[10][2], v["dht"][2])  # an empty sequence's


@pytest.mark.parametrize("t", [1, 3, 40, 300])
def test_ssm_steps_at_their_ends(t):
    """Steps of 0 keep the states and take no input, large ones replace them; rates of 0 and -inf; no gradient is NaN."""
    say("ssm ends", t)
    import torch
    v = ssm_inputs(Rand(27), 2, t, 48, 8, 1, torch.float32)
    v["dt_bias"] = None
    v["dt"][0], v["dt"][1] = -math.inf, 90.0
    got = ssm_run(v)
    assert torch.equal(got[1][0], v["h0"][0]) and all(torch.isfinite(g).all() for g in got)
    v["dt"][1] = -120.0  # e^-120 is below f32's range: a step of 0
    v["a"][:, 0], v["a"][:, 1] = 0.0, -math.inf
    got = ssm_run(v)
    assert torch.equal(got[1], v["h0"])


def test_ssm_small_steps_keep_their_digits():
    """Steps of e^-30 to e^-3: a state that decays by them, and an input that they scale, are right to f32's rounding."""
    say("ssm small steps")
    import torch
    v = ssm_inputs(Rand(29), 2, 33, 64, 4, 1, torch.float32)
    v["dt"] = torch.linspace(-30, -3, 33, device="cuda")[None, :, None].expand(2, 33, 64).contiguous()
    v["dt_bias"] = None
    ssm_check(v)


def test_ssm_stream_of_calls_is_the_whole():
    """The states that a call leaves are what the next one takes, by steps and by stretches, in place too."""
    say("ssm stream")
    import torch
    q, m = Rand(31), mod()
    v = ssm_inputs(q, 5, 61, 72, 16, 1, torch.float32)
    (y, ht), err = ssmref.ssm(*(v[k] for k in ("x", "dt", "a", "bm", "cm", "skip", "z", "dt_bias", "h0")))
    at, h = 0, v["h0"].clone()
    for n in (1, 1, 2, 5, 0, 30, 3, 19):
        cut = {k: v[k][:, at:at + n] for k in ("x", "dt", "bm", "cm", "z")}
        part, h = m.ssm(cut["x"], cut["dt"], v["a"], cut["bm"], cut["cm"], v["skip"], cut["z"], v["dt_bias"], h)
        seqref.close(part, y[:, at:at + n], err[0][:, at:at + n], f"y from {at}")
        at += n
    assert at == 61
    seqref.close(h, ht, err[1], "ht")
    L, S = m._lib(), m.FhcSeq
    for t in (0, 1, 40, 1000):  # through the C ABI, the new states over the old ones
        v = ssm_inputs(q, 2, t, 72, 16, 1, torch.bfloat16)
        x, dt, z, bm, cm = (v[k] for k in ("x", "dt", "z", "bm", "cm"))
        y, h = torch.empty_like(x), v["h0"].clone()
        g = m.SsmDesc(1, 2, t, 72, 16, 1, v["a"].data_ptr(), v["dt_bias"].data_ptr(), v["skip"].data_ptr(), None)
        n = L.fhc_ssm_workspace_bytes(g, 0)
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        sq = [S(p.data_ptr(), p.stride(0), p.stride(1)) for p in (x, dt, bm, cm, z)]
        rc = L.fhc_ssm_forward(g, *sq, h.data_ptr(), S(y.data_ptr(), y.stride(0), y.stride(1)), h.data_ptr(), None,
                               ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, m.fhconv.last_error()
        want = m.ssm(x, dt, v["a"], bm, cm, v["skip"], z, v["dt_bias"], v["h0"])
        assert torch.equal(h, want[1]) and torch.equal(y, want[0])


def test_ssm_views():
    """Channels, B and C out of wider rows, an element off every alignment; what lies beside the results stays."""
    say("ssm views")
    import torch
    q, m = Rand(33), mod()
    for dtype in (torch.bfloat16, torch.float32):
        for t, d, n in ((2, 37, 5), (50, 37, 16), (300, 70, 3)):
            v = ssm_inputs(q, 3, t, d, n, 1, dtype)
            wide = q.normal(3, t, 2 * d + 2 * n + 5, scale=0.5, dtype=dtype)  # as a projection leaves them
            v["z"], v["dt"] = wide[:, :, 1:1 + d], wide[:, :, d + 1:2 * d + 1]
            v["bm"], v["cm"] = wide[:, :, 2 * d + 2:2 * d + 2 + n], wide[:, :, 2 * d + n + 3:2 * d + 2 * n + 3]
            ssm_check(v)
            out = torch.full_like(wide, 7.0)
            view = out[:, :, 3:3 + d]
            g = m.SsmDesc({torch.bfloat16: 1, torch.float32: 2}[dtype], 3, t, d, n, 1, v["a"].data_ptr(), None, None, None)
            size = m._lib().fhc_ssm_workspace_bytes(g, 0)
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
            sq = [m.FhcSeq(p.data_ptr(), p.stride(0), p.stride(1)) for p in (v["x"], v["dt"], v["bm"], v["cm"], view)]
            rc = m._lib().fhc_ssm_forward(g, *sq[:4], None, None, sq[4], None, None, ws.data_ptr(), size,
                                          torch.cuda.current_stream().cuda_stream)
            assert rc == 0, m.fhconv.last_error()
            assert torch.equal(view, m.ssm(v["x"], v["dt"], v["a"], v["bm"], v["cm"])[0])
            view.fill_(7.0)
            assert (out == 7.0).all()


def test_ssm_sequences_that_share_their_elements():
    say("ssm shared")
    import torch
    q = Rand(35)
    for t in (2, 30, 300):
        v = ssm_inputs(q, 4, t, 40, 16, 1, torch.float16)
        for k in ("x", "dt", "bm", "dy"):
            one = q.normal(1, t, v[k].shape[2], scale=0.5, dtype=torch.float16)
            a, b = (ssm_run({**v, k: p}) for p in (one.expand(4, t, -1), one.expand(4, t, -1).contiguous()))
            assert all(torch.equal(p, r) for p, r in zip(a, b)), k


@pytest.mark.parametrize("t", [4, 64, 600])
def test_ssm_values_that_are_not_finite_stay_in_their_channel(t):
    """An infinite input changes nothing before its step, in another channel or another sequence."""
    say("ssm not finite", t)
    import torch
    m = mod()
    v = ssm_inputs(Rand(37), 2, t, 70, 16, 1, torch.float32)
    args = lambda: (v["x"], v["dt"], v["a"], v["bm"], v["cm"], v["skip"], v["z"], v["dt_bias"], v["h0"])  # noqa: E731
    clean = m.ssm(*args())
    at = t // 2 + 1
    v["x"][1, at, 69] = math.inf
    y, ht = m.ssm(*args())
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[1, at:, 69] = True
    assert torch.equal(y[~touched], clean[0][~touched]) and not torch.isfinite(y[1, at, 69])
    assert torch.equal(ht[0], clean[1][0]) and torch.equal(ht[1, :69], clean[1][1, :69])


@pytest.mark.parametrize("shape", [(2, 3, 20, 6, 2), (2, 30, 24, 16, 1), (1, 200, 16, 4, 1)], ids=str)
def test_ssm_gradient_against_differences(shape):
    say("ssm differences", shape)
    import torch
    q = Rand(39)
    v = ssm_inputs(q, *shape, torch.float32, ragged=True)
    names = ("x", "dt", "a", "bm", "cm", "skip", "z", "dt_bias", "h0")
    grads = dict(zip(names, ssm_run(v)[2:]))

    def loss(name, d):
        a = {k: v[k].double() for k in names}
        a[name] = a[name] + d
        (y, end), _ = ssmref.ssm(*(a[k] for k in names), v["lengths"])
        return float((y * v["dy"].double()).sum() + (end * v["dht"].double()).sum())

    for k, grad in grads.items():
        d, s = q.normal(*grad.shape).double(), 1e-5
        slope, want = (loss(k, s * d) - loss(k, -s * d)) / (2 * s), float((grad.double() * d).sum())
        assert abs(slope - want) <= 2e-5 * float((grad.double() * d).abs().sum()) + 1e-6, (k, slope, want)


@pytest.mark.parametrize("shape", [(4, 1, 64, 16, 1), (3, 50, 100, 16, 1), (1, 700, 64, 16, 1)], ids=str)
def test_ssm_in_a_graph_and_on_another_stream(shape):
    say("ssm graph", shape)
    import torch
    v = ssm_inputs(Rand(41), *shape, torch.bfloat16)
    replays(lambda: ssm_run(v, False), [v["x"], v["dt"], v["dy"], v["h0"]], 11)


def test_ssm_empty_sides():
    say("ssm empty")
    import torch
    for b, t, d in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        v = ssm_inputs(Rand(43), b, t, d, 4, 1, torch.float16)
        got = ssm_run(v)
        assert got[0].shape == got[2].shape == (b, t, d) and got[1].shape == (b, d, 4) and got[5].shape == (b, t, 4)
        if t == 0:
            assert torch.equal(got[1], v["h0"]) and torch.equal(got[10], v["dht"])
        if d == 0:
            assert not got[5].any() and not got[6].any()
        if 0 in (b, t):
            assert not got[4].any() and not got[7].any() and not got[9].any()


@pytest.mark.parametrize("shape", [(2, 3, 70, 5, 1), (2, 40, 70, 16, 2), (1, 700, 130, 30, 1)], ids=str)
def test_ssm_stays_in_its_buffers(shape):
    """The workspace and the kept states, of the stated sizes, between guards."""
    say("ssm buffers", shape)
    import torch
    m, L = mod(), mod()._lib()
    b, t, d, n, groups = shape
    v = ssm_inputs(Rand(45), *shape, torch.bfloat16)
    g = m.SsmDesc(1, b, t, d, n, groups, v["a"].data_ptr(), v["dt_bias"].data_ptr(), v["skip"].data_ptr(), None)
    seq = lambda p: m.FhcSeq(p.data_ptr(), p.stride(0), p.stride(1))  # noqa: E731
    st = torch.cuda.current_stream().cuda_stream

    def guarded(size):
        buf = torch.full((size + 512,), 0x5A, dtype=torch.uint8, device="cuda")
        return buf, buf.data_ptr() + 256

    keep, pk = guarded(L.fhc_ssm_states_bytes(g))
    ins = [seq(v[k]) for k in ("x", "dt", "bm", "cm", "z")]
    y, ht, dh0 = torch.empty_like(v["x"]), torch.empty_like(v["h0"]), torch.empty_like(v["h0"])
    outs = [torch.empty_like(v[k]) for k in ("x", "dt", "bm", "cm", "z")]
    da, db, ds = torch.empty_like(v["a"]), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    for back in (0, 1):
        size = L.fhc_ssm_workspace_bytes(g, back)
        ws, pw = guarded(size)
        if back:
            rc = L.fhc_ssm_backward(g, *ins, pk, seq(v["dy"]), v["dht"].data_ptr(), *(seq(o) for o in outs),
                                    da.data_ptr(), db.data_ptr(), ds.data_ptr(), dh0.data_ptr(), pw, size, st)
        else:
            rc = L.fhc_ssm_forward(g, *ins, v["h0"].data_ptr(), seq(y), ht.data_ptr(), pk, pw, size, st)
        assert rc == 0, m.fhconv.last_error()
        for buf in (ws, keep):
            assert (buf[:256] == 0x5A).all() and (buf[-256:] == 0x5A).all()
    want = ssm_run(v)
    assert all(torch.equal(a, b) for a, b in zip((y, ht, outs[0], outs[1], da, outs[2], outs[3], ds, outs[4], db, dh0), want))


def test_long_offsets():
    """Sequences whose elements lie past 2^31 elements and 2^32 bytes from the tensor's start."""
    say("long offsets")
    import torch
    q, m = Rand(47), mod()
    t, d, n, gap = 70, 64, 8, (1 << 31) + 64
    big = torch.zeros(gap + t * d, dtype=torch.float16, device="cuda")
    x = big.as_strided((2, t, d), (gap, d, 1))
    v = ssm_inputs(q, 2, t, d, n, 1, torch.float16)
    x.copy_(v["x"])
    kw = dict(skip=v["skip"], z=v["z"], dt_bias=v["dt_bias"], h0=v["h0"])
    for cut in (2, t):
        a, b = (m.ssm(p[:, :cut], v["dt"][:, :cut], v["a"], v["bm"][:, :cut], v["cm"][:, :cut],
                      **{**kw, "z": v["z"][:, :cut]}) for p in (x, v["x"]))
        assert all(torch.equal(p, r) for p, r in zip(a, b))
    w = q.normal(d, 4, dtype=torch.float16)
    assert torch.equal(m.short_conv(x, w)[0], m.short_conv(v["x"], w)[0])
    steps = big.as_strided((1, 3, d), (1, 1 << 30, 1))
    steps.copy_(v["x"][:1, :3])
    assert torch.equal(m.short_conv(steps, w)[0], m.short_conv(v["x"][:1, :3].contiguous(), w)[0])


# ---- the product with its epilogue --------------------------------------------------------------------------------

LINEAR = [  # rows, c, f: few rows; each size of tile; a split K; odd sizes
    (1, 1, 1), (4, 64, 40), (7, 129, 33), (32, 200, 500), (33, 200, 36), (100, 60, 61), (130, 1000, 132),
    (300, 2050, 70), (1003, 1020, 273), (700, 35, 2050), (2500, 130, 4100),
]
LINEAR_NAMES = ("y", "dx", "dw", "dbias")


def linear_inputs(q, rows, c, f, dtype, bias=True, residual=True):
    return dict(x=q.normal(rows, c, dtype=dtype), w=q.normal(f, c, scale=c ** -0.5, dtype=dtype),
                bias=q.normal(f, dtype=dtype) if bias else None, residual=q.normal(rows, f, dtype=dtype) if residual else None,
                dy=q.normal(rows, f, dtype=dtype))


def linear_run(v, act, serving=True):
    m = mod()
    y, kept = m.linear(v["x"], v["w"], v["bias"], v["residual"], act, train=True)
    assert not serving or _same(y, m.linear(v["x"], v["w"], v["bias"], v["residual"], act))
    return (y,) + m.linear_backward(v["x"], v["w"], kept, v["dy"], act, bias=v["bias"] is not None)


def linear_check(v, act):
    got = linear_run(v, act)
    ref, err = ssmref.linear(v["x"], v["w"], v["bias"], v["residual"], act, v["dy"])
    if v["bias"] is None:
        ref[3] = None
    compare(LINEAR_NAMES, got, ref, err)
    return got


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", LINEAR, ids=str)
def test_linear(shape, dtype, act):
    say("linear", shape, dtype, act)
    q = Rand(sum(shape))
    linear_check(linear_inputs(q, *shape, types()[dtype], bias=shape[0] % 4 != 3, residual=shape[1] % 2 == 0), act)


@pytest.mark.parametrize("shape", [(20, 64, 48), (300, 72, 48), (300, 65, 47), (200, 1000, 52)], ids=str)
def test_linear_views_and_in_place(shape):
    """Rows out of wider ones; the result over the residual; what lies beside stays."""
    say("linear views", shape)
    import torch
    m, L = mod(), mod()._lib()
    rows, c, f = shape
    for off in (0, 1, 4):
        q = Rand(49 + off)
        v = linear_inputs(q, rows, c, f, torch.bfloat16)
        v["x"] = q.normal(rows, c + 9, dtype=torch.bfloat16)[:, off:off + c]
        v["dy"] = q.normal(rows, f + 7, dtype=torch.bfloat16)[:, off:off + f]
        v["residual"] = q.normal(rows, f + 8, dtype=torch.bfloat16)[:, off:off + f]
        for act in ("none", "gelu"):
            want = linear_check(v, act)[0]
            wide = torch.full((rows, f + 8), 7.0, dtype=torch.bfloat16, device="cuda")
            view = wide[:, off:off + f]
            view.copy_(v["residual"])
            d = m.LinearDesc(1, m.LINEAR_ACTS[act], rows, c, f)
            n = L.fhc_linear_workspace_bytes(d, 0)
            ws = torch.full((n + 512,), 0x5A, dtype=torch.uint8, device="cuda")
            to = m.FhcRows(view.data_ptr(), f + 8)
            rc = L.fhc_linear_forward(d, m.FhcRows(v["x"].data_ptr(), c + 9), v["w"].data_ptr(), v["bias"].data_ptr(), to,
                                      to, None, ws.data_ptr() + 256, n, torch.cuda.current_stream().cuda_stream)
            assert rc == 0, m.fhconv.last_error()
            assert torch.equal(view, want)
            view.fill_(7.0)
            assert (wide == 7.0).all() and (ws[:256] == 0x5A).all() and (ws[-256:] == 0x5A).all()


def test_linear_some_gradients_only():
    say("linear some gradients")
    import torch
    m, L = mod(), mod()._lib()
    for shape in ((20, 33, 47), (300, 72, 48), (300, 65, 47)):
        for act in ("none", "silu"):
            rows, c, f = shape
            v = linear_inputs(Rand(51), *shape, torch.float16)
            want = linear_run(v, act)[1:]
            kept = m.linear(v["x"], v["w"], v["bias"], None, act, train=True)[1]
            d = m.LinearDesc(0, m.LINEAR_ACTS[act], rows, c, f)
            n = L.fhc_linear_workspace_bytes(d, 1)
            for pick in range(8):
                ws = torch.full((n + 512,), 0x5A, dtype=torch.uint8, device="cuda")
                out = [torch.full_like(w, 7.0) for w in want]
                to = m.FhcRows(out[0].data_ptr(), c) if pick & 1 else None
                rc = L.fhc_linear_backward(d, m.FhcRows(v["x"].data_ptr(), c), v["w"].data_ptr(),
                                           None if kept is None else kept.data_ptr(), m.FhcRows(v["dy"].data_ptr(), f), to,
                                           out[1].data_ptr() if pick & 2 else None,
                                           out[2].data_ptr() if pick & 4 else None, ws.data_ptr() + 256, n,
                                           torch.cuda.current_stream().cuda_stream)
                assert rc == 0, m.fhconv.last_error()
                for i in range(3):
                    assert torch.equal(out[i], want[i]) if pick >> i & 1 else (out[i] == 7.0).all(), (shape, act, pick, i)
                assert (ws[:256] == 0x5A).all() and (ws[-256:] == 0x5A).all()


def test_linear_empty_sides():
    say("linear empty")
    import torch
    for rows, c, f in ((0, 16, 24), (20, 0, 24), (300, 0, 24), (300, 16, 0), (20, 16, 0)):
        for act in ("none", "silu"):
            v = linear_inputs(Rand(53), rows, max(c, 1), f, torch.float16)
            v["x"], v["w"] = v["x"][:, :c], v["w"][:, :c].contiguous()
            y, dx, dw, dbias = linear_run(v, act)
            assert y.shape == (rows, f) and dx.shape == (rows, c) and dw.shape == (f, c) and dbias.shape == (f,)
            if c == 0 and f:
                b, r = v["bias"].double(), v["residual"].double()
                want = (b if act == "none" else b * torch.sigmoid(b)) + r
                seqref.close(y, want, 64 * seqref.U * (want.abs() + 1), "y")
            if rows == 0 or f == 0:
                assert not dw.any() and not dx.any() and not dbias.any()


def test_linear_values_that_are_not_finite_stay_in_their_rows():
    say("linear not finite")
    import torch
    m = mod()
    for shape in ((20, 40, 52), (300, 72, 48), (300, 65, 47), (140, 2048, 64)):
        v = linear_inputs(Rand(55), *shape, torch.bfloat16)
        clean = m.linear(v["x"], v["w"], v["bias"], v["residual"])
        v["x"][3], v["residual"][7, 5] = math.nan, math.inf
        y = m.linear(v["x"], v["w"], v["bias"], v["residual"])
        assert y[3].isnan().all() and math.isinf(y[7, 5])
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[3], keep[7, 5] = False, False
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("shape", [(8, 128, 256), (300, 1024, 256)], ids=str)
def test_linear_in_a_graph_and_on_another_stream(shape):
    say("linear graph", shape)
    import torch
    v = linear_inputs(Rand(57), *shape, torch.bfloat16)
    replays(lambda: linear_run(v, "silu", False), [v["x"], v["dy"], v["residual"]], 4)


def test_linear_gradient_against_differences():
    say("linear differences")
    import torch
    q = Rand(59)
    v = linear_inputs(q, 40, 48, 36, torch.float16)
    for act in ("none", "silu", "gelu"):
        grads = dict(zip(("x", "w", "bias"), linear_run(v, act)[1:]))

        def loss(name, d):
            a = {k: v[k].double() for k in ("x", "w", "bias", "residual")}
            a[name] = a[name] + d
            y = a["x"] @ a["w"].t() + a["bias"]
            return float(((y if act == "none" else seqref._act(y, act)[0]) * v["dy"].double()).sum())

        for k, grad in grads.items():
            d, s = q.normal(*grad.shape).double(), 1e-5
            slope, want = (loss(k, s * d) - loss(k, -s * d)) / (2 * s), float((grad.double() * d).sum())
            # dL/dv and the gradient are rounded to f16, each by half a step
            assert abs(slope - want) <= 4 * 2 ** -11 * float((grad.double() * d).abs().sum()), (act, k, slope, want)
