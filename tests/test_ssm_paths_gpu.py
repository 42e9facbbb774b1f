"""Calls of the short convolution, the selective scan and the product with its epilogue that the shapes of test_ssm_gpu.py
do not reach: weights' gradients over very many rows, states that grow, calls of very many sequences, and the kernels that
only larger calls take. On the GPU, against plain 64-bit forms or closed ones."""
import math

import pytest

import fhtest  # noqa: F401  (puts the package on sys.path)
import seqref
import ssmref
from seqref import U
from test_seq_gpu import Rand, mod, say, types
from test_ssm_gpu import (LINEAR_NAMES, SSM_NAMES, _same, compare, conv_check, conv_inputs, linear_check, linear_inputs, linear_run,
                          ssm_check, ssm_inputs)

pytestmark = pytest.mark.gpu


# ---- dL/dv in the product's backward pass -------------------------------------------------------------------------

def linear_split_ref(v, act):
    """ssmref.linear's results and bounds with dL/dv held as the sum of two numbers of the inputs' type: what is left is
    half a step of the second one (itself at most half a step of the first), or half the smallest number."""
    x, w, dy = (v[k].double() for k in ("x", "w", "dy"))
    import torch
    hs, fi = seqref.half_step(v["x"].dtype), torch.finfo(v["x"].dtype)
    ref, err = ssmref.linear(v["x"], v["w"], v["bias"], v["residual"], act, v["dy"])
    pre = x @ w.t() + (0 if v["bias"] is None else v["bias"].double())
    chain = lambda k: (2 * k / 32 + 34) * U  # noqa: E731  (two products along the same sum)
    ev = (w.shape[1] / 32 + 34) * U * (x.abs() @ w.abs().t()) + 2 * U * pre.abs()
    slope = seqref._act(pre, act)[1]
    dv, edv = dy * slope, dy.abs() * (1.2 * ev + 64 * U * (slope.abs() + 1)) + 2 * U * (dy * slope).abs()
    e = edv + hs * hs * (dv.abs() + edv) + fi.tiny * fi.eps / 2
    size = dv.abs() * (1 + 2 * hs)
    err[1] = e @ w.abs() + chain(w.shape[0]) * (size @ w.abs())
    err[2] = e.t() @ x.abs() + chain(x.shape[0]) * (size.t() @ x.abs())
    if v["bias"] is None:
        ref[3] = None
    return ref, err


SPLIT = [(1, 7, 9), (20, 64, 520), (300, 72, 48), (333, 65, 47), (130, 1000, 1032), (1003, 130, 273), (2100, 2050, 40)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SPLIT, ids=str)
def test_linear_gradients_keep_the_bits_of_dv(shape, dtype, act):
    """dx and dw are the products of dL/dv, not of its rounding to 16 bits."""
    say("linear dv", shape, dtype, act)
    v = linear_inputs(Rand(sum(shape) + 3), *shape, types()[dtype], bias=shape[0] % 2 == 0)
    ref, err = linear_split_ref(v, act)
    compare(LINEAR_NAMES, linear_run(v, act), ref, err)


@pytest.mark.parametrize("dtype,act", [("f16", "gelu"), ("bf16", "silu"), ("bf16", "none")])
@pytest.mark.parametrize("shape", SPLIT, ids=str)
def test_linear_gradients_of_a_rounded_dv(shape, dtype, act):
    """round_dv: within the rounding of dL/dv of the formula; without an activation there is nothing to round."""
    say("linear rounded dv", shape, dtype, act)
    m = mod()
    v = linear_inputs(Rand(sum(shape) + 4), *shape, types()[dtype])
    kept = m.linear(v["x"], v["w"], v["bias"], v["residual"], act, train=True)[1]
    got = m.linear_backward(v["x"], v["w"], kept, v["dy"], act, round_dv=True)
    ref, err = ssmref.linear(v["x"], v["w"], v["bias"], v["residual"], act, v["dy"])
    compare(LINEAR_NAMES[1:], got, ref[1:], err[1:])
    full = m.linear_backward(v["x"], v["w"], kept, v["dy"], act)
    assert _same(got[2], full[2]) and (act != "none" or all(_same(a, b) for a, b in zip(got, full)))


def test_linear_gradients_past_the_types_range():
    """A dL/dv that f16 does not hold is an infinity in its row's dx and its column's dw, and no NaN."""
    say("linear dv past the range")
    import torch
    m = mod()
    v = linear_inputs(Rand(67), 40, 24, 16, torch.float16, bias=False)
    v["x"].fill_(1.0), v["w"].fill_(0.1)  # v = 2.4, where silu's slope is 1.0998
    v["dy"][3, 5] = 65504.0
    for round_dv in (False, True):
        kept = m.linear(v["x"], v["w"], None, None, "silu", train=True)[1]
        dx, dw, _ = m.linear_backward(v["x"], v["w"], kept, v["dy"], "silu", round_dv=round_dv)
        assert (dx[3] == math.inf).all() and (dw[5] == math.inf).all()
        keep_x, keep_w = torch.arange(40) != 3, torch.arange(16) != 5
        assert torch.isfinite(dx[keep_x]).all() and torch.isfinite(dw[keep_w]).all()


# ---- the scan's weights' gradients over very many rows: equal terms, so that a long chain of f32 additions shows ----

def off_by(got, want):
    return float(((got.double() - want) / want).abs().max())


def test_ssm_weight_gradients_of_long_sequences():
    """512 columns of 8192 steps run as one segment. With rates of 0 every term of a sum is the same number, which adding
    one after the other in f32 rounds the same way at every step, a thousand half steps in all. A lane adds at most 256
    terms of da (16 of dskip and ddt_bias, then 16 lanes' sums), each rounded to half a step of the sum so far."""
    say("ssm long chains")
    import torch
    m, b, t = mod(), 512, 8192
    full = lambda c, *s: torch.full(s or (b, t, 1), c, device="cuda")  # noqa: E731
    dt = 20 + 0.4 * 2 ** -6  # softplus(dt) = dt to 1e-10
    c = 1 + 0.4 * 2 ** -15
    dt, c = (float(torch.tensor(k, dtype=torch.float32)) for k in (dt, c))
    a, none = full(0.0, 1, 1), full(0.0)
    # h = 1 and its gradient = 1 throughout: da = sum D; and dskip = sum dy x
    args = (full(1.0), full(dt), a, none, none)
    _, ht, states = m.ssm(*args, h0=full(1.0, b, 1, 1), train=True)
    out = m.ssm_backward(*args, states, full(c), dht=full(1.0, b, 1, 1))
    assert torch.equal(ht, full(1.0, b, 1, 1))
    da, dskip = off_by(out[2], b * t * dt), off_by(out[5], b * t * c)
    print("da off by", da / U, "dskip by", dskip / U, "half steps", flush=True)
    # a state's gradient of 1 against B = 1: ddt = x sigmoid(dt), 1 to 2e-9
    args = (full(c), full(dt), a, full(1.0), none)
    _, _, states = m.ssm(*args, train=True)
    bias = off_by(m.ssm_backward(*args, states, none, dht=full(1.0, b, 1, 1))[7], b * t * c)
    print("ddt_bias off by", bias / U, "half steps", flush=True)
    assert da <= (256 + 8) * U and dskip <= (32 + 4) * U and bias <= (32 + 24) * U


# ---- the convolution's weights' gradients over very many rows -----------------------------------------------------

def test_short_conv_weight_gradients_of_long_sequences():
    """2^27 equal steps: a thread adds at most 256 of them in f32, a workgroup of 32 threads a row 8 such sums."""
    say("short_conv long chains")
    import torch
    m, t, d, k = mod(), 1 << 27, 64, 4
    c = float(torch.tensor(1 + 0.4 * 2 ** -11, dtype=torch.float32))
    x, dy, w = torch.ones(d, device="cuda"), torch.full((d,), c, device="cuda"), torch.zeros(d, k, device="cuda")
    state = torch.ones(k - 1, d, device="cuda")
    g = m.ShortConvDesc(2, m.CONV_ACTS["none"], 1, t, d, k, w.data_ptr(), None, None)
    n = m._lib().fhc_short_conv_workspace_bytes(g)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    dw, db = torch.empty(d, k, device="cuda"), torch.empty(d, device="cuda")
    rc = m._lib().fhc_short_conv_backward(g, m.FhcSeq(x.data_ptr(), 0, 0), state.data_ptr(), m.FhcSeq(dy.data_ptr(), 0, 0),
                                          None, None, dw.data_ptr(), db.data_ptr(), None, ws.data_ptr(), n,
                                          torch.cuda.current_stream().cuda_stream)
    assert rc == 0, m.fhconv.last_error()
    print("dw off by", off_by(dw, t * c) / U, "dbias by", off_by(db, t * c) / U, "half steps", flush=True)
    assert off_by(dw, t * c) <= (256 + 8 + 2) * U and off_by(db, t * c) <= (256 + 8 + 2) * U


# ---- the product's bias' gradient over very many rows -------------------------------------------------------------

def test_linear_bias_gradient_of_many_rows():
    """2^24 equal rows: a thread adds at most 256 of them in f32."""
    say("linear many rows")
    import torch
    m, rows, f = mod(), 1 << 24, 8
    x = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(f, 1, dtype=torch.bfloat16, device="cuda")
    bias = torch.linspace(-1.0, 2.5, f, device="cuda").bfloat16()
    dy = torch.ones(rows, f, dtype=torch.bfloat16, device="cuda")
    _, kept = m.linear(x, w, bias, act="silu", train=True)
    db = m.linear_backward(x, w, kept, dy, "silu")[2]
    v = bias.double()
    slope = seqref._act(v, "silu")[1]
    off = (db.double() - rows * slope).abs()
    print("dbias off by", [round(float(k), 1) for k in off / (rows * U * slope.abs())], "half steps", flush=True)
    # the slope itself to 64 U (as in ssmref.linear), 256 terms and 4 threads' sums
    assert (off <= rows * (64 * U * (slope.abs() + 1) + (256 + 4) * U * slope.abs())).all()


# ---- states that grow ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 2048, 64, 16, 1), (2, 1500, 70, 4, 1)], ids=str)
def test_ssm_states_that_grow(shape):
    """Rates above 0 over long stretches of no input: states and gradients of 0 stay 0 however much a stretch would grow
    them, and what lies at the sequence's other end is that of a call of those steps alone."""
    say("ssm growing", shape)
    import torch
    v = ssm_inputs(Rand(61), *shape, torch.float32)
    v["a"], v["h0"], v["dht"], v["dt_bias"] = v["a"].abs(), None, None, None
    m, t, steps = mod(), shape[1], ("x", "dt", "z", "bm", "cm", "dy")
    kw = lambda q: {k: q[k] for k in ("skip", "z")}  # noqa: E731
    v["dt"].fill_(1.0)
    v["dt"][:, -3:], v["dt"][:, :3] = -3.0, -3.0
    fwd = {**v, "x": v["x"].clone()}
    fwd["x"][:, :-3] = 0.0
    end = {k: q[:, -3:].contiguous() if k in steps else q for k, q in fwd.items()}
    y, ht = m.ssm(fwd["x"], fwd["dt"], v["a"], v["bm"], v["cm"], **kw(fwd))
    ref, err = ssmref.ssm(end["x"], end["dt"], v["a"], end["bm"], end["cm"], **kw(end))
    compare(("y", "ht"), (y[:, -3:], ht), ref, err)
    assert not y[:, :-3].any()
    back = {**v, "x": torch.zeros_like(v["x"]), "dy": v["dy"].clone()}
    back["dy"][:, 3:] = 0.0
    start = {k: q[:, :3].contiguous() if k in steps else q for k, q in back.items()}
    args = (back["x"], back["dt"], v["a"], v["bm"], v["cm"])
    states = m.ssm(*args, train=True, **kw(back))[2]
    got = m.ssm_backward(*args, states, back["dy"], **kw(back))
    ref, err = ssmref.ssm(start["x"], start["dt"], v["a"], start["bm"], start["cm"], **kw(start), dy=start["dy"])
    per_step = (0, 1, 3, 4, 6)  # of got: dx, ddt, dbm, dcm, dz
    compare(SSM_NAMES[2:], [g[:, :3] if i in per_step else g for i, g in enumerate(got)], ref[2:], err[2:])
    assert not any(got[i][:, 3:].any() for i in per_step)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_ssm_stretches_that_grow_or_shrink_by_more_than_a_float(sign):
    """64 steps that grow the states by e^95 or shrink them by that, which f32 does not hold, from 2^-100 or 2^100 on."""
    say("ssm far decays", sign)
    import torch
    m, t, d = mod(), 1024, 64
    x, one = torch.zeros(1, t, d, device="cuda"), torch.ones(1, t, 1, device="cuda")
    dt = torch.full((1, t, d), -60.0, device="cuda")
    dt[:, 64:128] = -4.0
    step = math.log1p(math.exp(-4.0))
    a = torch.full((d, 1), sign * 95.0 / (64 * step), device="cuda")
    h0 = torch.full((1, d, 1), 2.0 ** (-100 * sign), device="cuda")
    want = 2.0 ** (-100 * sign) * math.exp(float(a[0, 0].double()) * 64 * step)
    # the exponents' errors: 95 times the steps' (16 U), their products' and sum's (64 + 4 U); 6 U a decay
    tol = (95 * (16 + 64 + 4) + 6 * 64) * U
    y, ht, states = m.ssm(x, dt, a, one, one, h0=h0, train=True)
    dh0 = m.ssm_backward(x, dt, a, one, one, states, x, dht=h0)[8]
    print("off by", off_by(ht, want) / U, off_by(dh0, want) / U, "half steps", flush=True)
    assert off_by(ht, want) <= tol and off_by(dh0, want) <= tol


# ---- calls of very many sequences ---------------------------------------------------------------------------------

@pytest.mark.parametrize("t", [1, 5])
def test_ssm_of_very_many_sequences(t):
    """2^23 sequences: as many as a launch of 256 threads a sequence has room for."""
    say("ssm many sequences", t)
    import torch
    q, m, b, n = Rand(63), mod(), 1 << 23, 9
    v = ssm_inputs(q, 4096, t, 1, n, 1, torch.bfloat16)
    names = ("x", "dt", "bm", "cm", "z", "h0")
    few = m.ssm(v["x"], v["dt"], v["a"], v["bm"], v["cm"], v["skip"], v["z"], v["dt_bias"], v["h0"])
    wide = {k: v[k].repeat(b // 4096, 1, 1) for k in names}
    y, ht = m.ssm(wide["x"], wide["dt"], v["a"], wide["bm"], wide["cm"], v["skip"], wide["z"], v["dt_bias"], wide["h0"])
    assert torch.equal(y.view(-1, 4096, t, 1), few[0].expand(b // 4096, 4096, t, 1))
    assert torch.equal(ht.view(-1, 4096, 1, n), few[1].expand(b // 4096, 4096, 1, n))
    ref, err = ssmref.ssm(*(v[k] for k in ("x", "dt", "a", "bm", "cm", "skip", "z", "dt_bias", "h0")))
    compare(("y", "ht"), few, ref, err)


def test_ssm_step_of_many_sequences_and_channels():
    """65536 sequences of 4112 channels of 64 states, more workgroups than a launch has: they walk the sequences."""
    say("ssm step many")
    import torch
    q, m, b, d, n = Rand(65), mod(), 65536, 4112, 64
    x, dt = (q.normal(256, 1, d, dtype=torch.bfloat16) for _ in range(2))
    bm, cm = (q.normal(b, 1, n, dtype=torch.bfloat16) for _ in range(2))
    a, y = -q.uniform(d, n, lo=0.5, hi=2.0), torch.empty(b, 1, d, dtype=torch.bfloat16, device="cuda")
    wide = [p.repeat(b // 256, 1, 1) for p in (x, dt)] + [bm, cm]
    g = m.SsmDesc(1, b, 1, d, n, 1, a.data_ptr(), None, None, None)  # through the C ABI: no states in or out
    sq = [m.FhcSeq(p.data_ptr(), p.stride(0), p.stride(1)) for p in wide + [y]]
    rc = m._lib().fhc_ssm_forward(g, *sq[:4], None, None, sq[4], None, None, None, 0,
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0, m.fhconv.last_error()
    for at in (0, 4096, 65280, 65408):  # the last ones are a workgroup's second sequences
        cut = slice(at, at + 128)
        want = m.ssm(wide[0][cut], wide[1][cut], a, bm[cut], cm[cut])[0]
        assert torch.equal(y[cut], want), at


# ---- kernels that only larger calls take --------------------------------------------------------------------------

LARGER = [  # rows, c, f: few rows with four waves a workgroup, whole and odd widths; 128 x 128 tiles of an unsplit K, and
    (5, 72, 4100), (20, 65, 4099), (32, 200, 8192),  # their pairs of columns and single ones; 256 x 256 tiles likewise;
    (1003, 130, 2734), (1003, 130, 2735), (1003, 136, 2736), (2500, 130, 4102), (2500, 130, 4101),
    (40, 4200, 64), (40, 4096, 70),  # a K in 16 and more parts
]


@pytest.mark.parametrize("dtype,act", [("f16", "gelu"), ("bf16", "silu"), ("bf16", "none")])
@pytest.mark.parametrize("shape", LARGER, ids=str)
def test_linear_larger_calls(shape, dtype, act):
    say("linear larger", shape, dtype, act)
    linear_check(linear_inputs(Rand(sum(shape) + 5), *shape, types()[dtype]), act)


@pytest.mark.parametrize("shape", [(4, 1100, 4097, 4), (3, 700, 4096, 2)], ids=str)
def test_short_conv_several_items_a_thread(shape):
    """More chunks than workgroups' rows: the backward pass walks them."""
    say("short_conv items", shape)
    import torch
    conv_check(conv_inputs(Rand(sum(shape) + 5), *shape, torch.bfloat16, ragged=shape[2] % 2 == 1))


def test_stream_argument():
    """stream=: the work, and what it allocates, on that stream."""
    say("stream argument")
    import torch
    m, q = mod(), Rand(65)
    c = conv_inputs(q, 3, 40, 72, 4, torch.bfloat16)
    s = ssm_inputs(q, 3, 40, 72, 16, 1, torch.bfloat16)
    p = linear_inputs(q, 100, 72, 48, torch.bfloat16)
    kw = {k: s[k] for k in ("skip", "z", "dt_bias")}

    def run(**on):
        y, ht, states = m.ssm(s["x"], s["dt"], s["a"], s["bm"], s["cm"], h0=s["h0"], train=True, **kw, **on)
        out = (y, ht) + m.ssm_backward(s["x"], s["dt"], s["a"], s["bm"], s["cm"], states, s["dy"], dht=s["dht"], **kw, **on)
        out += m.short_conv(c["x"], c["w"], c["bias"], state=c["state"], **on)
        out += m.short_conv_backward(c["x"], c["w"], c["bias"], c["dy"], state=c["state"], dstate=c["dstate"], **on)
        y, kept = m.linear(p["x"], p["w"], p["bias"], p["residual"], "gelu", train=True, **on)
        return out + (y,) + m.linear_backward(p["x"], p["w"], kept, p["dy"], "gelu", **on)

    want = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = run(stream=stream)
    stream.synchronize()
    assert all(_same(a, b) for a, b in zip(got, want))
