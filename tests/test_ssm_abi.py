"""What the short convolution, the selective scan and the product with its epilogue refuse (include/fhc_seq.h): every
refusal is an error status with a message before any device work, so these run without a GPU; the pointers are never
followed."""
import ctypes

import pytest

import fhtest  # noqa: F401
from test_seq_abi import P, mod, refused


def ref(v):
    return None if v is None else ctypes.byref(v)


def seq(v):
    return None if v is None else ctypes.byref(mod().FhcSeq(*v))


def conv_call(back, **kw):
    m = mod()
    a = dict(dtype=1, act=0, b=2, t=5, d=8, k=4, w=P, bias=P, lengths=None)
    s = {n: (P, 40, 8) for n in ("x", "y", "dy", "dx")}
    p = dict(state=P, state_out=P, dstate_out=P, dw=P, dbias=P, dstate=P, ws=P, ws_bytes=1 << 40)
    for d in (a, s, p):
        d.update({k: v for k, v in kw.items() if k in d})
    g = None if kw.get("desc", 1) is None else ctypes.byref(m.ShortConvDesc(*a.values()))
    L = m._lib()
    if back:
        return L.fhc_short_conv_backward(g, seq(s["x"]), p["state"], seq(s["dy"]), p["dstate_out"], seq(s["dx"]), p["dw"],
                                         p["dbias"], p["dstate"], p["ws"], p["ws_bytes"], None)
    return L.fhc_short_conv_forward(g, seq(s["x"]), p["state"], seq(s["y"]), p["state_out"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dtype=3), "dtype 3"), (dict(act=1), "act 1"), (dict(k=1), "1 taps"),
    (dict(k=5), "5 taps"), (dict(b=1 << 20, d=1 << 12), "columns"), (dict(t=0xFFFFFFFF), "steps"), (dict(w=None), "null w"),
    (dict(w=P + 1), "not aligned"), (dict(bias=P + 1), "not aligned"), (dict(lengths=P + 2), "not aligned"),
    (dict(x=None), "null x"), (dict(x=(None, 40, 8)), "null pointer of x"), (dict(y=(P + 1, 40, 8)), "not aligned"),
    (dict(y=(P, 40, 7)), "overlap"), (dict(y=(P, 3, 8)), "overlap"), (dict(state=P + 1), "not aligned"),
    (dict(state_out=P + 1), "not aligned"),
])
def test_short_conv_forward_refuses(bad, text):
    refused(conv_call(False, **bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dy=None), "null dy"), (dict(dx=(P, 40, 4)), "overlap"),
    (dict(dw=P + 2), "not aligned"), (dict(dbias=P + 2), "not aligned"), (dict(dstate=P + 1), "not aligned"),
    (dict(dstate_out=P + 1), "not aligned"), (dict(ws=None), "null workspace"), (dict(ws_bytes=8), "workspace of 8"),
    (dict(ws=P + 16), "256-byte"),
])
def test_short_conv_backward_refuses(bad, text):
    refused(conv_call(True, **bad), text)


def test_short_conv_nothing_to_do_is_fine():
    assert conv_call(False, b=0) == 0 and conv_call(False, d=0) == 0 and conv_call(True, d=0) == 0
    assert conv_call(True, b=0, dw=None, dbias=None) == 0
    assert mod()._lib().fhc_short_conv_workspace_bytes(None) == 0


def ssm_call(back, **kw):
    m = mod()
    a = dict(dtype=1, b=2, t=5, d=8, n=4, groups=2, a=P, dt_bias=P, skip=P, lengths=None)
    s = {n: (P, 40, 8) for n in ("x", "dt", "bm", "cm", "z", "y", "dy", "dx", "ddt", "dbm", "dcm", "dz")}
    p = dict(h0=P, ht=P, states=P, dht=P, da=P, ddt_bias=P, dskip=P, dh0=P, ws=P, ws_bytes=1 << 40)
    for d in (a, s, p):
        d.update({k: v for k, v in kw.items() if k in d})
    g = None if kw.get("desc", 1) is None else ctypes.byref(m.SsmDesc(*a.values()))
    L = m._lib()
    ins = [seq(s[n]) for n in ("x", "dt", "bm", "cm", "z")]
    if back:
        return L.fhc_ssm_backward(g, *ins, p["states"], seq(s["dy"]), p["dht"],
                                  *(seq(s[n]) for n in ("dx", "ddt", "dbm", "dcm", "dz")), p["da"], p["ddt_bias"],
                                  p["dskip"], p["dh0"], p["ws"], p["ws_bytes"], None)
    return L.fhc_ssm_forward(g, *ins, p["h0"], seq(s["y"]), p["ht"], p["states"], p["ws"], p["ws_bytes"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dtype=5), "dtype 5"), (dict(n=0), "0 states"), (dict(n=65), "65 states"),
    (dict(groups=0), "0 groups"), (dict(groups=3), "3 groups of 8"), (dict(b=1 << 20, d=1 << 12), "columns"),
    (dict(t=0xFFFFFFFF), "steps"), (dict(a=None), "null a"), (dict(a=P + 2), "not aligned"),
    (dict(dt_bias=P + 2), "not aligned"), (dict(skip=P + 1), "not aligned"), (dict(lengths=P + 1), "not aligned"),
    (dict(x=None), "null x"), (dict(dt=(None, 40, 8)), "null pointer of dt"), (dict(bm=(P + 1, 40, 8)), "not aligned"),
    (dict(cm=None), "null cm"), (dict(z=(P + 1, 40, 8)), "not aligned"), (dict(y=(P, 40, 4)), "overlap"),
    (dict(y=None), "null y"), (dict(h0=P + 2), "not aligned"), (dict(ht=P + 2), "not aligned"),
    (dict(states=P + 16), "256-byte"),
])
def test_ssm_forward_refuses(bad, text):
    refused(ssm_call(False, **bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(states=None), "null states"), (dict(states=P + 8), "256-byte"),
    (dict(dy=None), "null dy"), (dict(dx=(P, 40, 4)), "overlap"), (dict(ddt=None), "null ddt"),
    (dict(dbm=(P, 40, 7)), "overlap"), (dict(dcm=None), "null dcm"), (dict(dz=None), "null dz"),
    (dict(z=None), "dz without z"), (dict(da=P + 1), "not aligned"), (dict(dh0=P + 2), "not aligned"),
    (dict(ws=None), "null workspace"), (dict(ws_bytes=16), "workspace of 16"), (dict(ws=P + 128), "256-byte"),
])
def test_ssm_backward_refuses(bad, text):
    refused(ssm_call(True, **bad), text)


def test_ssm_workspace_is_checked_where_time_is_cut():
    m = mod()
    g = m.SsmDesc(1, 1, 4000, 64, 16, 1, P, None, None, None)
    need = m._lib().fhc_ssm_workspace_bytes(g, 0)
    assert need > 0
    s = {n: (P, 64 * 4000, 64) for n in ("x", "dt", "bm", "cm", "z", "y")}
    kw = dict(b=1, t=4000, d=64, n=16, groups=1, **s)
    refused(ssm_call(False, ws=None, **kw), "null workspace")
    refused(ssm_call(False, ws_bytes=need - 1, **kw), "needed")


def test_ssm_nothing_to_do_is_fine():
    assert ssm_call(False, b=0) == 0 and ssm_call(False, d=0) == 0
    none = dict(da=None, ddt_bias=None, dskip=None)
    assert ssm_call(True, b=0, **none) == 0 and ssm_call(True, d=0, t=0, **none) == 0
    L = mod()._lib()
    assert L.fhc_ssm_states_bytes(None) == 0 and L.fhc_ssm_workspace_bytes(None, 1) == 0


def linear_call(back, **kw):
    m = mod()
    a = dict(dtype=1, act=0, rows=100, c=16, f=24)
    r = dict(x=(P, 16), residual=(P, 24), y=(P, 24), dy=(P, 24), dx=(P, 16))
    p = dict(w=P, bias=P, saved=P, dw=P, dbias=P, ws=P, ws_bytes=1 << 40)
    for d in (a, r, p):
        d.update({k: v for k, v in kw.items() if k in d})
    d = None if kw.get("desc", 1) is None else ctypes.byref(m.LinearDesc(*a.values()))
    r = {k: None if v is None else ctypes.byref(m.FhcRows(*v)) for k, v in r.items()}
    L = m._lib()
    if back:
        return L.fhc_linear_backward(d, r["x"], p["w"], p["saved"], r["dy"], r["dx"], p["dw"], p["dbias"], p["ws"],
                                     p["ws_bytes"], None)
    return L.fhc_linear_forward(d, r["x"], p["w"], p["bias"], r["residual"], r["y"], p["saved"], p["ws"], p["ws_bytes"],
                                None)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dtype=2), "neither f16 nor bf16"), (dict(act=3), "act 3"),
    (dict(f=(1 << 20) + 1), "channels"), (dict(rows=0x7FFFFF01), "rows"), (dict(x=None), "null x"),
    (dict(x=(P, 15)), "apart"), (dict(w=None), "null w"), (dict(w=P + 1), "not aligned"), (dict(y=(None, 24)), "null pointer"),
    (dict(y=(P, 23)), "apart"), (dict(residual=(P, 20)), "apart"), (dict(residual=(None, 24)), "null pointer of residual"),
    (dict(bias=P + 1), "not aligned"), (dict(saved=P + 16), "saved is not"), (dict(ws=None), "null workspace"),
    (dict(ws_bytes=16), "workspace of 16"), (dict(ws=P + 128), "256-byte"),
])
def test_linear_forward_refuses(bad, text):
    refused(linear_call(False, **bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dy=None), "null dy"), (dict(dy=(P, 23)), "apart"), (dict(x=None), "null x"),
    (dict(dx=(P, 15)), "apart"), (dict(w=None), "null w"), (dict(saved=None), "null saved"),
    (dict(saved=P + 8), "saved is not"), (dict(dw=P + 1), "not aligned"), (dict(dbias=P + 2), "not aligned"),
    (dict(ws=None), "null workspace"), (dict(ws_bytes=16), "workspace of 16"),
])
def test_linear_backward_refuses(bad, text):
    refused(linear_call(True, **bad), text)


def test_linear_nothing_to_do_is_fine():
    assert linear_call(False, rows=0) == 0 and linear_call(False, f=0) == 0
    assert linear_call(True, rows=0, x=None, dy=None, dx=None, dw=None, dbias=None) == 0
    m = mod()
    L = m._lib()
    assert L.fhc_linear_workspace_bytes(None, 0) == 0 and L.fhc_linear_saved_bytes(None) == 0
    assert L.fhc_linear_saved_bytes(m.LinearDesc(1, 2, 100, 16, 24)) == 0  # no activation: nothing to keep


def test_launches_of_too_many_threads_are_refused():
    m = mod()
    far = (P, 1, 1)
    s = {n: far for n in ("x", "dt", "bm", "cm", "z", "y")}
    refused(ssm_call(False, b=0x7FFFFFFF, t=20, d=1, n=64, groups=1, ws_bytes=1 << 62, **s), "too many workgroups")
    refused(conv_call(False, b=0x3FFFFFFF, t=4096, d=1, x=far, y=far), "too many workgroups")
    assert m is mod()


def test_tensors_are_checked_before_the_call():
    import torch
    m = mod()
    x, a, bc = torch.zeros(2, 3, 4), torch.zeros(4, 5), torch.zeros(2, 3, 5)
    with pytest.raises(m.FhcError, match="current GPU"):
        m.ssm(x, x, a, bc, bc)
    with pytest.raises(m.FhcError, match="f16, bf16 or f32"):
        m.ssm(x.double(), x, a, bc, bc)
    with pytest.raises(m.FhcError, match="current GPU"):
        m.short_conv(x, torch.zeros(4, 3))
    with pytest.raises(m.FhcError, match="sequences, steps, channels"):
        m.short_conv(x[0], torch.zeros(4, 3))
    with pytest.raises(m.FhcError, match="none of silu, none"):
        m.short_conv(x, torch.zeros(4, 3), act="gelu")
    with pytest.raises(m.FhcError, match="rows, channels"):
        m.linear(x, a)
    with pytest.raises(m.FhcError, match="none of silu, gelu, none"):
        m.linear(x[0], a, act="relu")


def test_tensors_that_require_gradients_are_refused_while_autograd_records():
    import torch
    m = mod()
    x, a, bc, d, rows = torch.zeros(2, 3, 4), torch.zeros(4, 5), torch.zeros(2, 3, 5), torch.zeros(4), torch.zeros(6, 4)
    states, w, st = torch.zeros(1, dtype=torch.uint8), torch.zeros(4, 3), torch.zeros(2, 2, 4)
    calls = [(m.short_conv, [x, w, d]), (m.short_conv_backward, [x, w, d, x]), (m.ssm, [x, x, a, bc, bc, d, x, d]),
             (m.ssm_backward, [x, x, a, bc, bc, states, x, d, x, d]), (m.linear, [rows, w.t().contiguous(), w[0], rows]),
             (m.linear_backward, [rows, w.t().contiguous(), None, rows])]
    for call, args in calls:
        for k, t in enumerate(args):
            if t is None or t is states:
                continue
            with pytest.raises(m.FhcError, match="requires gradients"):
                call(*(args[:k] + [t.clone().requires_grad_()] + args[k + 1:]))
    with pytest.raises(m.FhcError, match="requires gradients"):
        m.short_conv(x, w, state=st.requires_grad_())


def test_ssm_workspace_is_the_same_with_and_without_lengths():
    m = mod()
    for n, t, d in ((16, 2051, 1532), (64, 512, 1024), (3, 100, 64)):
        for back in (0, 1):
            plain, ragged = (m._lib().fhc_ssm_workspace_bytes(m.SsmDesc(1, 6, t, d, n, 2, P, None, None, q), back)
                             for q in (None, P))
            assert plain == ragged
