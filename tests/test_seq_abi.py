"""What the operators on rows of channels refuse (include/fhc_seq.h): every refusal is an error status with a message
before any device work, so these run without a GPU; the pointers are never followed."""
import ctypes

import pytest

import fhtest  # noqa: F401

P = 0x10000  # an aligned address that nothing reads


def mod():
    import fhseq
    return fhseq


def glr_args(**kw):
    m = mod()
    a = dict(dtype=1, b=2, t=5, d=8, rate=8.0, lam=P, lengths=None)
    seqs = dict(x=(P, 40, 8), r=(P, 40, 8), i=(P, 40, 8), y=(P, 40, 8), dy=(P, 40, 8), dx=(P, 40, 8), dr=(P, 40, 8),
                di=(P, 40, 8))
    a.update({k: v for k, v in kw.items() if k in a})
    seqs.update({k: v for k, v in kw.items() if k in seqs})
    g = ctypes.byref(m.GlrDesc(*a.values()))
    return g, {k: None if v is None else ctypes.byref(m.FhcSeq(*v)) for k, v in seqs.items()}


def glr_forward(**kw):
    L = mod()._lib()
    g, s = glr_args(**kw)
    return L.fhc_glr_forward(kw.get("desc", g), s["x"], s["r"], s["i"], None, s["y"], None, None, kw.get("ws", P),
                             kw.get("ws_bytes", 1 << 40), None)


def glr_backward(**kw):
    L = mod()._lib()
    g, s = glr_args(**kw)
    return L.fhc_glr_backward(g, s["x"], s["r"], s["i"], kw.get("states", P), s["dy"], None, s["dx"], s["dr"], s["di"],
                              kw.get("dlam", P), None, kw.get("ws", P), kw.get("ws_bytes", 1 << 40), None)


def refused(rc, text):
    msg = mod().fhconv.last_error()
    assert rc == -1 and text in msg, (rc, msg)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), "dtype 3"), (dict(rate=float("nan")), "rate"), (dict(rate=-1.0), "rate"),
    (dict(b=1 << 20, d=1 << 12), "columns"), (dict(t=0xFFFFFFFF), "steps"), (dict(lam=None), "null lam"),
    (dict(x=None), "null x"), (dict(r=(None, 40, 8)), "null pointer of r"), (dict(i=(P + 1, 40, 8)), "not aligned"),
    (dict(y=(P, 40, 4)), "overlap"), (dict(y=(P, 3, 8)), "overlap"), (dict(desc=None), "null descriptor"),
])
def test_glr_forward_refuses(bad, text):
    refused(glr_forward(**bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(states=None), "null states"), (dict(dlam=None), "null dlam"), (dict(dy=None), "null dy"),
    (dict(dx=(P, 40, 4)), "overlap"), (dict(ws=None), "null workspace"), (dict(ws_bytes=8), "workspace of 8"),
    (dict(ws=P + 16), "256-byte"), (dict(dtype=9), "dtype 9"),
])
def test_glr_backward_refuses(bad, text):
    refused(glr_backward(**bad), text)


def test_glr_workspace_is_checked_where_chunks_are_chained():
    g, _ = glr_args(t=1000)
    need = mod()._lib().fhc_glr_workspace_bytes(g, 0)
    assert need > 0
    kw = dict(t=1000, x=(P, 8000, 8), r=(P, 8000, 8), i=(P, 8000, 8), y=(P, 8000, 8))
    refused(glr_forward(ws=None, **kw), "null workspace")
    refused(glr_forward(ws_bytes=need - 1, **kw), "needed")


def test_glr_nothing_to_do_is_fine():
    assert glr_forward(b=0) == 0 and glr_forward(d=0) == 0 and glr_backward(d=0) == 0
    L = mod()._lib()
    assert L.fhc_glr_states_bytes(None) == 0 and L.fhc_glr_workspace_bytes(None, 1) == 0


def norm_call(back, **kw):
    m = mod()
    L = m._lib()
    a = dict(dtype=1, rows=6, c=16, rows_per_group=3, alpha=1.0, eps=1e-6, w_post=P, w_pre=P, gate=P)
    r = {k: (P, 16) for k in ("x", "o", "y", "u", "dy", "du", "dx", "dout")}
    a.update({k: v for k, v in kw.items() if k in a})
    r.update({k: v for k, v in kw.items() if k in r})
    n = None if kw.get("desc", 1) is None else ctypes.byref(m.NormDesc(*a.values()))
    r = {k: None if v is None else ctypes.byref(m.FhcRows(*v)) for k, v in r.items()}
    if back:
        return L.fhc_norm_block_backward(n, r["x"], r["o"], r["dy"], r["du"], r["dx"], r["dout"], kw.get("dw_post", P),
                                         kw.get("dgate", P), P, kw.get("ws", P), kw.get("ws_bytes", 1 << 40), None)
    return L.fhc_norm_block(n, r["x"], r["o"], r["y"], r["u"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dtype=4), "dtype 4"), (dict(c=16385), "channels"),
    (dict(rows=1 << 31), "rows"), (dict(rows_per_group=0), "rows_per_group"), (dict(alpha=float("inf")), "alpha"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(w_pre=P + 1), "not aligned"),
    (dict(x=None), "null x"), (dict(o=(None, 16)), "null pointer of o"), (dict(y=(P, 15)), "apart"),
    (dict(u=(P + 1, 16)), "not aligned"), (dict(y=None, u=None), "neither y nor u"), (dict(o=None), "without o"),
])
def test_norm_block_refuses(bad, text):
    refused(norm_call(False, **bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(dx=None), "null dx"), (dict(dout=None), "null dout"), (dict(dy=None, du=None), "neither dy nor du"),
    (dict(o=None), "without o"), (dict(gate=None), "dgate without a gate"), (dict(ws=None), "null workspace"),
    (dict(ws_bytes=100), "workspace of 100"), (dict(ws=P + 8), "256-byte"), (dict(c=20000), "channels"),
])
def test_norm_block_backward_refuses(bad, text):
    refused(norm_call(True, **bad), text)


def test_norm_block_nothing_to_do_is_fine():
    assert norm_call(False, rows=0) == 0 and norm_call(False, c=0) == 0 and norm_call(True, c=0) == 0


def ffn_call(back, **kw):
    m = mod()
    L = m._lib()
    a = dict(dtype=1, act=0, rows=100, c=16, f=24)
    r = {k: (P, 16) for k in ("x", "y", "dy", "dx")}
    w = dict(wg=P, wu=P, wd=P, saved=P, dwg=P, dwu=P, dwd=P, ws=P, ws_bytes=1 << 40)
    for d in (a, r, w):
        d.update({k: v for k, v in kw.items() if k in d})
    d = None if kw.get("desc", 1) is None else ctypes.byref(m.FfnDesc(*a.values()))
    r = {k: None if v is None else ctypes.byref(m.FhcRows(*v)) for k, v in r.items()}
    if back:
        return L.fhc_ffn_backward(d, r["x"], w["wg"], w["wu"], w["wd"], w["saved"], r["dy"], r["dx"], w["dwg"],
                                  w["dwu"], w["dwd"], w["ws"], w["ws_bytes"], None)
    return L.fhc_ffn_forward(d, r["x"], w["wg"], w["wu"], w["wd"], r["y"], w["saved"], w["ws"], w["ws_bytes"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(desc=None), "null descriptor"), (dict(dtype=2), "neither f16 nor bf16"), (dict(act=2), "act 2"),
    (dict(c=(1 << 20) + 1), "channels"), (dict(rows=0x7FFFFF01), "rows"), (dict(x=None), "null x"),
    (dict(y=(None, 16)), "null pointer of y"), (dict(y=(P, 15)), "apart"), (dict(x=(P + 1, 16)), "not aligned"),
    (dict(wu=None), "null wu"), (dict(wd=P + 1), "not aligned"), (dict(saved=P + 16), "saved is not"),
    (dict(ws=None), "null workspace"), (dict(ws_bytes=16), "workspace of 16"), (dict(ws=P + 128), "256-byte"),
])
def test_ffn_forward_refuses(bad, text):
    refused(ffn_call(False, **bad), text)


@pytest.mark.parametrize("bad,text", [
    (dict(dy=None), "null dy"), (dict(saved=None), "null saved"), (dict(saved=P + 8), "saved is not"),
    (dict(dx=(P, 3)), "apart"), (dict(wg=None), "null wg"), (dict(dwu=P + 1), "not aligned"),
    (dict(ws=None), "null workspace"), (dict(ws_bytes=16), "workspace of 16"), (dict(dtype=7), "neither"),
])
def test_ffn_backward_refuses(bad, text):
    refused(ffn_call(True, **bad), text)


def test_ffn_nothing_to_do_is_fine():
    assert ffn_call(False, rows=0) == 0 and ffn_call(False, c=0) == 0 and ffn_call(True, c=0) == 0


def test_tensors_are_checked_before_the_call():
    import torch
    m = mod()
    x = torch.zeros(2, 3, 4)
    with pytest.raises(m.FhcError, match="current GPU"):
        m.glr(x, x, x, torch.zeros(4))
    with pytest.raises(m.FhcError, match="f16, bf16 or f32"):
        m.glr(x.double(), x, x, torch.zeros(4))
    with pytest.raises(m.FhcError, match="rows, channels"):
        m.norm_block(x, x, None, None, None)


def test_launches_of_too_many_threads_are_refused():
    """One column of 2^31 steps and 2^25 groups of 64 rows each ask for more threads than a launch has."""
    refused(glr_forward(b=1, d=1, t=0x7FFFFF00), "too many workgroups")
    refused(glr_backward(b=1, d=1, t=0x7FFFFF00), "too many workgroups")
    m = mod()
    L = m._lib()
    n = m.NormDesc(1, 0x7FFFFFFF, 1, 64, 1.0, 1e-6, None, None, P)
    rows = ctypes.byref(m.FhcRows(P, 1))
    refused(L.fhc_norm_block_backward(ctypes.byref(n), rows, rows, rows, rows, rows, rows, P, P, P, P, 1 << 40, None),
            "too many workgroups")


@pytest.mark.parametrize("c,f", [(0, 4096), (4096, 0), (300, 520), (2048, 8192)])
def test_ffn_sizes_without_rows(c, f):
    """A batch may be empty, and so may the channels or the features: the sizes are those of the copies of the weights."""
    import ctypes
    m = mod()
    L = m._lib()
    for rows in (0, 1, 100):
        d = ctypes.byref(m.FfnDesc(1, 0, rows, c, f))
        for back in (0, 1):
            assert L.fhc_ffn_workspace_bytes(d, back) < 1 << 30
        assert L.fhc_ffn_saved_bytes(d) < 1 << 30


def test_ffn_backward_without_rows_reads_no_descriptor():
    assert ffn_call(True, rows=0, x=None, dy=None, dx=None, dwg=None, dwu=None, dwd=None) == 0
    assert ffn_call(True, rows=0, x=(None, 0), dy=(None, 0), dx=(None, 0), dwg=None, dwu=None, dwd=None) == 0
    assert ffn_call(False, rows=0, x=None, y=None) == 0


def test_tensors_that_require_gradients_are_refused_while_autograd_records():
    import torch
    m = mod()
    x, rows, w = torch.zeros(2, 3, 4), torch.zeros(5, 4), torch.zeros(6, 4)
    d, lam, c = w.t().contiguous(), torch.zeros(4), torch.ones(4)
    states = torch.zeros(1, dtype=torch.uint8)
    calls = [(m.glr, [x, x, x, lam]), (m.glr_backward, [x, x, x, lam, states, x]),
             (m.norm_block, [rows, rows, c, None, c]), (m.norm_block_backward, [rows, rows, c, None, c, rows, rows]),
             (m.ffn, [rows, w, w, d]), (m.ffn_backward, [rows, w, w, d, states, rows])]
    for call, args in calls:
        for k, a in enumerate(args):
            if a is None or a is states:
                continue
            grad = args[:k] + [a.clone().requires_grad_()] + args[k + 1:]
            with pytest.raises(m.FhcError, match="requires gradients"):
                call(*grad)
            with torch.no_grad(), pytest.raises(m.FhcError, match="current GPU"):  # the next check
                call(*grad)
    with pytest.raises(m.FhcError, match="requires gradients"):
        m.glr(x, x, x, lam, h0=torch.zeros(2, 4, requires_grad=True))


@pytest.mark.parametrize("rows,c,f", [(51840, 128, 512), (6000, 33, 4096), (40000, 250, 1 << 20)])
def test_ffn_in_one_kernel_takes_no_room_for_the_hidden_layer(rows, c, f):
    import ctypes
    m = mod()
    up = lambda n: (n + 7) // 8 * 8  # noqa: E731
    copies = 2 * (rows * up(c) + 2 * f * up(c) + c * up(f)) + 4 * 256  # of the rows and the three weights
    assert m._lib().fhc_ffn_workspace_bytes(ctypes.byref(m.FfnDesc(0, 0, rows, c, f)), 0) <= copies
