"""The operators of a recurrent block on token rows (the pixels of a feature map over the frames of a stream, or the
tokens of sequences), as measurable cases: a gated linear recurrence, the norms around a block with its gate and the
scaled residual, and a gated feed-forward block, each forward and as a training step.

`run` computes them in their plain form, elementary torch operations in 32 bits, or, where `own` is true, through the
library (flyhigh-engine_amd/fhseq.py). Every case draws its inputs from its seed on the GPU.

The recurrence, per channel of every sequence (rate a constant, lam a weight, r and i the two gates' logits):
    log a_t = -rate * softplus(lam) * sigmoid(r_t)
    h_t     = a_t * h_(t-1) + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t
Positions at and past a sequence's length leave the state as it is, read nothing, and give 0.

The norms around a block (o the block's output, x the residual stream, gate one vector per group of rows):
    y = alpha * x + gate * w_post * o / rms(o)        rms(v) = sqrt(mean(v^2) + eps)
    u = w_pre * y / rms(y)                            the next block's input

The gated feed-forward block: y = (act(x wg^T) * (x wu^T)) wd^T.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
RATE, EPS = 8.0, 1e-6


def listed():
    return [
        # one token of each of 64 sequences with the state that a server holds between tokens: latency counts
        dict(name="glr_step", kind="glr_forward", b=64, t=1, d=2048, dtype="bf16", ragged=False, time_major=False),
        # a stream of 24 frames' feature maps at 1/16 of the 864x480 network (30 x 54 pixels of 128 channels): every
        # pixel carries a state from frame to frame, a frame's map is one time step in memory
        dict(name="glr_frames", kind="glr_forward", b=1620, t=24, d=128, dtype="f16", ragged=False, time_major=True),
        # one long sequence read into a state: few rows, a long axis
        dict(name="glr_long", kind="glr_forward", b=1, t=65536, d=2048, dtype="bf16", ragged=False, time_major=False),
        # a training step on sequences of different lengths, at an odd length and a width off the powers of two
        dict(name="glr_train_ragged", kind="glr_train", b=6, t=4099, d=1532, dtype="bf16", ragged=True,
             time_major=False),
        # the norms of one decoded token for each of 16 sequences
        dict(name="norm_step", kind="norm_forward", groups=16, rows=1, c=2048, dtype="bf16"),
        # a serving batch at an odd width, whose rows are not 16-byte aligned
        dict(name="norm_odd", kind="norm_forward", groups=3, rows=5003, c=1931, dtype="f16"),
        # a training step on the network's 1/8 feature maps: 8 images of 60 x 108 pixels, a gate vector per image
        dict(name="norm_train_maps", kind="norm_train", groups=8, rows=6480, c=128, dtype="f16"),
        # a training step on wide rows, four sequences with a gate each
        dict(name="norm_train_wide", kind="norm_train", groups=4, rows=4096, c=4096, dtype="bf16"),
        # one decoded token for each of 4 sequences: the weights are read for four rows
        dict(name="ffn_step", kind="ffn_forward", rows=4, c=2048, f=8192, act="silu", dtype="bf16"),
        # a serving batch at sizes that fill no tile
        dict(name="ffn_ragged", kind="ffn_forward", rows=1003, c=1020, f=2734, act="gelu", dtype="f16"),
        # a training step on the network's 1/8 feature maps, 8 images of 60 x 108 pixels: many rows, few channels
        dict(name="ffn_train_maps", kind="ffn_train", rows=51840, c=128, f=512, act="silu", dtype="f16"),
        # a training step at a size where the matrix products are all that counts
        dict(name="ffn_train_large", kind="ffn_train", rows=8192, c=2048, f=8192, act="silu", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["glr_forward", "glr_train", "norm_forward", "norm_train", "ffn_forward", "ffn_train"])
    dtype = rng.choice(["f16", "bf16"] if kind.startswith("ffn") else ["f16", "bf16", "bf16", "f32"])
    wide = 2 if dtype == "f32" else 1
    if kind.startswith("glr"):
        d = _log(rng, 32, 4096)
        d = d if rng.random() < 0.3 else max(8, d // 8 * 8)  # some widths are odd, most are not
        most = (1 << (26 if kind == "glr_train" else 27)) // (wide * d)  # of b * t
        t = _log(rng, 1, min(most, 65536))
        return dict(kind=kind, b=_log(rng, 1, min(most // t, 4096)), t=t, d=d, dtype=dtype, ragged=rng.random() < 0.4,
                    time_major=rng.random() < 0.3)
    if kind.startswith("norm"):
        c = _log(rng, 32, 8192)
        c = c if rng.random() < 0.3 else max(8, c // 8 * 8)
        groups = _log(rng, 1, 256)
        rows = _log(rng, 1, (1 << 26) // (wide * c * groups))
        return dict(kind=kind, groups=groups, rows=rows, c=c, dtype=dtype)
    c, f = _log(rng, 64, 4096), _log(rng, 128, 8192)
    if rng.random() < 0.7:
        c, f = max(8, c // 8 * 8), max(8, f // 8 * 8)
    rows = _log(rng, 1, min(65536, (1 << 37) // (c * f), (1 << 26) // c))
    return dict(kind=kind, rows=rows, c=c, f=f, act=rng.choice(["silu", "gelu"]), dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ty = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=ty):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if case["kind"].startswith("glr"):
        b, t, d = case["b"], case["t"], case["d"]

        def seq():
            return normal(t, b, d).transpose(0, 1) if case["time_major"] else normal(b, t, d)

        s["x"], s["r"], s["i"] = seq(), seq(), seq()
        # decays of 0.9 to 0.999 a step where the gate is open
        u = torch.rand(d, generator=g, device="cuda", dtype=torch.float64) * 0.099 + 0.9
        s["lam"] = torch.log(torch.expm1(-torch.log(u) / RATE)).float()
        s["h0"] = normal(b, d, dtype=torch.float32)
        s["lengths"] = None
        if case["ragged"]:  # a batch's longest sequence sets t; others may be empty
            n = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            n[0] = t
            s["lengths"] = n
        if case["kind"] == "glr_train":
            s["dy"], s["dht"] = seq(), normal(b, d, dtype=torch.float32)
    elif case["kind"].startswith("norm"):
        rows, c = case["groups"] * case["rows"], case["c"]
        s["x"], s["o"] = normal(rows, c), normal(rows, c, scale=3.0)
        s["w_post"] = (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(ty)
        s["w_pre"] = (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(ty)
        s["gate"] = normal(case["groups"], c, scale=0.5)
        s["alpha"] = math.sqrt(0.5)
        if case["kind"] == "norm_train":
            s["dy"], s["du"] = normal(rows, c), normal(rows, c)
    else:
        rows, c, f = case["rows"], case["c"], case["f"]
        s["x"] = normal(rows, c)
        s["wg"], s["wu"] = normal(f, c, scale=c ** -0.5), normal(f, c, scale=c ** -0.5)
        s["wd"] = normal(c, f, scale=f ** -0.5)
        if case["kind"] == "ffn_train":
            s["dy"] = normal(rows, c)
    return s


def _fhseq():
    pkg = os.path.join(ROOT, "flyhigh-engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import fhseq
    return fhseq


def _run_own(s):
    m, kind = _fhseq(), s["kind"]
    if kind == "glr_forward":
        return m.glr(s["x"], s["r"], s["i"], s["lam"], RATE, h0=s["h0"], lengths=s["lengths"])
    if kind == "glr_train":
        y, ht, states = m.glr(s["x"], s["r"], s["i"], s["lam"], RATE, h0=s["h0"], lengths=s["lengths"], train=True)
        grads = m.glr_backward(s["x"], s["r"], s["i"], s["lam"], states, s["dy"], RATE, dht=s["dht"],
                               lengths=s["lengths"])
        return (y, ht) + grads
    if kind == "norm_forward":
        return m.norm_block(s["x"], s["o"], s["w_post"], s["gate"], s["w_pre"], s["alpha"], EPS, s["rows"])
    if kind == "norm_train":
        out = m.norm_block(s["x"], s["o"], s["w_post"], s["gate"], s["w_pre"], s["alpha"], EPS, s["rows"])
        return out + m.norm_block_backward(s["x"], s["o"], s["w_post"], s["gate"], s["w_pre"], s["dy"], s["du"],
                                           s["alpha"], EPS, s["rows"])
    if kind == "ffn_forward":
        return m.ffn(s["x"], s["wg"], s["wu"], s["wd"], s["act"])
    y, saved = m.ffn(s["x"], s["wg"], s["wu"], s["wd"], s["act"], train=True)
    return (y,) + m.ffn_backward(s["x"], s["wg"], s["wu"], s["wd"], saved, s["dy"], s["act"])


def _scan(a, h):
    """h_t += a_t * h_(t-1) along dimension 1, by doubling: log2(T) elementwise passes."""
    k = 1
    while k < h.shape[1]:
        h = torch.cat([h[:, :k], h[:, k:] + a[:, k:] * h[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return h


def _plain_glr(s, train):
    x, r, i = s["x"].float(), s["r"].float(), s["i"].float()
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    sp = torch.nn.functional.softplus(s["lam"])
    la = -RATE * sp * sr
    a = torch.exp(la)
    m = torch.sqrt(-torch.expm1(2 * la))
    in_b = m * si * x
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(x.shape[1], device=x.device)[None, :] < s["lengths"][:, None])[:, :, None]
        a, in_b = torch.where(live, a, 1.0), torch.where(live, in_b, 0.0)
    h = _scan(a, torch.cat([(in_b[:, :1] + a[:, :1] * s["h0"][:, None]), in_b[:, 1:]], 1))
    y = h if live is None else torch.where(live, h, 0.0)
    out = (y.to(s["x"].dtype), h[:, -1].contiguous())
    if not train:
        return out
    dy = s["dy"].float()
    dy = dy if live is None else torch.where(live, dy, 0.0)
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dht"][:, None]], 1)
    # the adjoint runs the other way: g_t = dy_t + a_(t+1) g_(t+1)
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(nxt.flip(1), dy.flip(1)).flip(1)
    before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    # d(loss) / d(log a): a h_(t-1) from the decay, -a^2 / m from the input's normalisation
    dla = g * (a * before - torch.where(m > 0, a * a / m, 0.0) * si * x)
    db = g * m
    grads = [db * si, dla * la * (1 - sr), db * x * si * (1 - si)]
    dlam = dla * -RATE * sr
    if live is not None:
        grads = [torch.where(live, v, 0.0) for v in grads]
        dlam = torch.where(live, dlam, 0.0)
    dlam = (dlam.sum((0, 1), dtype=torch.float64) * torch.sigmoid(s["lam"].double())).float()
    return out + tuple(v.to(s["x"].dtype) for v in grads) + (dlam, g[:, 0] * a[:, 0])


def _plain_norm(s, train):
    x, o, ty = s["x"].float(), s["o"].float(), s["x"].dtype
    wp, wn = s["w_post"].float(), s["w_pre"].float()
    gate = s["gate"].float().repeat_interleave(s["rows"], 0)
    so = torch.rsqrt(o.square().mean(1, keepdim=True) + EPS)
    no = o * so
    y = s["alpha"] * x + gate * wp * no
    sy = torch.rsqrt(y.square().mean(1, keepdim=True) + EPS)
    ny = y * sy
    out = (y.to(ty), (wn * ny).to(ty))
    if not train:
        return out
    du = s["du"].float()
    dn = du * wn
    dtot = s["dy"].float() + sy * (dn - ny * (dn * ny).mean(1, keepdim=True))
    q = dtot * no
    dgate = (q.reshape(s["groups"], s["rows"], -1).sum(1, dtype=torch.float64) * wp.double()).float()
    dw_post = (q * gate).sum(0, dtype=torch.float64).float()
    dw_pre = (du * ny).sum(0, dtype=torch.float64).float()
    dno = dtot * gate * wp
    do = so * (dno - no * (dno * no).mean(1, keepdim=True))
    return out + ((s["alpha"] * dtot).to(ty), do.to(ty), dw_post, dgate, dw_pre)


def _gate(v, act):
    """act(v) = v * sigmoid(k(v)) and its derivative; gelu in its tanh form is v * sigmoid(2 c (v + 0.044715 v^3))."""
    if act == "silu":
        k, dk = v, 1.0
    else:
        c = 2 * math.sqrt(2 / math.pi)
        k, dk = c * (v + 0.044715 * v ** 3), c * (1 + 3 * 0.044715 * v * v)
    p = torch.sigmoid(k)
    return v * p, p + v * p * (1 - p) * dk


def _plain_ffn(s, train):
    x, wg, wu, wd, ty = s["x"].float(), s["wg"].float(), s["wu"].float(), s["wd"].float(), s["x"].dtype
    g, u = x @ wg.t(), x @ wu.t()
    ag, dag = _gate(g, s["act"])
    h = ag * u
    y = (h @ wd.t()).to(ty)
    if not train:
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * dag, dh * ag
    return (y, (dg @ wg + du @ wu).to(ty), (dg.t() @ x).to(ty), (du.t() @ x).to(ty), (dy.t() @ h).to(ty))


def run(state):
    if own:
        return _run_own(state)
    train = state["kind"].endswith("train")
    return (_plain_glr if state["kind"].startswith("glr") else
            _plain_norm if state["kind"].startswith("norm") else _plain_ffn)(state, train)


def work(case):
    e, train = (4 if case["dtype"] == "f32" else 2), case["kind"].endswith("train")
    if case["kind"].startswith("glr"):
        # forward: x, r, i in, y out, the state in and out; a training step: x, r, i once more and dy in, dx, dr, di out
        n, st = case["b"] * case["t"] * case["d"], 4 * case["b"] * case["d"]
        if not train:
            return {"bytes": n * e * 4 + 2 * st + 4 * case["d"], "flops": n * 20}
        return {"bytes": n * e * 8 + 4 * st + 8 * case["d"], "flops": n * 60}
    if case["kind"].startswith("norm"):
        # forward: x, o in, y, u out; a training step: x, o, dy, du in, y, u, dx, do out
        n, g, c = case["groups"] * case["rows"] * case["c"], case["groups"] * case["c"], case["c"]
        if not train:
            return {"bytes": n * e * 4 + e * (g + 2 * c), "flops": n * 10}
        return {"bytes": n * e * 8 + e * (g + 2 * c) + 4 * (g + 2 * c), "flops": n * 40}
    r, c, f = case["rows"], case["c"], case["f"]
    if not train:
        return {"bytes": e * (2 * r * c + 3 * c * f), "flops": 6 * r * c * f}
    # backward: dh, dx (two products), the three weights' gradients
    return {"bytes": e * (4 * r * c + 6 * c * f), "flops": 18 * r * c * f}


def _exact_glr(s, train):
    x, r, i, lam, h = (s[k].double() for k in ("x", "r", "i", "lam", "h0"))
    open_r, open_i = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    la = -RATE * torch.log1p(torch.exp(lam)) * open_r
    a = torch.exp(la)
    norm = torch.sqrt(-torch.expm1(2 * la))
    b = norm * open_i * x
    steps = x.shape[1]
    if s["lengths"] is not None:
        past = torch.arange(steps, device=x.device).view(1, -1, 1) >= s["lengths"].view(-1, 1, 1)
        a = a.masked_fill(past, 1.0)
        b = b.masked_fill(past, 0.0)
    hs = torch.empty_like(b)
    for t in range(steps):  # the definition, a step after the other
        h = torch.addcmul(b[:, t], a[:, t], h)
        hs[:, t] = h
    y = hs if s["lengths"] is None else hs.masked_fill(past, 0.0)
    out = [y, h]
    if not train:
        return out
    dy, g = s["dy"].double(), s["dht"].double()
    if s["lengths"] is not None:
        dy = dy.masked_fill(past, 0.0)
    gs = torch.empty_like(b)
    for t in range(steps - 1, -1, -1):
        g = g + dy[:, t]
        gs[:, t] = g
        g = g * a[:, t]
    dh0 = g
    if s["lengths"] is not None:
        gs = gs.masked_fill(past, 0.0)
    prev = torch.cat([s["h0"].double()[:, None], hs[:, :-1]], 1)
    dla = gs * (prev * a - open_i * x * a * a / norm)
    dsp = (dla * -RATE * open_r).sum((0, 1))
    return out + [gs * norm * open_i, dla * la * (1 - open_r), gs * norm * x * open_i * (1 - open_i),
                  dsp / (1 + torch.exp(-lam)), dh0]


def _exact_norm(s, train):
    names = ["x", "o", "w_post", "w_pre", "gate"]
    v = {k: s[k].double().requires_grad_(train) for k in names}
    shape = (s["groups"], s["rows"], -1)
    x, o = v["x"].view(shape), v["o"].view(shape)
    y = s["alpha"] * x + v["gate"][:, None] * v["w_post"] * o / torch.sqrt((o * o).mean(2, keepdim=True) + EPS)
    u = v["w_pre"] * y / torch.sqrt((y * y).mean(2, keepdim=True) + EPS)
    out = [w.detach().reshape(s["x"].shape) for w in (y, u)]
    if not train:
        return out
    torch.autograd.backward((y, u), (s["dy"].double().view(shape), s["du"].double().view(shape)))
    return out + [v[k].grad for k in ("x", "o", "w_post", "gate", "w_pre")]


def _exact_ffn(s, train):
    v = {k: s[k].double().requires_grad_(train) for k in ("x", "wg", "wu", "wd")}
    g = torch.mm(v["x"], v["wg"].t())
    if s["act"] == "silu":
        ag = g / (1 + torch.exp(-g))
    else:
        ag = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    y = torch.mm(ag * torch.mm(v["x"], v["wu"].t()), v["wd"].t())
    if not train:
        return y
    y.backward(s["dy"].double())
    return [y.detach()] + [v[k].grad for k in ("x", "wg", "wu", "wd")]


def exact(case, seed):
    s = prepare(case, seed)
    train = case["kind"].endswith("train")
    return (_exact_glr if case["kind"].startswith("glr") else
            _exact_norm if case["kind"].startswith("norm") else _exact_ffn)(s, train)
