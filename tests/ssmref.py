"""Plain 64-bit forms of the short convolution, the selective scan and the product with its epilogue, with a bound on the
error of a 32-bit evaluation beside each result (in the way of seqref.py): U is f32's half step, and each intermediate's
bound is its inputs' carried through the operation plus its own roundings. An output may be off by its bound plus half a
step of its type."""
import torch

from seqref import U, _act, half_step


# The vector unit's exponential gives 0 where its result is below the smallest normal number: a decay is off by up to that,
# and so is a sum of products.
TINY = 2.0 ** -126


def live_of(b, t, lengths, device):
    live = torch.ones((b, t, 1), dtype=torch.bool, device=device)
    if lengths is not None:
        live = (torch.arange(t, device=device)[None] < lengths.clamp(0, t)[:, None])[:, :, None]
    return live


def short_conv(x, w, bias, act, state=None, lengths=None, dy=None, dstate=None):
    """(results, bounds): y, the state that is left, and with dy also dx, dw, dbias, the state's gradient."""
    b, t, d = x.shape
    k, dev = w.shape[1], x.device
    live = live_of(b, t, lengths, dev)
    x, w = torch.where(live, x.double(), 0.0), w.double()
    before = torch.zeros((b, k - 1, d), dtype=torch.float64, device=dev) if state is None else state.double()
    bias = torch.zeros(d, dtype=torch.float64, device=dev) if bias is None else bias.double()
    e = torch.cat([before, x], 1)
    v, size = bias.expand(b, t, d), bias.abs().expand(b, t, d)
    for j in range(k):
        v, size = v + w[:, j] * e[:, j:j + t], size + (w[:, j] * e[:, j:j + t]).abs()
    ev = (k + 1) * U * size  # a chain of k fused additions
    if act == "silu":
        a, da = _act(v, "silu")
        ea, eda = 1.2 * ev + 64 * U * a.abs(), 1.2 * ev + 64 * U * (da.abs() + 1)
    else:
        a, da, ea, eda = v, torch.ones_like(v), ev, torch.zeros_like(v)
    at = live.sum(1)[:, :1] + torch.arange(k - 1, device=dev)[None]
    seqs = torch.arange(b, device=dev)[:, None]
    zero = lambda q: torch.where(live, q, 0.0)  # noqa: E731
    end = e[seqs, at]
    res, err = [zero(a), end], [zero(ea), torch.zeros_like(end)]
    if dy is None:
        return res, err
    dv, edv = zero(dy.double() * da), zero(dy.double().abs() * eda + 2 * U * (dy.double() * da).abs())
    de, ede, sde = torch.zeros_like(e), torch.zeros_like(e), torch.zeros_like(e)
    for j in range(k):
        de[:, j:j + t] += w[:, j] * dv
        ede[:, j:j + t] += w[:, j].abs() * edv
        sde[:, j:j + t] += (w[:, j] * dv).abs()
    if dstate is not None:
        de[seqs, at] += dstate.double()
        sde[seqs, at] += dstate.double().abs()
    ede += (k + 2) * U * sde
    # a thread adds the terms of its chunks of 32 steps, 256 at most are added behind it, the rest in f64; past 2048
    # workgroups of at least 64 channels a thread has several chunks
    chain = (32 + 256 + b * t * d / (1 << 17)) * U
    dw = torch.stack([(dv * e[:, j:j + t]).sum((0, 1)) for j in range(k)], 1)
    edw = torch.stack([(edv * e[:, j:j + t].abs() + chain * (dv * e[:, j:j + t]).abs()).sum((0, 1)) for j in range(k)], 1)
    res += [zero(de[:, k - 1:]), dw, dv.sum((0, 1)), de[:, :k - 1]]
    err += [zero(ede[:, k - 1:]), edw, (edv + chain * dv.abs()).sum((0, 1)), ede[:, :k - 1]]
    return res, err


def ssm(x, dt, a, bm, cm, skip=None, z=None, dt_bias=None, h0=None, lengths=None, dy=None, dht=None):
    """(results, bounds): y, ht, and with dy also dx, ddt, da, dbm, dcm, dskip, dz, ddt_bias, dh0."""
    b, t, d = x.shape
    n, dev, f64 = a.shape[1], x.device, torch.float64
    groups = bm.shape[2] // n
    live = live_of(b, t, lengths, dev)
    zero = lambda q: torch.where(live, q, 0.0)  # noqa: E731
    x, dt, bm, cm = (zero(q.double()) for q in (x, dt, bm, cm))
    a = a.double()
    skip = torch.zeros(d, dtype=f64, device=dev) if skip is None else skip.double()
    v = dt if dt_bias is None else dt + dt_bias.double()
    share = torch.arange(d, device=dev) // (d // groups)
    step = zero(torch.nn.functional.softplus(v, threshold=1000))
    # softplus: the sum's rounding, the exponential's argument and result, the polynomial: (3 |v| + 16) U of the step
    rel = (3 * v.abs() + 16) * U
    u = step * x
    if z is None:
        gate, egate, dgate, edgate = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    else:
        z = zero(z.double())
        gate, dgate = _act(z, "silu")
        egate, edgate = (z.abs() + 16) * U * gate.abs(), 64 * U * (dgate.abs() + 1)
    vec = lambda m: m.view(b, t, groups, n)  # noqa: E731
    bv, cv = vec(bm), vec(cm)
    h = torch.zeros((b, d, n), dtype=f64, device=dev) if h0 is None else h0.double()
    e = torch.zeros_like(h)
    # cut into segments, a state comes through products of decays of f32 sums of up to t steps: exp(-s) s <= 0.37
    fold = 0.4 * t * U if t > 64 else 0.0
    hs, es, ps, eps = [h], [e], [], []
    decay = lambda i: torch.exp(step[:, i, :, None] * a)  # noqa: E731
    erel = lambda i: (step[:, i, :, None] * a).abs() * (rel[:, i, :, None] + 4 * U) + 6 * U  # noqa: E731
    top = torch.zeros_like(h)
    for i in range(t):
        q, on = decay(i), live[:, i, :, None]
        inp = u[:, i, :, None] * bv[:, i, share]
        e = q * e + on * (erel(i) * (q * h).abs() + (rel[:, i, :, None] + 6 * U) * inp.abs() + TINY * (h.abs() + 1))
        h = q * h + inp
        top = torch.maximum(top, h.abs())
        hs.append(h), es.append(e)
        ch, cs = cv[:, i, share], cv[:, i, share].abs()
        ps.append((ch * h).sum(2))
        eps.append((cs * (e + fold * top) + (n + 6) * U * (ch * h).abs()).sum(2))
    stack = lambda q: torch.stack(q, 1) if q else x.new_zeros((b, 0, d))  # noqa: E731
    p, ep = stack(ps) + skip * x, stack(eps) + 3 * U * (skip * x).abs()
    y, ey = zero(p * gate), zero(ep * gate.abs() + p.abs() * egate + 2 * U * (p * gate).abs())
    res, err = [y, h], [ey, e + fold * top]
    if dy is None:
        return res, err
    dy = zero(dy.double())
    q, eq = zero(dy * gate), zero(dy.abs() * egate + 2 * U * (dy * gate).abs())
    c = torch.zeros_like(h) if dht is None else dht.double()
    ec, topg = torch.zeros_like(c), c.abs()
    da, eda = torch.zeros_like(a), torch.zeros_like(a)
    chain = t * max(1.0, 1.0 + b * groups * -(-d // groups // 64) / 2048) + 16  # a lane's own sums of da, dskip, ddt_bias
    s1s, es1s, s2s, es2s, dbs, edbs, dcs, edcs = ([] for _ in range(8))
    across = lambda m: m.view(b, groups, -1, n).sum(2)  # noqa: E731
    blocks = -(-(d // groups) // 64)
    for i in range(t - 1, -1, -1):
        on, k, hp, ehp = live[:, i, :, None], decay(i), hs[i], es[i] + fold * top
        hn, ehn = hs[i + 1], es[i + 1] + fold * top
        ch, bh = cv[:, i, share], bv[:, i, share]
        qi, eqi, ui = q[:, i, :, None], eq[:, i, :, None], u[:, i, :, None]
        g = c + ch * qi
        topg = torch.maximum(topg, g.abs())
        eg = ec + on * (ch.abs() * eqi + 2 * U * (c.abs() + (ch * qi).abs())) + fold * topg
        s1s.append((bh * g).sum(2)), es1s.append((bh.abs() * eg + (n + 4) * U * (bh * g).abs()).sum(2))
        dbs.append(across(ui * g))
        edbs.append(across(ui.abs() * eg + (rel[:, i, :, None] + (12 + blocks) * U) * (ui * g).abs()))
        dcs.append(across(qi * hn))
        edcs.append(across(qi.abs() * ehn + eqi * hn.abs() + (12 + blocks) * U * (qi * hn).abs()))
        ec = k * (eg - fold * topg) + on * ((erel(i) + 2 * U) * (k * g).abs() + TINY * (g.abs() + 1))
        c = k * g
        past, epast = c * hp, (ec + fold * topg) * hp.abs() + c.abs() * ehp + 2 * U * (c * hp).abs()
        s2s.append((past * a).sum(2))
        es2s.append((a.abs() * epast + (n + 8) * U * (past * a).abs()).sum(2))
        term = past * step[:, i, :, None]
        da += term.sum(0)
        eda += (epast * step[:, i, :, None] + (rel[:, i, :, None] + (chain + 4) * U) * term.abs()).sum(0)
    back = lambda m, s: torch.stack(m[::-1], 1) if m else x.new_zeros((b, 0) + s)  # noqa: E731
    s1, es1, s2, es2 = (back(m, (d,)) for m in (s1s, es1s, s2s, es2s))
    sg = torch.sigmoid(v)
    dx, edx = step * s1 + skip * q, step * es1 + (rel + 4 * U) * (step * s1).abs() + skip.abs() * eq + 3 * U * (skip * q).abs()
    ddt = (s2 + x * s1) * sg
    eddt = (es2 + x.abs() * es1 + 4 * U * (s2.abs() + (x * s1).abs())) * sg + (v.abs() + 16) * U * ddt.abs()
    dz = dy * p * dgate
    edz = dy.abs() * (ep * dgate.abs() + p.abs() * edgate) + 4 * U * dz.abs()
    wide = lambda m: back(m, (groups, n)).flatten(2)  # noqa: E731
    res += [zero(dx), zero(ddt), da, zero(wide(dbs)), zero(wide(dcs)), (q * x).sum((0, 1)), None if z is None else zero(dz),
            zero(ddt).sum((0, 1)), c]
    err += [zero(edx), zero(eddt), eda, zero(wide(edbs)), zero(wide(edcs)),
            (eq * x.abs() + chain * U * (q * x).abs()).sum((0, 1)), None if z is None else zero(edz),
            zero(eddt + chain * U * ddt.abs()).sum((0, 1)), ec + fold * topg]
    return res, err


def linear(x, w, bias, residual, act, dy=None):
    """(results, bounds): y, and with dy also dx, dw, dbias. dL/dv is rounded to the inputs' type on the way (where there
    is an activation), so half a step of it is in the bounds."""
    hs, tiny = half_step(x.dtype), torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps / 2
    x, w = x.double(), w.double()
    rows, c = x.shape
    f = w.shape[0]
    chain = lambda k: (k / 32 + 34) * U  # noqa: E731  (32 products a matrix instruction, then one sum after the other)
    v, ev = x @ w.t(), chain(c) * (x.abs() @ w.abs().t())
    if bias is not None:
        v = v + bias.double()
        ev = ev + 2 * U * v.abs()
    if act == "none":
        a, da, ea, eda = v, torch.ones_like(v), ev, torch.zeros_like(v)
    else:
        a, da = _act(v, act)
        ea, eda = 1.2 * ev + 64 * U * a.abs(), 1.2 * ev + 64 * U * (da.abs() + 1)
    y, ey = a, ea
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2 * U * y.abs()
    if dy is None:
        return [y], [ey]
    dy = dy.double()
    dv, edv = dy * da, dy.abs() * eda + 2 * U * (dy * da).abs() * (act != "none")
    edr = edv + (hs * (dv.abs() + edv) + tiny) * (act != "none")
    res = [y, dv @ w, dv.t() @ x, dv.sum(0)]
    err = [ey, edr @ w.abs() + chain(f) * (dv.abs() @ w.abs()), edr.t() @ x.abs() + chain(rows) * (dv.abs().t() @ x.abs()),
           (edv + (rows / 4 + 4) * U * dv.abs()).sum(0)]
    return res, err
