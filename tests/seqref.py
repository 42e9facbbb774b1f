"""Plain 64-bit forms of the operators on rows of channels, with a bound on the error of a 32-bit evaluation beside
each result. The bounds follow the formulas: U is f32's half step (2^-24), and each intermediate's bound is its
inputs' carried through the operation plus its own roundings. An output may be off by its bound plus half a step of
its type."""
import torch

U = 2.0 ** -24

# A gate's sigmoid, decay and input factor in f32: the exponent's argument is rounded (|v| U), the exponential, the sum
# and the reciprocal add about 6 U; log a carries that and the weight's 6 U, and a = exp(log a) multiplies it by
# |log a|. For logits up to 8 and |log a| up to 2 no factor is off by more than 64 U.
STEP = 64 * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, ref, bound, what):
    """got within bound of ref, plus the rounding to got's type (of a subnormal: half the smallest one)."""
    fi = torch.finfo(got.dtype)
    tol = bound * (1 + fi.eps) + half_step(got.dtype) * ref.abs() + fi.tiny * fi.eps / 2
    g = got.double()
    assert torch.isfinite(g).all(), f"{what}: {int((~torch.isfinite(g)).sum())} values are not finite"
    off = (g - ref).abs() - tol
    at = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0, (
        f"{what}: {int((off > 0).sum())} of {off.numel()} off, worst at {at}: got {g.flatten()[at]:.9g}, "
        f"wanted {ref.flatten()[at]:.9g} +- {tol.flatten()[at]:.3g}")


def glr(x, r, i, lam, rate, h0=None, lengths=None, dy=None, dht=None):
    """(results, bounds): y, ht, and with dy also dx, dr, di, dlam, dh0."""
    x, r, i = (v.double() for v in (x, r, i))
    b, t, d = x.shape
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    la = -rate * torch.nn.functional.softplus(lam.double()) * sr
    a, v = torch.exp(la), -torch.expm1(2 * la)
    m, w = v.sqrt(), si * x
    live = torch.ones((b, t, 1), dtype=torch.bool, device=x.device)
    if lengths is not None:
        live = (torch.arange(t, device=x.device)[None] < lengths.clamp(0, t)[:, None])[:, :, None]
    a, inp = torch.where(live, a, 1.0), torch.where(live, m * w, 0.0)
    h = torch.zeros((b, d), dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    e = torch.zeros_like(h)
    hs, es, prev, eprev = [], [], [], []
    for k in range(t):
        prev.append(h), eprev.append(e)
        e = a[:, k] * e + STEP * (a[:, k] * h.abs() + inp[:, k].abs()) * live[:, k]
        h = a[:, k] * h + inp[:, k]
        hs.append(h), es.append(e)
    stack = lambda q: torch.stack(q, 1) if q else x.new_zeros((b, 0, d))  # noqa: E731
    y, ey = torch.where(live, stack(hs), 0.0), torch.where(live, stack(es), 0.0)
    res, err = [y, h], [ey, e]
    if dy is None:
        return res, err
    dy = torch.where(live, dy.double(), 0.0)
    c = torch.zeros_like(h) if dht is None else dht.double()
    ce = torch.zeros_like(c)
    gs, ges = [], []
    for k in range(t - 1, -1, -1):
        g, ge = dy[:, k] + c, ce + U * (dy[:, k].abs() + c.abs()) * live[:, k]
        gs.append(g), ges.append(ge)
        c, ce = a[:, k] * g, a[:, k] * (ge + STEP * g.abs() * live[:, k])
    g, ge, hp, he = stack(gs[::-1]), stack(ges[::-1]), stack(prev), stack(eprev)
    q = torch.where(v > 0, a * a / m.clamp_min(1e-300), 0.0) * w
    dla = g * (a * hp - q)
    dle = ge * (a * hp.abs() + q.abs()) + g.abs() * (a * he + STEP * 2 * (a * hp.abs() + q.abs()))
    dx, dr, di = g * m * si, dla * la * (1 - sr), g * m * w * (1 - si)
    rows = [torch.where(live, z, 0.0) for z in (dx, dr, di)]
    errs = [torch.where(live, z, 0.0) for z in (
        ge * m * si + STEP * 2 * dx.abs(), dle * (la * (1 - sr)).abs() + STEP * 2 * dr.abs(),
        ge * (m * w * (1 - si)).abs() + STEP * 2 * di.abs())]
    sl = torch.sigmoid(lam.double())
    terms, te = torch.where(live, dla * sr, 0.0), torch.where(live, dle * sr, 0.0)
    # a lane adds its own terms in f32, up to a whole sequence of them, the rest in f64
    dlam, le = -rate * sl * terms.sum((0, 1)), rate * sl * (te + (STEP + 2 * t * U) * terms.abs()).sum((0, 1))
    return res + rows + [dlam, c], err + errs + [le, ce]


def norm_block(x, o, w_post, gate, w_pre, alpha, eps, rpg, dy=None, du=None):
    """(results, bounds): y, u, and with dy or du also dx, do, dw_post, dgate, dw_pre (None where not defined)."""
    one = torch.ones((), dtype=torch.float64, device=x.device)
    x = x.double()
    rows, c = x.shape
    o_ = torch.zeros_like(x) if o is None else o.double()
    wp = one if w_post is None else w_post.double()
    wn = one if w_pre is None else w_pre.double()
    ga = one if gate is None else gate.double().repeat_interleave(rpg, 0)[:rows]
    k = 32 * U  # a mean of squares over a row in f32 (chains of up to 32 additions), its square root's inverse
    ro = 1 / torch.sqrt((o_ * o_).mean(1, keepdim=True) + eps)
    no = o_ * ro
    zo = ga * wp * no
    y = alpha * x + zo
    ey = k * ((alpha * x).abs() + 3 * zo.abs())
    ry = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    ery = k + (y.abs() * ey).mean(1, keepdim=True) * ry * ry  # relative
    ny = y * ry
    eny = ey * ry + ny.abs() * (ery + k)
    res, err = [y, wn * ny], [ey, wn.abs() * eny + k * (wn * ny).abs()]
    if dy is None and du is None:
        return res, err
    dy = torch.zeros_like(x) if dy is None else dy.double()
    du = torch.zeros_like(x) if du is None else du.double()
    dn = wn * du
    mn = (dn * ny).mean(1, keepdim=True)
    emn = (dn.abs() * (eny + 2 * k * ny.abs())).mean(1, keepdim=True)
    d = dy + ry * (dn - ny * mn)
    ed = k * dy.abs() + ry * ((ery + 2 * k) * (dn.abs() + ny.abs() * mn.abs()) + eny * mn.abs() + ny.abs() * emn)
    z = ga * wp * d
    mz = (z * no).mean(1, keepdim=True)
    # the kernel takes this mean as a sum of three, so its roundings count at the size of their terms
    emz = (no.abs() * ga.abs() * wp.abs() * (ed + 4 * k * (dy.abs() + ry * (dn.abs() + ny.abs() * mn.abs())))).mean(
        1, keepdim=True)
    do = ro * (z - no * mz)
    edo = ro * ((ga * wp).abs() * ed + 4 * k * (z.abs() + no.abs() * mz.abs()) + no.abs() * emz)
    grow = lambda q: (q + torch.zeros_like(x)).split(rpg if gate is not None else max(rows, 1))  # noqa: E731
    per = lambda q: torch.stack([s.sum(0) for s in grow(q)]) if rows else x.new_zeros((0, c))  # noqa: E731
    s = (2 + rows) * U + k  # sums over rows
    q, eq = d * no, ed * no.abs() + 3 * k * (d * no).abs()
    res += [alpha * d, None if o is None else do, (ga * q).sum(0), wp * per(q), (du * ny).sum(0)]
    err += [abs(alpha) * ed + k * (alpha * d).abs(), None if o is None else edo,
            (ga.abs() * (eq + s * q.abs())).sum(0), wp.abs() * per(eq + s * q.abs()),
            (du.abs() * (eny + s * ny.abs())).sum(0)]
    return res, err


def _act(v, act):
    """act(v) and its derivative."""
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * (1 - p))
    s, b = (2 / torch.pi) ** 0.5, 0.044715
    th = torch.tanh(s * (v + b * v ** 3))
    return 0.5 * v * (1 + th), 0.5 * (1 + th) + 0.5 * v * (1 - th * th) * s * (1 + 3 * b * v * v)


def ffn(x, wg, wu, wd, act, dy=None):
    """(results, bounds): y, and with dy also dx, dwg, dwu, dwd. h and the gradients at the two projections are rounded
    to the inputs' type on the way, so half a step of each is in the bounds."""
    hs, tiny = half_step(x.dtype), torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps / 2
    x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
    rows, c = x.shape
    f = wg.shape[0]
    chain = lambda k: (k / 32 + 34) * U  # noqa: E731  (32 products a matrix instruction, then one sum after the other)
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (chain(c) * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a, da = _act(g, act)
    ea = 1.2 * eg + 64 * U * a.abs()  # |act'| < 1.13; the exponent's argument is rounded, |k(v)| at most 60 where it counts
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + 2 * U * h.abs()
    ehr = eh + hs * (h.abs() + eh) + tiny
    y, ey = h @ wd.t(), ehr @ wd.abs().t() + chain(f) * (h.abs() @ wd.abs().t())
    if dy is None:
        return [y], [ey]
    dy = dy.double()
    dh, edh = dy @ wd, chain(c) * (dy.abs() @ wd.abs())
    eda = 1.2 * eg + 64 * U * (da.abs() + 1)  # |act''| < 1
    dg, du = dh * u * da, dh * a
    edg = edh * (u * da).abs() + dh.abs() * (eu * da.abs() + u.abs() * eda) + 4 * U * dg.abs()
    edu = edh * a.abs() + dh.abs() * ea + 2 * U * du.abs()
    edg, edu = edg + hs * (dg.abs() + edg) + tiny, edu + hs * (du.abs() + edu) + tiny
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + chain(2 * f) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    res, err = [y, dx], [ey, edx]
    for p, ep in ((dg, edg), (du, edu)):
        res.append(p.t() @ x), err.append(ep.t() @ x.abs() + chain(rows) * (p.abs().t() @ x.abs()))
    res.append(dy.t() @ h), err.append(dy.abs().t() @ ehr + chain(rows) * (dy.abs().t() @ h.abs()))
    return res, err
