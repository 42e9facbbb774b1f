"""Recurrent blocks on rows of channels over the operators of fhseq, u a block's normed input and x the residual stream.

RecurrentBlock: a gated linear recurrence and a gated feed-forward block, each behind norms, a gate and a scaled residual:

    s, state = glr(u wx^T, u wr^T, u wi^T, lam, state),   y1, u1 = norm_block(x, s wo^T, post1, gate1, pre1)
    y, u'    = norm_block(y1, ffn(u1, wg, wu, wd), post2, gate2, pre2)

Its square projections are plain library products.

StateSpaceBlock: a selective state space scan behind a short convolution, gated, with a residual:

    v, z = u wi^T,   s, taps = short_conv(v, wc, bc, taps),   r, B, C = s wp^T
    o, h = ssm(s, r wt^T, a, B, C, skip, z, dt_bias, h),   y = o wo^T + x

The sequences are tokens, or a stream's feature maps: an NHWC map of h x w pixels is h * w sequences, and a frame is one
step of each (``forward`` on [pixels, 1, channels] with the state that the last frame left). ``python fhblock.py`` streams
frames through both blocks and trains one of each.
"""
from __future__ import annotations

import torch

import fhseq

PROJECTIONS = ("wx", "wr", "wi")


class RecurrentBlock:
    """Weights of one block of ``c`` channels, ``f`` wide inside, in ``dtype`` (f16, bf16). The recurrence's rates start
    at decays of 0.9 to 0.999 a step."""

    def __init__(self, c, f, dtype=torch.bfloat16, act="silu", alpha=0.5 ** 0.5, eps=1e-6, rate=8.0, seed=0,
                 device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def normal(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) * cols ** -0.5).to(dtype)

        self.c, self.act, self.alpha, self.eps, self.rate = c, act, alpha, eps, rate
        u = torch.rand(c, generator=g, device=device, dtype=torch.float64) * 0.099 + 0.9
        self.p = {k: normal(c, c) for k in PROJECTIONS + ("wo",)}
        self.p.update(wg=normal(f, c), wu=normal(f, c), wd=normal(c, f))
        self.p["lam"] = torch.log(torch.expm1(-torch.log(u) / rate)).float()
        for k in ("post1", "pre1", "post2", "pre2"):
            self.p[k] = torch.ones(c, dtype=dtype, device=device)

    def forward(self, x, u, state=None, gate1=None, gate2=None, lengths=None, train=False):
        """x, u [sequences, steps, c]: the residual stream and this block's normed input; state [sequences, c] f32 or
        None (zeros); gate1, gate2 [sequences, c] or None; lengths as in ``fhseq.glr``: past them the recurrence's output
        is 0, and the rest of the block works on x and u there as on any row, so they have to be finite. Returns (y, the
        next block's input, the state after the last step), with train also what ``backward`` takes."""
        p, (b, t, c) = self.p, x.shape
        xr, ur = x.reshape(-1, c), u.reshape(-1, c)
        v, r, i = ((ur @ p[k].t()).view(b, t, c) for k in PROJECTIONS)
        out = fhseq.glr(v, r, i, p["lam"], self.rate, h0=state, lengths=lengths, train=train)
        s = out[0].reshape(-1, c)
        o1 = s @ p["wo"].t()
        rows = max(t, 1)
        if t == 0:  # no rows, no groups of them
            gate1, gate2 = (None if g is None else g[:0] for g in (gate1, gate2))
        y1, u1 = fhseq.norm_block(xr, o1, p["post1"], gate1, p["pre1"], self.alpha, self.eps, rows)
        o2 = fhseq.ffn(u1, p["wg"], p["wu"], p["wd"], self.act, train=train)
        kept = None
        if train:
            o2, ffn_kept = o2
            kept = (xr, ur, v, r, i, s, o1, y1, u1, o2, out[2], ffn_kept, gate1, gate2, lengths)
        y, un = fhseq.norm_block(y1, o2, p["post2"], gate2, p["pre2"], self.alpha, self.eps, rows)
        res = (y.view(b, t, c), un.view(b, t, c), out[1])
        return res + (kept,) if train else res

    def backward(self, kept, dy, du, dstate=None):
        """The gradients of a loss with dy, du (of forward's first two results, either may be None) and dstate: a dict
        of the weights' ("wx", .. "pre2") and "x", "u", "state", "gate1", "gate2" (None where there was none)."""
        xr, ur, v, r, i, s, o1, y1, u1, o2, states, ffn_kept, gate1, gate2, lengths = kept
        p, (b, t, c) = self.p, v.shape
        rows = max(t, 1)

        def flat(d):
            return None if d is None else d.reshape(-1, c)

        g = {}
        dy1, do2, g["post2"], g["gate2"], g["pre2"] = fhseq.norm_block_backward(
            y1, o2, p["post2"], gate2, p["pre2"], flat(dy), flat(du), self.alpha, self.eps, rows)
        du1, g["wg"], g["wu"], g["wd"] = fhseq.ffn_backward(u1, p["wg"], p["wu"], p["wd"], ffn_kept, do2, self.act)
        dx, do1, g["post1"], g["gate1"], g["pre1"] = fhseq.norm_block_backward(
            xr, o1, p["post1"], gate1, p["pre1"], dy1, du1, self.alpha, self.eps, rows)
        g["wo"] = do1.t() @ s
        ds = (do1 @ p["wo"]).view(b, t, c)
        dv, dr, di, g["lam"], g["state"] = fhseq.glr_backward(v, r, i, p["lam"], states, ds, self.rate, dht=dstate,
                                                              lengths=lengths)
        du0 = None
        for k, d in zip(PROJECTIONS, (dv, dr, di)):
            d = d.reshape(-1, c)
            g[k] = d.t() @ ur
            du0 = d @ p[k] if du0 is None else du0.addmm_(d, p[k])
        g["x"], g["u"] = dx.view(b, t, c), du0.view(b, t, c)
        if t == 0:
            for k in ("gate1", "gate2"):
                g[k] = None if g[k] is None else g[k].new_zeros(b, c)
        return g


class StateSpaceBlock:
    """Weights of one block of ``c`` channels, ``e`` wide inside, with ``n`` states a channel, B and C shared by the
    channels of each of ``groups`` groups, steps of ``rank`` numbers and ``taps`` taps, in ``dtype`` (f16, bf16). The
    states decay at rates of 1 to n times the step, which starts at 0.001 to 0.1."""

    def __init__(self, c, e, n=16, groups=1, rank=None, taps=4, dtype=torch.bfloat16, seed=0, device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        rank = max(c // 16, 1) if rank is None else rank

        def normal(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) * cols ** -0.5).to(dtype)

        self.c, self.e, self.n, self.groups, self.rank, self.taps = c, e, n, groups, rank, taps
        first = 0.001 * 100.0 ** torch.rand(e, generator=g, device=device, dtype=torch.float64)
        self.p = dict(wi=normal(2 * e, c), wc=normal(e, taps), bc=torch.zeros(e, dtype=dtype, device=device),
                      wp=normal(rank + 2 * groups * n, e), wt=normal(e, rank), wo=normal(c, e))
        self.p["rates"] = torch.log(torch.arange(1, n + 1, device=device).float()).repeat(e, 1)  # a = -exp(rates)
        self.p["skip"] = torch.ones(e, device=device)
        self.p["dt_bias"] = torch.log(torch.expm1(first)).float()

    def _split(self, m):
        return torch.split(m, (self.rank, self.groups * self.n, self.groups * self.n), 2)

    def forward(self, x, u, state=None, lengths=None, train=False):
        """x, u [sequences, steps, c]: the residual stream and this block's normed input; state (taps [sequences, taps -
        1, e], h [sequences, e, n] f32) as an earlier call returned it, or None (zeros); lengths as in ``fhseq.ssm``: past
        them y is x, and the state is that of a sequence's last step; u has to be finite there. Returns (y, state), with
        train also what ``backward`` takes."""
        p, (b, t, c), e = self.p, x.shape, self.e
        before, h0 = (None, None) if state is None else state
        ur = u.reshape(-1, c)
        v, z = fhseq.linear(ur, p["wi"]).view(b, t, 2 * e).split(e, 2)  # no copies: the halves of a row
        s, after = fhseq.short_conv(v, p["wc"], p["bc"], state=before, lengths=lengths)
        m = fhseq.linear(s.reshape(-1, e), p["wp"]).view(b, t, p["wp"].shape[0])
        r, bm, cm = self._split(m)
        dt = fhseq.linear(r.flatten(0, 1), p["wt"]).view(b, t, e)
        a = -torch.exp(p["rates"])
        out = fhseq.ssm(s, dt, a, bm, cm, p["skip"], z, p["dt_bias"], h0, lengths, train)
        y = fhseq.linear(out[0].reshape(-1, e), p["wo"], residual=x.reshape(-1, c)).view(b, t, c)
        res = (y, (after, out[1]))
        return res + ((ur, v, z, before, s, m, dt, a, out[0], out[2], lengths),) if train else res

    def backward(self, kept, dy, dstate=None):
        """The gradients of a loss with dy and dstate (of forward's state; it or either of its two may be None): a dict of
        the weights' ("wi", .. "dt_bias") and "x", "u", "taps", "h"."""
        ur, v, z, before, s, m, dt, a, o, states, lengths = kept
        p, (b, t, e), c = self.p, s.shape, self.c
        dafter, dend = (None, None) if dstate is None else dstate
        r, bm, cm = self._split(m)
        g = dict(x=dy)
        do, g["wo"], _ = fhseq.linear_backward(o.reshape(-1, e), p["wo"], None, dy.reshape(-1, c), bias=False)
        ds, ddt, da, dbm, dcm, g["skip"], dz, g["dt_bias"], g["h"] = fhseq.ssm_backward(
            s, dt, a, bm, cm, states, do.view(b, t, e), p["skip"], z, p["dt_bias"], dend, lengths)
        g["rates"] = da * a
        dr, g["wt"], _ = fhseq.linear_backward(r.flatten(0, 1), p["wt"], None, ddt.reshape(-1, e), bias=False)
        dm = torch.cat((dr.view(b, t, self.rank), dbm, dcm), 2)
        ds1, g["wp"], _ = fhseq.linear_backward(s.reshape(-1, e), p["wp"], None, dm.flatten(0, 1), bias=False)
        dv, g["wc"], g["bc"], g["taps"] = fhseq.short_conv_backward(v, p["wc"], p["bc"], ds + ds1.view(b, t, e), "silu",
                                                                    before, dafter, lengths)
        du, g["wi"], _ = fhseq.linear_backward(ur, p["wi"], None, torch.cat((dv, dz), 2).flatten(0, 1), bias=False)
        g["u"] = du.view(b, t, c)
        return g


def main():
    torch.manual_seed(0)
    c, f, h, w, frames = 128, 512, 30, 54, 24
    maps = torch.randn(frames, h * w, c, device="cuda").half()
    for block in (RecurrentBlock(c, f, torch.float16), StateSpaceBlock(c, 2 * c, dtype=torch.float16)):

        def stream():
            state = None
            for m in maps:  # a frame: one step of every pixel
                state = block.forward(m[:, None], m[:, None], state)[-1]
            return state

        stream()
        torch.cuda.synchronize()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        state = stream()
        end.record()
        torch.cuda.synchronize()
        whole = block.forward(maps.transpose(0, 1), maps.transpose(0, 1))[-1]
        off = max((s.float() - q.float()).abs().max().item() for s, q in zip(state, whole))
        print(f"{type(block).__name__}: {frames} maps of {h} x {w} x {c}, a frame at a time: "
              f"{begin.elapsed_time(end) / frames * 1e3:.0f} us a frame; against the whole stream at once: state off by "
              f"{off:.2g}")

    b, t = 8, 256
    x = torch.randn(b, t, c, device="cuda").bfloat16()
    goal = torch.roll(x, 1, 1)  # the value one step ago, which only the state carries
    for block in (RecurrentBlock(c, f, torch.bfloat16, seed=1), StateSpaceBlock(c, 2 * c, seed=1)):
        masters = {k: q.float() for k, q in block.p.items()}
        for step in range(101):
            if isinstance(block, RecurrentBlock):
                _, u, _, kept = block.forward(x, x, train=True)
            else:
                u, _, kept = block.forward(torch.zeros_like(x), x, train=True)
            err = u.float() - goal.float()
            if step % 25 == 0:
                print(f"{type(block).__name__}, step {step}: mean square {err.square().mean().item():.4f}")
            du = (err * (2 / err.numel()) * 1024).bfloat16()
            grads = block.backward(kept, None, du) if isinstance(block, RecurrentBlock) else block.backward(kept, du)
            for k, q in masters.items():
                d = grads[k].float() / 1024
                q -= 0.02 * d / (d.square().mean().sqrt() + 1e-12) * q.square().mean().sqrt()
                block.p[k].copy_(q)


if __name__ == "__main__":
    main()
