"""A recurrent block on rows of channels over the operators of fhseq: a gated linear recurrence and a gated feed-forward
block, each behind norms, a gate and a scaled residual. With u the block's normed input and x the residual stream:

    s, state = glr(u wx^T, u wr^T, u wi^T, lam, state),   y1, u1 = norm_block(x, s wo^T, post1, gate1, pre1)
    y, u'    = norm_block(y1, ffn(u1, wg, wu, wd), post2, gate2, pre2)

The sequences are tokens, or a stream's feature maps: an NHWC map of h x w pixels is h * w sequences, and a frame is one
step of each (``forward`` on [pixels, 1, channels] with the state that the last frame left). The square projections are
plain library products. ``python fhblock.py`` streams frames through a block and trains one.
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


def main():
    torch.manual_seed(0)
    c, f, h, w, frames = 128, 512, 30, 54, 24
    block = RecurrentBlock(c, f, torch.float16)
    maps = torch.randn(frames, h * w, c, device="cuda").half()

    def stream():
        state = None
        for m in maps:  # a frame: one step of every pixel
            y, _, state = block.forward(m[:, None], m[:, None], state)
        return y, state

    stream()
    torch.cuda.synchronize()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    y, state = stream()
    end.record()
    torch.cuda.synchronize()
    whole = block.forward(maps.transpose(0, 1), maps.transpose(0, 1))
    print(f"{frames} maps of {h} x {w} x {c}, a frame at a time: {begin.elapsed_time(end) / frames * 1e3:.0f} us a frame; "
          f"against the whole stream at once: state off by {(state - whole[2]).abs().max().item():.2g}")

    b, t = 8, 256
    block = RecurrentBlock(c, f, torch.bfloat16, seed=1)
    x = torch.randn(b, t, c, device="cuda").bfloat16()
    goal = torch.roll(x, 1, 1)  # the value one step ago, which only the state carries
    masters = {k: q.float() for k, q in block.p.items()}
    for step in range(101):
        y, u, _, kept = block.forward(x, x, train=True)
        err = u.float() - goal.float()
        if step % 25 == 0:
            print(f"step {step}: mean square {err.square().mean().item():.4f}")
        grads = block.backward(kept, None, (err * (2 / err.numel()) * 1024).bfloat16())
        for k, q in masters.items():
            d = grads[k].float() / 1024
            q -= 0.02 * d / (d.square().mean().sqrt() + 1e-12) * q.square().mean().sqrt()
            block.p[k].copy_(q)


if __name__ == "__main__":
    main()
