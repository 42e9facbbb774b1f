"""The recurrent block (fhblock.py): its operators run together as a user runs them, over streams and in training."""
import pytest

import fhtest  # noqa: F401  (puts the package on sys.path)
import seqref

pytestmark = pytest.mark.gpu


def plain(block, x, u, state, gate1, gate2):
    """The block in 64 bits from the same weights, without the roundings between its operators."""
    import torch
    p = {k: v.double() for k, v in block.p.items()}
    b, t, c = x.shape

    def norm(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + block.eps)

    v, r, i = (u @ p[k].t() for k in ("wx", "wr", "wi"))
    (s, end), _ = seqref.glr(v, r, i, p["lam"], block.rate, state)
    y1 = block.alpha * x + gate1[:, None] * p["post1"] * norm(s @ p["wo"].t())
    u1 = p["pre1"] * norm(y1)
    a, _ = seqref._act(u1 @ p["wg"].t(), block.act)
    y = block.alpha * y1 + gate2[:, None] * p["post2"] * norm((a * (u1 @ p["wu"].t())) @ p["wd"].t())
    return y, p["pre2"] * norm(y), end


def inputs(b, t, c, seed, dtype):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return n(b, t, c).to(dtype), n(b, t, c).to(dtype), n(b, c), n(b, c).to(dtype), n(b, c).to(dtype), n


@pytest.mark.parametrize("shape", [(3, 50, 64, 96), (5, 1, 72, 130)], ids=str)
def test_block_against_64_bits(shape):
    import fhblock
    import torch
    b, t, c, f = shape
    print("block", shape, flush=True)
    for dtype in (torch.float16, torch.bfloat16):
        block = fhblock.RecurrentBlock(c, f, dtype, seed=3)
        x, u, state, g1, g2, _ = inputs(b, t, c, 4, dtype)
        got = block.forward(x, u, state, g1, g2)
        want = plain(block, x.double(), u.double(), state.double(), g1.double(), g2.double())
        # eight roundings to the type lie between the inputs and the last output, each off by half a step of values of
        # the outputs' size; they add as independent errors do, so sqrt(8) < 3 of them, in the mean over an output
        step = torch.finfo(dtype).eps / 2
        for name, a, w in zip(("y", "u", "state"), got, want):
            err = (a.double() - w).square().mean().sqrt() / w.square().mean().sqrt()
            assert err <= 3 * step, (name, float(err), step)


def test_block_a_frame_at_a_time_is_the_whole_stream():
    """The state that a step leaves is what the next one takes: steps one by one give the whole call's values."""
    import fhblock
    import torch
    print("block stream", flush=True)
    b, t, c = 70, 20, 64
    block = fhblock.RecurrentBlock(c, 96, torch.float16, seed=5)
    x, u, state, g1, g2, _ = inputs(b, t, c, 6, torch.float16)
    whole = block.forward(x, u, state, g1, g2)
    for k in range(t):
        y, un, state = block.forward(x[:, k:k + 1], u[:, k:k + 1], state, g1, g2)
        # the same operations on the same rows; only the recurrence's order of f32 sums differs, before a rounding to f16
        assert (y[:, 0].float() - whole[0][:, k].float()).abs().max() <= 2 ** -6
        assert (un[:, 0].float() - whole[1][:, k].float()).abs().max() <= 2 ** -6
    assert (state - whole[2]).abs().max() <= 1e-3 * whole[2].abs().max()


def test_block_gradients_along_directions():
    """Every gradient along a random direction against central differences of the 64-bit block."""
    import fhblock
    import torch
    print("block gradients", flush=True)
    b, t, c, f = 4, 30, 48, 80
    block = fhblock.RecurrentBlock(c, f, torch.float16, seed=7)
    x, u, state, g1, g2, n = inputs(b, t, c, 8, torch.float16)
    dy, du, ds = n(b, t, c).half(), n(b, t, c).half(), n(b, c)
    kept = block.forward(x, u, state, g1, g2, train=True)[3]
    grads = block.backward(kept, dy, du, ds)
    args = dict(x=x, u=u, state=state, gate1=g1, gate2=g2)
    weights = dict(block.p)

    def loss(name, d):
        a = {k: v.double() for k, v in args.items()}
        block.p = {k: v.double() for k, v in weights.items()}
        (a if name in a else block.p)[name] = (a if name in a else block.p)[name] + d
        y, un, end = plain(block, a["x"], a["u"], a["state"], a["gate1"], a["gate2"])
        block.p = weights
        return float((y * dy.double()).sum() + (un * du.double()).sum() + (end * ds.double()).sum())

    for k, grad in grads.items():
        d, s = n(*grad.shape).double(), 1e-5
        slope = (loss(k, s * d) - loss(k, -s * d)) / (2 * s)
        want = float((grad.double() * d).sum())
        # up to a dozen f16 roundings on a gradient's way, each half a step of what it rounds
        assert abs(slope - want) <= 12 * 2 ** -11 * float((grad.double() * d).abs().sum()), (k, slope, want)


def test_block_learns():
    import fhblock
    import torch
    print("block learns", flush=True)
    block = fhblock.RecurrentBlock(64, 128, torch.bfloat16, seed=9)
    x = inputs(8, 64, 64, 10, torch.bfloat16)[0]
    goal = torch.roll(x, 1, 1).float()
    losses = []
    for _ in range(30):
        _, u, _, kept = block.forward(x, x, train=True)
        err = u.float() - goal
        losses.append(float(err.square().mean()))
        grads = block.backward(kept, None, (err / err.numel() * 2048).bfloat16())
        for k, q in block.p.items():
            d = grads[k].float()
            q -= (0.02 * d / (d.square().mean().sqrt() + 1e-12) * q.float().square().mean().sqrt()).to(q.dtype)
    assert losses[-1] < 0.8 * losses[0], losses


def test_block_of_no_steps():
    """A call of no steps leaves the state, and its gradients are 0 bar the state's, with and without gates."""
    import fhblock
    import torch
    print("block of no steps", flush=True)
    b, c = 3, 64
    block = fhblock.RecurrentBlock(c, 96, torch.bfloat16, seed=11)
    x, u, state, g1, g2, n = inputs(b, 0, c, 12, torch.bfloat16)
    ds = n(b, c)
    for a1, a2 in ((None, None), (g1, g2), (g1, None)):
        y, un, end, kept = block.forward(x, u, state, a1, a2, train=True)
        assert y.shape == un.shape == (b, 0, c) and torch.equal(end, state)
        g = block.backward(kept, torch.zeros_like(x), torch.zeros_like(x), ds)
        assert torch.equal(g.pop("state"), ds)
        for k, gate in (("gate1", a1), ("gate2", a2)):
            assert (g[k] is None) == (gate is None) and (gate is None or g[k].shape == gate.shape), k
        assert g["x"].shape == g["u"].shape == (b, 0, c)
        assert not any(v.any() for v in g.values() if v is not None)
