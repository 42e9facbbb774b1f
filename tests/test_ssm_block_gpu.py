"""The state space block (fhblock.StateSpaceBlock): projections, short convolution and selective scan run together as a user
runs them, over whole sequences, a token at a time, in a captured graph and in training."""
import pytest

import fhtest  # noqa: F401  (puts the package on sys.path)

pytestmark = pytest.mark.gpu


def sequence(block, p, x, u, before, h):
    """One sequence [steps, c] through the block in 64 bits, without the roundings between its operators."""
    import torch
    from torch.nn.functional import silu, softplus
    t, e, n, k = x.shape[0], block.e, block.n, block.taps
    v, z = (u @ p["wi"].t()).split(e, 1)
    rows = torch.cat([before, v])
    s = silu(p["bc"] + sum(rows[j:j + t] * p["wc"][:, j] for j in range(k)))
    r, bm, cm = torch.split(s @ p["wp"].t(), (block.rank, block.groups * n, block.groups * n), 1)
    step = softplus(r @ p["wt"].t() + p["dt_bias"], threshold=1000)
    a, share = -torch.exp(p["rates"]), torch.arange(e, device=x.device) // (e // block.groups)
    y = []
    for i in range(t):
        h = torch.exp(step[i, :, None] * a) * h + (step[i] * s[i])[:, None] * bm[i].view(-1, n)[share]
        y.append((cm[i].view(-1, n)[share] * h).sum(1) + p["skip"] * s[i])
    y = torch.stack(y) if y else s
    return (y * silu(z)) @ p["wo"].t() + x, rows[t:], h


def plain(block, p, x, u, before, h, lengths=None):
    import torch
    ends = [x.shape[1]] * x.shape[0] if lengths is None else [min(max(int(q), 0), x.shape[1]) for q in lengths]
    out = [sequence(block, p, x[i, :m], u[i, :m], before[i], h[i]) for i, m in enumerate(ends)]
    y = torch.stack([torch.cat([o[0], x[i, m:]]) for i, (m, o) in enumerate(zip(ends, out))])
    return y, torch.stack([o[1] for o in out]), torch.stack([o[2] for o in out])


def make(b, t, c, e, seed, dtype, **kw):
    import fhblock
    import torch
    block = fhblock.StateSpaceBlock(c, e, dtype=dtype, seed=seed, **kw)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    block.p["bc"].copy_(0.3 * n(e))
    return block, n(b, t, c).to(dtype), n(b, t, c).to(dtype), n(b, block.taps - 1, e).to(dtype), n(b, e, block.n), n


SHAPES = [((3, 50, 64, 96), dict(n=16), None), ((5, 1, 72, 130), dict(n=5, groups=2, taps=3, rank=3), None),
          ((4, 37, 40, 72), dict(n=8, taps=2), (37, 0, 1, 20)), ((1, 200, 48, 64), dict(n=16, groups=2), None)]


@pytest.mark.parametrize("shape,kw,lengths", SHAPES, ids=str)
def test_block_against_64_bits(shape, kw, lengths):
    import torch
    b, t, c, e = shape
    print("state space block", shape, kw, flush=True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for dtype in (torch.float16, torch.bfloat16):
        block, x, u, before, h, n = make(b, t, c, e, 3, dtype, **kw)
        dy, dafter, dh = n(b, t, c).to(dtype), n(*before.shape).to(dtype), n(*h.shape)
        y, (after, end), kept = block.forward(x, u, (before, h), lens, train=True)
        grads = block.backward(kept, dy, (dafter, dh))
        p = {k: v.double().requires_grad_() for k, v in block.p.items()}
        args = dict(x=x, u=u, taps=before, h=h)
        args = {k: v.double().requires_grad_() for k, v in args.items()}
        want = plain(block, p, args["x"], args["u"], args["taps"], args["h"], lengths)
        (sum((q * d.double()).sum() for q, d in zip(want, (dy, dafter, dh)))).backward()
        half = torch.finfo(dtype).eps / 2

        def check(name, got, ref, steps):
            err, size = (got.double() - ref).square().mean().sqrt(), ref.square().mean().sqrt()
            assert err <= steps * half * size, (name, dtype, float(err), steps * half * float(size))

        # Ten roundings to the type lie between the inputs and the last output, each off by half a step of values of what it
        # rounds; they add as independent errors do, so sqrt(10) < 4 of them, in the mean over an output. A gradient has
        # those of the values that it is made of and as many of its own behind it: sqrt(20) < 5.
        for name, q, w in zip(("y", "taps", "h"), (y, after, end), want):
            check(name, q, w.detach(), 4)
        everything = dict(p, **args)
        assert set(grads) == set(everything)
        for name, q in grads.items():
            assert q.shape == everything[name].shape
            check("d" + name, q, everything[name].grad, 5)


def test_block_gradients_along_directions():
    """Gradients along their own direction against central differences of the 64-bit block."""
    import torch
    print("state space block gradients", flush=True)
    b, t, c, e = 3, 24, 40, 56
    block, x, u, before, h, n = make(b, t, c, e, 7, torch.float16, n=8)
    dy, dafter, dh = n(b, t, c).half(), n(*before.shape).half(), n(*h.shape)
    grads = block.backward(block.forward(x, u, (before, h), train=True)[2], dy, (dafter, dh))
    p = {k: v.double() for k, v in block.p.items()}
    p.update(x=x.double(), u=u.double(), taps=before.double(), h=h.double())

    def loss(q):
        out = plain(block, q, q["x"], q["u"], q["taps"], q["h"])
        return float(sum((o * d.double()).sum() for o, d in zip(out, (dy, dafter, dh))))

    for k, grad in grads.items():
        d = grad.double() / grad.double().square().mean().sqrt()
        s = 1e-4
        slope = (loss(dict(p, **{k: p[k] + s * d})) - loss(dict(p, **{k: p[k] - s * d}))) / (2 * s)
        want = float((grad.double() * d).sum())
        # the slope is the true gradient's part along this one, whose error is at most 5 half steps of it in the mean (as
        # above); the differences' own error is of the order of s^2
        assert abs(slope - want) <= (5 * 2 ** -11 + 1e-4) * abs(want), (k, slope, want)


@pytest.mark.parametrize("captured", [False, True])
def test_block_a_token_at_a_time_is_the_whole_sequence(captured):
    """The state that a step leaves is what the next one takes, eagerly and in a graph of one step, replayed."""
    import torch
    print("state space block, tokens", captured, flush=True)
    b, t, c, e = 6, 30, 64, 96
    block, x, u, before, h, _ = make(b, t, c, e, 5, torch.float16)
    whole = block.forward(x, u, (before, h))
    at = [q.clone() for q in (x[:, :1], u[:, :1], before, h)]

    def step():
        y, state = block.forward(at[0], at[1], (at[2], at[3]))
        at[2].copy_(state[0]), at[3].copy_(state[1])
        return y

    graph = None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        at[2].copy_(before), at[3].copy_(h)
    for k in range(t):
        at[0].copy_(x[:, k:k + 1]), at[1].copy_(u[:, k:k + 1])
        if captured:
            graph.replay()
        else:
            y = step()
        # Products of few rows and the scan's steps add in another order: f32 sums that differ in their last bits before
        # roundings to f16, so a value now and then is a step off, and the ten roundings add up to no more than that of
        # the 64-bit test: its bound twice, in the mean.
        err, size = (y[:, 0].double() - whole[0][:, k].double()).square().mean().sqrt(), whole[0].double().square().mean().sqrt()
        assert err <= 8 * 2 ** -11 * size, (k, float(err), float(size))
    for q, w in zip(at[2:], whole[1]):
        assert (q.double() - w.double()).square().mean().sqrt() <= 8 * 2 ** -11 * w.double().square().mean().sqrt()


def test_block_of_no_steps():
    """A call of no steps leaves the state, and its gradients are 0 bar the state's."""
    import torch
    print("state space block of no steps", flush=True)
    block, x, u, before, h, n = make(3, 0, 48, 64, 11, torch.bfloat16)
    y, (after, end), kept = block.forward(x, u, (before, h), train=True)
    assert y.shape == (3, 0, 48) and torch.equal(after, before) and torch.equal(end, h)
    dafter, dh = n(*before.shape).bfloat16(), n(*h.shape)
    g = block.backward(kept, torch.zeros_like(x), (dafter, dh))
    assert torch.equal(g.pop("taps"), dafter) and torch.equal(g.pop("h"), dh)
    assert not any(v.any() for v in g.values())


def test_examples_train_and_stream(capsys):
    """The example runs, and what it trains stays finite."""
    import fhblock
    print("example", flush=True)
    fhblock.main()
    out = capsys.readouterr().out
    assert out.count("us a frame") == 2 and out.count("mean square") == 10 and "nan" not in out and "inf" not in out
