"""Linear attention, the norms around a block and gradient clipping used together, as a small stack of blocks trains and answers with them, against
the same stack written out in 64 bits.

Tolerance: relative to a tensor's largest value, 2048 roundings of 2^-24.  On its way an element passes two blocks of a projection (32 terms), a
chunk of attention (16 + 16 products, 64 tokens, 40 of an exponent), two norms (2 * 32) and a gate, about 360 roundings, forward and backward alike, and
the norms keep errors in proportion: 1440, rounded up."""
import pytest
import torch
import torch.nn.functional as F

from mamba_unet_amd import clip_grad_norm, linear_attention_fn, linear_attention_step, norm_gate_residual

pytestmark = pytest.mark.gpu
D, H, G, DK, DV, BLOCKS = 32, 4, 2, 16, 8, 2
TOL = 2048 * 2.0 ** -24


def parameters(seed=0):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r) * s[-1] ** -0.5  # noqa: E731
    return [{"q": n(G * DK, D), "k": n(G * DK, D), "v": n(H * DV, D), "z": n(H * DV, D), "g": n(H, D), "w1": 1 + 0.1 * n(H * DV), "w2": 1 + 0.1 * n(D), "a": 0.5 + 0.1 * n(D)}
            for _ in range(BLOCKS)]


def project(p, h):
    q, k, v, z, g = (F.linear(h, p[m]) for m in ("q", "k", "v", "z", "g"))
    return q.unflatten(-1, (G, DK)), k.unflatten(-1, (G, DK)), v.unflatten(-1, (H, DV)), z, F.logsigmoid(g)


def model(ps, x):
    """(B, L, D) -> the last block's (x, h)"""
    h, last = x, []
    for p in ps:
        q, k, v, z, g = project(p, h)
        y, s = linear_attention_fn(q, k, v, g, return_last_state=True)
        x, h = norm_gate_residual(x, y.flatten(-2), p["w1"], p["w2"], z=z, res_scale=p["a"], rms=True)
        last.append(s)
    return x, h, last


def token(ps, x, states, slots):
    h = x
    for p, s in zip(ps, states):
        q, k, v, z, g = project(p, h)
        y = linear_attention_step(s, q, k, v, g, state_indices=slots)
        x, h = norm_gate_residual(x, y.flatten(-2), p["w1"], p["w2"], z=z, res_scale=p["a"], rms=True)
    return x, h


def plain(ps, x):
    rms = lambda t, w: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) * w  # noqa: E731
    h = x
    for p in ps:
        q, k, v, z, g = project(p, h)
        S, out = x.new_zeros(x.shape[0], H, DK, DV), []
        for t in range(x.shape[1]):
            kt, qt = (m[:, t].repeat_interleave(H // G, 1) for m in (k, q))
            S = g[:, t].exp()[..., None, None] * S + kt[..., None] * v[:, t, :, None]
            out.append(DK ** -0.5 * (qt[..., None] * S).sum(-2))
        u = rms(torch.stack(out, 1).flatten(-2), p["w1"]) * F.silu(z)
        x = x + p["a"] * u
        h = rms(x, p["w2"])
    return x, h


def close(got, want, what):
    err = float((got.cpu().double() - want).abs().max() / want.abs().max())
    assert err <= TOL, f"{what}: {err:.1e}"


def leaves(ps, **kw):
    return [{n: t.to(**kw).requires_grad_() for n, t in p.items()} for p in ps]


def flat(ps):
    return [p[n] for p in ps for n in sorted(p)]


def train(ps, x, target):
    _, h, _ = model(ps, x)
    h.backward((h.detach() - target) * (2.0 / h.numel()))          # of the mean square
    return clip_grad_norm(flat(ps), 0.01)


def test_training_step_against_64_bits():
    ps, r = parameters(), torch.Generator().manual_seed(1)
    x, target = torch.randn(3, 150, D, generator=r), torch.randn(3, 150, D, generator=r)
    ref = leaves(ps, dtype=torch.float64)
    want = plain(ref, x.double())
    ((want[1] - target.double()) ** 2).mean().backward()
    norm = torch.stack([t.grad.norm() for t in flat(ref)]).norm()
    assert norm > 0.01
    own = leaves(ps, device="cuda")
    got = model(own, x.cuda())
    close(got[0].detach(), want[0].detach(), "x")
    close(got[1].detach(), want[1].detach(), "h")
    n = train(own, x.cuda(), target.cuda())
    close(n, norm, "norm")
    for p, o in zip(ref, own):
        for m in p:
            close(o[m].grad, p[m].grad * (0.01 / (norm + 1e-6)), m)


def test_captured_training_step_replays():
    ps, r = parameters(2), torch.Generator().manual_seed(3)
    xs, ts = torch.randn(4, 2, 200, D, generator=r).cuda(), torch.randn(4, 2, 200, D, generator=r).cuda()
    eager = leaves(ps, device="cuda")
    wants = []
    for x, t in zip(xs, ts):
        for p in flat(eager):
            p.grad = None
        n = train(eager, x, t)
        wants.append([n.clone()] + [p.grad.clone() for p in flat(eager)])
    own = leaves(ps, device="cuda")
    x, t = xs[0].clone(), ts[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            for p in flat(own):
                p.grad = None
            train(own, x, t)
    torch.cuda.current_stream().wait_stream(side)
    for p in flat(own):
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = train(own, x, t)
    for i in (0, 1, 2, 3, 1):
        x.copy_(xs[i])
        t.copy_(ts[i])
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip([n] + [p.grad for p in flat(own)], wants[i]):
            assert float((got - want).abs().max()) <= TOL * float(want.abs().max())
        model(eager, xs[i])[1].sum().item()                       # eager work of the same operators between the replays


def test_prompts_then_tokens_against_whole_sequences():
    ps, r = parameters(4), torch.Generator().manual_seed(5)
    x = torch.randn(3, 90, D, generator=r)
    want = plain([{n: t.double() for n, t in p.items()} for p in ps], x.double())
    ps = [{n: t.cuda() for n, t in p.items()} for p in ps]
    x, slots = x.cuda(), torch.tensor([6, 0, 3], device="cuda")
    with torch.no_grad():
        _, _, last = model(ps, x[:, :80].contiguous())
        pools = [torch.zeros(8, H, DK, DV, device="cuda").index_copy_(0, slots, s) for s in last]
        for i in range(80, 90):
            xo, h = token(ps, x[:, i].contiguous(), pools, slots)
            close(xo, want[0][:, i], "x")
            close(h, want[1][:, i], "h")
    for s in pools:
        assert not s[[1, 2, 4, 5, 7]].any()
