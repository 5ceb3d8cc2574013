"""norm_gate_residual against its formula in 64 bits.

Tolerances.  u = 2^-24.  A row's statistics are sums over D values (TPR threads x at most 32 each, then a tree): D-independent, below 48 roundings;
a normalised value, the gate (exp2 and a reciprocal, each within 2 u, its exponent |z| u with |z| < 8) and the products add fewer than 48 more.
So x' and h are within 96 u of the magnitudes |x| + |drop a u| they are made of, carried through the second norm, and the row gradients within the
same of the row's root mean square gradient times the norm's gain.  Parameter gradients are sums over n rows, at most n / 256 + 600 additions each:
norm-wise (96 + n / 256 + 600) u of the sums of magnitudes."""
import pytest
import torch

from mamba_unet_amd import norm_gate_residual

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def formula(t, rms, eps=1e-5):
    def norm(v, w, b):
        v = v if rms else v - v.mean(-1, keepdim=True)
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w
        return v if b is None else v + b
    u = norm(t["y"], t["w1"], t["b1"])
    if t["z"] is not None:
        u = u * t["z"] * torch.sigmoid(t["z"])
    if t["a"] is not None:
        u = u * t["a"]
    if t["drop"] is not None:
        u = u * t["drop"].view((-1,) + (1,) * (u.dim() - 1))
    x = t["x"] + u
    return x, norm(x, t["w2"], t["b2"])


def make(shape, res, io, gate=True, bias=True, scale=True, drop=True, seed=0, mean=0.0):
    r = torch.Generator().manual_seed(seed)
    D = shape[-1]
    rnd = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    return {"x": (rnd(*shape) + mean).to(res), "y": (rnd(*shape) + mean).to(io), "z": rnd(*shape).to(io) if gate else None, "w1": 1 + 0.2 * rnd(D),
            "b1": 0.2 * rnd(D) if bias else None, "a": 0.5 * rnd(D) if scale else None, "w2": 1 + 0.2 * rnd(D), "b2": 0.2 * rnd(D) if bias else None,
            "drop": (torch.rand(shape[0], generator=r) < 0.7).float() / 0.7 if drop else None, "dx": rnd(*shape).to(res), "dh": rnd(*shape).to(io)}


NAMES = ("x", "y", "z", "w1", "b1", "a", "w2", "b2")


def call(t, rms):
    return norm_gate_residual(t["x"], t["y"], t["w1"], t["w2"], post_bias=t["b1"], pre_bias=t["b2"], z=t["z"], res_scale=t["a"], drop_scale=t["drop"],
                              eps=1e-5, rms=rms)


def run(t, rms, dev="cuda", use=(True, True)):
    d = {n: None if v is None else v.to(dev) for n, v in t.items()}
    leaves = [n for n in NAMES if d[n] is not None]
    for n in leaves:
        d[n].requires_grad_()
    x, h = call(d, rms)
    outs = [(x, d["dx"])] * use[0] + [(h, d["dh"])] * use[1]
    grads = torch.autograd.grad([o for o, _ in outs], [d[n] for n in leaves], [g for _, g in outs], allow_unused=True)
    return {"x'": x.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def want(t, rms, use=(True, True)):
    d = {n: None if v is None else v.double().requires_grad_(n in NAMES) for n, v in t.items()}
    leaves = [n for n in NAMES if d[n] is not None]
    x, h = formula(d, rms)
    grads = torch.autograd.grad((x * d["dx"]).sum() * use[0] + (h * d["dh"]).sum() * use[1], [d[n] for n in leaves], allow_unused=True)
    return {"x'": x.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def check(got, ref, rows, D):
    for n, g in got.items():
        w = ref[n]
        if w is None:
            assert g is None or not g.any(), n
            continue
        assert torch.isfinite(g).all(), n
        err = (g.cpu().double() - w).abs()
        if n in ("x'", "h", "dx", "dy", "dz"):
            # the row's own scale, its largest value: statistics reach every element of a row
            lim = HALF[g.dtype] * w.abs() + 96 * U * (w.abs().amax(-1, keepdim=True) + 8)
        else:
            # terms of random sign: their magnitudes' sum over n rows is at most about n times a term's largest size (< 64 here)
            lim = HALF[g.dtype] * w.abs() + (96 + rows / 256 + 600) * U * 8 * rows ** 0.5
        assert bool((err <= lim).all()), f"{n}: {float((err / lim).max()):.2f} of the tolerance"


SHAPES = [(1, 1), (3, 5), (2, 3, 16), (7, 33), (5, 96), (4, 100), (2, 9, 128), (3, 136), (6, 512), (2, 515), (3, 1001), (5, 1024), (3, 1032), (2, 2048),
          (2, 2050), (3, 4096), (2, 4100), (2, 8192), (2, 7777)]


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)], ids=["fp32", "mixed", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_outputs_and_every_gradient(shape, types, rms):
    if not rms and shape[-1] == 1:
        pytest.skip("LayerNorm of one channel: the deviation is 0 and only eps is left")
    t = make(shape, *types)
    check(run(t, rms), want(t, rms), t["x"].numel() // shape[-1], shape[-1])


@pytest.mark.parametrize("on", [(0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1)], ids=["none", "gate", "bias", "scale", "drop"])
def test_optional_parts(on):
    t = make((4, 6, 64), torch.float32, torch.bfloat16, *map(bool, on))
    check(run(t, True), want(t, True), 24, 64)


@pytest.mark.parametrize("use", [(True, False), (False, True)], ids=["x", "h"])
def test_one_output_used(use):
    t = make((4, 6, 64), torch.float32, torch.float32)
    check(run(t, False, use=use), want(t, False, use), 24, 64)


def test_many_rows():
    t = make((3, 700, 96), torch.float32, torch.float32)
    check(run(t, False), want(t, False), 2100, 96)


def test_gradients_against_differences():
    """Central differences of <dx, x'> + <dh, h>, computed in 64 bits at the operator's own fp32 inputs, step 2^-12: third order below 2^-20."""
    t = make((3, 40), torch.float32, torch.float32, drop=False, seed=4)
    got = run(t, False)
    d = {n: None if v is None else v.double() for n, v in t.items()}
    r = torch.Generator().manual_seed(5)
    for n in NAMES:
        e = torch.randn(t[n].shape, generator=r, dtype=torch.float64) * 2.0 ** -12
        f = lambda s: sum(((o * g).sum() for o, g in zip(formula({**d, n: d[n] + s * e}, False), (d["dx"], d["dh"]))), torch.zeros((), dtype=torch.float64))  # noqa: E731,B023
        diff, lin = float(f(1) - f(-1)), float(2 * (got["d" + n].cpu().double() * e).sum())
        assert abs(diff - lin) <= 2.0 ** -18 * float(got["d" + n].cpu().double().norm() * e.norm()) * 64, n


def test_gate_and_stream_as_slices_of_wider_tensors():
    t = make((2, 9, 64), torch.bfloat16, torch.bfloat16)
    d = {n: v.cuda() for n, v in t.items()}
    want_x, want_h = call(d, True)
    wide = torch.randn(2, 9, 192, device="cuda").bfloat16()
    wide[..., :64], wide[..., 64:128], wide[..., 128:] = d["x"], d["y"], d["z"]
    for views in ({"x": wide[..., :64], "y": wide[..., 64:128], "z": wide[..., 128:]}, {"z": d["z"].transpose(0, 1).contiguous().transpose(0, 1)},
                  {"y": torch.cat([d["y"].flatten(), d["y"].new_zeros(1)])[:-1].view(2, 9, 64)}):
        x, h = call({**d, **views}, True)
        assert torch.equal(x, want_x) and torch.equal(h, want_h)
    odd = torch.zeros(2 * 9 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 9, 64)
    odd.copy_(d["y"])
    x, h = call({**d, "y": odd}, True)
    assert torch.equal(x, want_x) and torch.equal(h, want_h)


def test_large_means_and_extreme_gates():
    """A row mean 1000 times its spread costs LayerNorm no digits beyond the input's; gates of +-100 are 0 or z, not NaN."""
    t = make((4, 256), torch.float32, torch.float32, bias=False, drop=False)
    t["y"] = (t["y"] + 1000).float()
    t["z"] = torch.where(t["z"] > 0, 100.0, -100.0)
    got, ref = run(t, False), want(t, False)
    # y carries its own rounding of 2^-24 * 1000 per unit of spread (it is given in fp32: exact); the mean's rounding is 1000 u of the spread
    err = (got["x'"].cpu().double() - ref["x'"]).abs()
    assert bool((err <= 2000 * U * 64 * ref["x'"].abs().amax() + 1e-30).all())
    assert all(torch.isfinite(v).all() for v in got.values())


def test_empty_and_nan_rows():
    e = norm_gate_residual(torch.zeros(0, 5, 64, device="cuda", requires_grad=True), torch.zeros(0, 5, 64, device="cuda"), torch.ones(64, device="cuda", requires_grad=True),
                           torch.ones(64, device="cuda"))
    assert e[0].shape == (0, 5, 64)
    (e[0].sum() + e[1].sum()).backward()
    t = make((4, 96), torch.float32, torch.float32)
    clean = run(t, False)
    t["y"][2] = float("nan")
    got = run(t, False)
    keep = [0, 1, 3]
    for n in ("x'", "h", "dx", "dy", "dz"):
        assert torch.equal(got[n][keep], clean[n][keep]) and (n in ("dz",) or torch.isnan(got[n][2]).all()), n


def test_captured_and_repeated_runs_are_equal():
    t = make((6, 50, 96), torch.float32, torch.bfloat16)
    d = {n: v.cuda() for n, v in t.items()}

    def step():
        leaves = {n: d[n].detach().requires_grad_() for n in NAMES}
        x, h = call({**d, **leaves}, True)
        return (x, h, *torch.autograd.grad([x, h], list(leaves.values()), [d["dx"], d["dh"]]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        for n, v in make((6, 50, 96), torch.float32, torch.bfloat16, seed=30 + seed).items():
            d[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [5, 64, 65, 1032, 5000])
def test_rows_at_any_offset_and_distance(D, types):
    t = make((3, 4, D), *types)
    d = {n: v.cuda() for n, v in t.items()}
    want_x, want_h = call(d, False)
    for at, pitch in ((1, D + 1), (3, D + 5), (2, D + 7)):
        views = {}
        for n in ("x", "y", "z"):
            wide = torch.full((3, 4, pitch), float("nan"), device="cuda", dtype=d[n].dtype).flatten()
            wide = torch.cat([wide.new_zeros(at), wide])[at:].view(3, 4, pitch)
            views[n] = wide[..., pitch - D:] if n == "z" else wide[..., :D]
            views[n].copy_(d[n])
        x, h = call({**d, **views}, False)
        assert torch.equal(x, want_x) and torch.equal(h, want_h)
