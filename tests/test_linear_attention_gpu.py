"""Linear attention with a decay for each head (linear_attention_fn, linear_attention_step) against the recurrence in 64 bits.

Tolerances.  Every result is a sum of products with decay factors; the same formula on absolute values gives the sum A of the terms'
magnitudes.  In fp32 each term passes through at most `steps` roundings of relative size u = 2^-24: dk + dv products and the
additions of a chunk (at most 64 tokens), one addition and one decay a chunk after it, and a decay exp2(x) whose exponent carries
|x| u (|x| <= 40 matters: below, the term is 2^-40 of A).  So |error| <= steps * u * A, plus half a step of the output's type (bf16: 2^-8
of the value).  A decay's gradient is taken as differences of sums over its chunk: there A is the sum over the chunk's tokens."""
import pytest
import torch

from mamba_unet_amd import linear_attention_fn, linear_attention_step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def recurrence(q, k, v, g, s0, scale, do=None, ds=None):
    """One sequence in 64 bits: q, k (L, H, dk), v (L, H, dv), g (L, H), s0 (H, dk, dv) -> out, last and, with do, every gradient."""
    L = q.shape[0]
    S, out, states = s0, [], [s0]
    for t in range(L):
        S = g[t].exp()[:, None, None] * S + k[t, :, :, None] * v[t, :, None, :]
        states.append(S)
        out.append(scale * (q[t, :, None, :] @ S)[:, 0])
    out = torch.stack(out) if L else v.clone()
    if do is None:
        return out, S
    D, dq, dk, dv, dg = ds, torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g)
    for t in range(L - 1, -1, -1):
        D = D + scale * q[t, :, :, None] * do[t, :, None, :]
        dq[t] = scale * (states[t + 1] @ do[t, :, :, None])[..., 0]
        dk[t] = (D @ v[t, :, :, None])[..., 0]
        dv[t] = (k[t, :, None, :] @ D)[:, 0]
        dg[t] = g[t].exp() * (D * states[t]).sum((1, 2))
        D = g[t].exp()[:, None, None] * D
    return out, S, dq, dk, dv, dg, D


def make(lens, packed, H, G, dk, dv, dtype, decay="token", init=True, seed=0, span=1.0):
    r = torch.Generator().manual_seed(seed)
    rows, L = (1, sum(lens)) if packed else (len(lens), lens[0])
    t = {"q": torch.randn(rows, L, G, dk, generator=r), "k": torch.randn(rows, L, G, dk, generator=r), "v": torch.randn(rows, L, H, dv, generator=r),
         "do": torch.randn(rows, L, H, dv, generator=r)}
    t = {n: x.to(dtype) for n, x in t.items()}
    t["g"] = -torch.rand(*((H,) if decay == "head" else (rows, L, H)), generator=r) * span
    t["s0"] = torch.randn(len(lens), H, dk, dv, generator=r) if init else None
    t["ds"] = torch.randn(len(lens), H, dk, dv, generator=r)
    return t


def reference(t, lens, packed, scale, absolute=False):
    """Every output and gradient in 64 bits, laid out as the operator's; with `absolute` from the inputs' magnitudes."""
    f = lambda x: x.abs().double() if absolute else x.double()  # noqa: E731
    rows, L, G, dk = t["q"].shape
    H, dv = t["v"].shape[2:]
    rep = H // G
    g = t["g"].double().expand(rows, L, H)
    res = {n: torch.zeros(rows, L, H, d, dtype=torch.float64) for n, d in (("out", dv), ("dq", dk), ("dk", dk), ("dv", dv))}
    res["dg"] = torch.zeros(rows, L, H, dtype=torch.float64)
    res["last"], res["ds0"] = torch.zeros(len(lens), H, dk, dv, dtype=torch.float64), torch.zeros(len(lens), H, dk, dv, dtype=torch.float64)
    at = 0
    for n, m in enumerate(lens):
        row, lo = (0, at) if packed else (n, 0)
        at += m
        sl = slice(lo, lo + m)
        s0 = f(t["s0"][n]) if t["s0"] is not None else torch.zeros(H, dk, dv, dtype=torch.float64)
        a = recurrence(f(t["q"])[row, sl].repeat_interleave(rep, 1), f(t["k"])[row, sl].repeat_interleave(rep, 1), f(t["v"])[row, sl], g[row, sl], s0,
                       scale, f(t["do"])[row, sl], f(t["ds"])[n])
        for name, x in zip(("out", "dq", "dk", "dv", "dg"), (a[0], a[2], a[3], a[4], a[5])):
            res[name][row, sl] = x
        res["last"][n], res["ds0"][n] = a[1], a[6]
        if absolute:            # the terms that meet in a chunk's differences
            both = (f(t["q"])[row, sl].repeat_interleave(rep, 1) * a[2]).sum(-1) + (f(t["k"])[row, sl].repeat_interleave(rep, 1) * a[3]).sum(-1)
            for c in range(0, m, 64):
                res["dg"][row, lo + c:lo + min(c + 64, m)] += both[c:c + 64].sum(0)
    for name in ("dq", "dk"):
        res[name] = res[name].view(rows, L, G, rep, dk).sum(3)
    if t["g"].dim() == 1:
        res["dg"] = res["dg"].sum((0, 1))
    return res


def run(t, lens, packed, grad=True, **kw):
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    if grad:
        for n in ("q", "k", "v", "g", "s0"):
            if d[n] is not None:
                d[n].requires_grad_()
    cu = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda() if packed else None
    out, last = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], initial_state=d["s0"], cu_seqlens=cu, return_last_state=True, **kw)
    res = {"out": out.detach(), "last": last.detach()}
    if grad:
        names = [n for n in ("q", "k", "v", "g", "s0") if d[n] is not None]
        got = torch.autograd.grad([out, last], [d[n] for n in names], [d["do"], d["ds"]])
        res.update(zip(["d" + n for n in names], got))
    return res


def check(got, want, size, steps, extra=1.0):
    for n, x in got.items():
        lim = HALF[x.dtype] * want[n].abs() + steps * U * size[n] * extra + 1e-30
        err = (x.cpu().double() - want[n]).abs()
        assert torch.isfinite(x).all(), n
        assert bool((err <= lim).all()), f"{n}: {float((err / lim).max()):.2f} of the tolerance"


def steps_of(lens, dk, dv):
    return dk + dv + 64 + 40 + 2 * (max(lens) // 32 + 1)


CASES = [
    # lens, packed, H, G, dk, dv, decay, init
    ([1], False, 1, 1, 1, 1, "token", True),
    ([1, 1], False, 4, 2, 64, 64, "token", False),
    ([2], False, 3, 3, 16, 64, "head", True),
    ([63], False, 2, 1, 64, 64, "token", True),
    ([64], False, 2, 2, 64, 64, "token", True),
    ([65, 65], False, 4, 2, 64, 32, "token", True),
    ([33], False, 2, 2, 128, 128, "token", True),
    ([100], False, 4, 1, 128, 64, "head", False),
    ([130], False, 2, 2, 33, 7, "token", True),
    ([130], False, 2, 1, 100, 96, "token", True),
    ([70], False, 3, 1, 24, 128, "head", True),
    ([70], False, 2, 2, 16, 100, "token", False),
    ([700], False, 2, 1, 64, 64, "token", True),
    ([600], False, 1, 1, 128, 128, "token", True),
    ([70, 0, 1, 5, 64, 300], True, 4, 2, 64, 64, "token", True),
    ([0, 31, 0, 33, 0], True, 2, 2, 128, 64, "token", True),
    ([0, 0, 3], True, 2, 1, 16, 16, "head", False),
    ([257, 129], True, 3, 3, 50, 128, "token", False),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_forward_and_every_gradient(case, dtype):
    lens, packed, H, G, dk, dv, decay, init = case
    t = make(lens, packed, H, G, dk, dv, dtype, decay, init)
    scale = dk ** -0.5
    check(run(t, lens, packed), reference(t, lens, packed, scale), reference(t, lens, packed, scale, True), steps_of(lens, dk, dv))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_split_over_segments_equals_one_walk(dtype):
    """A long sequence of few heads is cut into segments; many copies of it in a batch are not: the same numbers within rounding."""
    t = make([3000], False, 2, 1, 64, 64, dtype, seed=3, span=0.05)
    one = run(t, [3000], False)
    n = 300
    big = {k: (x if x is None or k == "g" and x.dim() == 1 else x.expand(n, *x.shape[1:])) for k, x in t.items()}
    d = {k: x.cuda() for k, x in big.items()}
    with torch.no_grad():
        out, last = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], initial_state=d["s0"], return_last_state=True)
    size = reference(t, [3000], False, 64 ** -0.5, True)
    for got, name in ((out[:1], "out"), (last[:1], "last")):
        # both sides are rounded
        lim = 2 * (HALF[got.dtype] * one[name].cpu().double().abs() + steps_of([3000], 64, 64) * U * size[name])
        assert bool(((got - one[name]).cpu().double().abs() <= lim).all()), name
    assert torch.equal(out[0], out[n - 1]) and torch.equal(last[0], last[n - 1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_decays_that_reset(dtype):
    """-inf, the type's lowest value and decays far below exp's range reset the state; the decays behind a reset keep their digits."""
    t = make([150], False, 2, 1, 64, 64, dtype, seed=5, span=0.02)
    g = t["g"]
    g[0, 10, 0], g[0, 11, 0], g[0, 70, 0], g[0, 71, 1], g[0, 149, 1] = -float("inf"), torch.finfo(torch.float32).min, -1e4, -200.0, -float("inf")
    ref, size = dict(t), dict(t)
    ref["g"] = g.clamp(min=-150.0)                 # exp(-150) is 0 in fp32; the 64-bit recurrence has no 0 * inf either way
    got = run(t, [150], False)
    check(got, reference(ref, [150], False, 0.125), reference(ref, [150], False, 0.125, True), steps_of([150], 64, 64))
    before = run({n: (x if x is None or n in ("s0", "ds") else x[:, 72:149] if x.dim() > 1 else x) for n, x in t.items()} | {"s0": None}, [77], False, grad=False)
    assert torch.isfinite(before["out"]).all()


def test_strided_views_of_a_fused_projection():
    """q, k, v as slices of one tensor, and with the head axis in front, are used in place; an odd offset is copied: the same results."""
    H, dk, L = 4, 64, 130
    fused = torch.randn(2, L, 3 * H * dk, generator=torch.Generator().manual_seed(1)).cuda().bfloat16()
    g = -torch.rand(2, L, H, generator=torch.Generator().manual_seed(2)).cuda()
    views = [x.unflatten(2, (H, dk)) for x in fused.split(H * dk, 2)]
    want = linear_attention_fn(*[x.contiguous() for x in views], g)
    assert torch.equal(linear_attention_fn(*views, g), want)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in views]
    assert torch.equal(linear_attention_fn(*heads_first, g.transpose(1, 2).contiguous().transpose(1, 2)), want)
    odd = torch.empty(2 * L * H * dk + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, L, H, dk)
    odd.copy_(views[0])
    assert torch.equal(linear_attention_fn(odd, views[1], views[2], g), want)
    assert torch.equal(linear_attention_fn(views[0], views[1], views[2].flip(3).flip(3), g), want)


def test_rows_outside_every_sequence_and_bad_offsets():
    """Rows in front of the first and behind the last sequence give zeros, whatever they hold; offsets outside the row are clamped."""
    t = make([90], False, 2, 2, 64, 64, torch.float32, init=False)
    d = {n: x.cuda().requires_grad_(n in ("q", "k", "v", "g")) for n, x in t.items() if x is not None and n != "ds"}
    poison = {n: d[n].detach().clone() for n in ("q", "k", "v", "g")}
    for n in poison:
        poison[n][:, :7] = float("nan")
        poison[n][:, 60:] = float("nan")
        poison[n].requires_grad_()
    cu = torch.tensor([7, 40, 60], dtype=torch.int32, device="cuda")
    out = linear_attention_fn(poison["q"], poison["k"], poison["v"], poison["g"], cu_seqlens=cu)
    grads = torch.autograd.grad(out, [poison[n] for n in ("q", "k", "v", "g")], d["do"])
    for x in (out, *grads):
        assert torch.isfinite(x).all() and not x[:, :7].any() and not x[:, 60:].any()
    for lo, hi in ((7, 40), (40, 60)):
        want = linear_attention_fn(*[d[n][:, lo:hi] for n in ("q", "k", "v", "g")])
        assert torch.allclose(out[:, lo:hi], want, rtol=1e-5, atol=1e-6)
    for bad in ([-5, 90], [0, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1]):
        got = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], cu_seqlens=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert torch.equal(got, linear_attention_fn(d["q"], d["k"], d["v"], d["g"]))
    # descending offsets: an empty sequence, and the hint may be too small
    got = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], cu_seqlens=torch.tensor([90, 0], dtype=torch.int32, device="cuda"))
    assert not got.any()
    got = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], cu_seqlens=torch.tensor([0, 90], dtype=torch.int32, device="cuda"), max_seqlen=1)
    assert torch.allclose(got, linear_attention_fn(d["q"], d["k"], d["v"], d["g"]), rtol=1e-5, atol=1e-6)


def test_empty_rows_and_partial_gradients():
    q = torch.zeros(2, 0, 2, 16, device="cuda", requires_grad=True)
    v, g, s0 = torch.zeros(2, 0, 2, 16, device="cuda"), torch.zeros(2, 0, 2, device="cuda"), torch.randn(2, 2, 16, 16, device="cuda", requires_grad=True)
    out, last = linear_attention_fn(q, q, v, g, initial_state=s0, return_last_state=True)
    assert out.shape == (2, 0, 2, 16) and torch.equal(last, s0)
    last.backward(torch.ones_like(last))
    assert torch.equal(s0.grad, torch.ones_like(s0))
    # only the last state, only the output: the other's gradient is 0
    t = make([70], False, 2, 1, 64, 64, torch.float32)
    d = {n: x.cuda().requires_grad_(n in ("q", "k", "v", "g", "s0")) for n, x in t.items()}
    out, last = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], initial_state=d["s0"], return_last_state=True)
    a = torch.autograd.grad(out, [d[n] for n in ("q", "k", "v", "g", "s0")], d["do"], retain_graph=True)
    b = torch.autograd.grad(last, [d[n] for n in ("q", "k", "v", "g", "s0")], d["ds"], retain_graph=True)
    both = torch.autograd.grad([out, last], [d[n] for n in ("q", "k", "v", "g", "s0")], [d["do"], d["ds"]])
    assert not b[0].any()
    size = reference(t, [70], False, 0.125, True)
    for n, x, y, z in zip(("dq", "dk", "dv", "dg", "ds0"), a, b, both):
        assert bool(((x + y - z).cpu().double().abs() <= 3 * steps_of([70], 64, 64) * U * size[n]).all()), n


def test_gradients_against_differences():
    """Central differences of <do, out> + <ds, last> along random directions.  The sum is linear in q, v (and in k, s0) so those differences are exact up
    to rounding; for g the step is 2^-7 and the third-order term below 2^-14 of the change's own size."""
    t = make([90], False, 2, 1, 32, 32, torch.float32, seed=8, span=0.3)
    got = run(t, [90], False)

    def value(**kw):
        d = {n: x.cuda() for n, x in {**t, **kw}.items()}
        out, last = linear_attention_fn(d["q"], d["k"], d["v"], d["g"], initial_state=d["s0"], return_last_state=True)
        return float((out.double() * d["do"]).sum() + (last.double() * d["ds"]).sum())

    size = reference(t, [90], False, 32 ** -0.5, True)
    r = torch.Generator().manual_seed(9)
    for n in ("q", "k", "v", "g", "s0"):
        step = torch.randn(t[n].shape, generator=r) * 2.0 ** -7
        up, down = t[n] + step, t[n] - step
        diff = value(**{n: up}) - value(**{n: down})
        want = float((got["d" + n].cpu().double() * (up.double() - down.double())).sum())
        # rounding of the two values (norm-wise: independent errors of u-size terms) and the third order in g
        noise = steps_of([90], 32, 32) * U * (float(size["out"].norm()) * 6 + float(size["last"].norm()) * 6)
        assert abs(diff - want) <= noise + 2.0 ** -10 * float((size["d" + n] * step.abs().double()).norm()) * 2, (n, diff, want)


def test_captured_forward_and_backward_replay():
    t = make([300], False, 4, 2, 64, 64, torch.bfloat16, "head")
    d = {n: x.cuda() for n, x in t.items()}
    names = ("q", "k", "v", "g", "s0")

    def step():
        leaves = [d[n].detach().requires_grad_() for n in names]
        out, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
        return (out, last, *torch.autograd.grad([out, last], leaves, [d["do"], d["ds"]]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        new = make([300], False, 4, 2, 64, 64, torch.bfloat16, "head", seed=20 + seed)
        for n in d:
            d[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_results_do_not_change_between_calls_and_streams():
    t = make([500], False, 4, 1, 128, 64, torch.bfloat16)
    a = run(t, [500], False)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = run(t, [500], False)
    side.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n]), n


# ---------------------------------------------------------------------------------------------------- one token

STEP_CASES = [(1, 0, 1, 1, 1, 1, "token"), (3, 0, 4, 2, 64, 64, "token"), (5, 9, 4, 4, 16, 64, "head"), (2, 2, 2, 1, 128, 128, "token"),
              (7, 8, 6, 3, 50, 65, "token"), (4, 6, 2, 2, 33, 4, "head"), (64, 70, 8, 2, 128, 64, "token"), (2, 3, 2, 1, 100, 96, "token")]


def step_inputs(B, pool, H, G, dk, dv, decay, dtype, seed=0):
    r = torch.Generator().manual_seed(seed)
    t = {"q": torch.randn(B, G, dk, generator=r).to(dtype), "k": torch.randn(B, G, dk, generator=r).to(dtype), "v": torch.randn(B, H, dv, generator=r).to(dtype),
         "g": -torch.rand(*((H,) if decay == "head" else (B, H)), generator=r), "state": torch.randn(pool or B, H, dk, dv, generator=r)}
    t["idx"] = torch.randperm(pool, generator=r)[:B].to(torch.int32) if pool else None
    return t


def step_reference(t, scale, absolute=False):
    f = lambda x: x.abs().double() if absolute else x.double()  # noqa: E731
    B, G, dk = t["q"].shape
    H, dv = t["v"].shape[1:]
    state, out = f(t["state"]), torch.zeros(B, H, dv, dtype=torch.float64)
    g = t["g"].double().expand(B, H)
    for b in range(B):
        s = b if t["idx"] is None else int(t["idx"][b])
        if not 0 <= s < state.shape[0]:
            continue
        q, k = f(t["q"])[b].repeat_interleave(H // G, 0), f(t["k"])[b].repeat_interleave(H // G, 0)
        state[s] = g[b].exp()[:, None, None] * state[s] + k[:, :, None] * f(t["v"])[b][:, None, :]
        out[b] = scale * (q[:, None, :] @ state[s])[:, 0]
    return out, state


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", STEP_CASES, ids=[str(i) for i in range(len(STEP_CASES))])
def test_single_token(case, dtype):
    t = step_inputs(*case, dtype)
    scale = t["q"].shape[2] ** -0.5
    want, size = step_reference(t, scale), step_reference(t, scale, True)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    out = linear_attention_step(d["state"], d["q"], d["k"], d["v"], d["g"], state_indices=d["idx"])
    # a state element: two roundings of products, one of the sum, exp within 2 u; the output adds dk products
    check({"out": out, "state": d["state"]}, dict(zip(("out", "state"), want)), dict(zip(("out", "state"), size)), t["q"].shape[2] + 8)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_step_slots_named_twice_padded_or_outside(wide):
    """Requests of one slot are applied in order; -1 and indices outside the pool give zeros and change nothing."""
    t = step_inputs(8, 5, 4, 2, 64, 64, "token", torch.float32)
    t["idx"] = torch.tensor([3, -1, 0, 3, 5, 3, 2 ** 31 - 1, 0]).to(wide)
    want, size = step_reference(t, 0.125), step_reference(t, 0.125, True)
    d = {n: x.cuda() for n, x in t.items()}
    for _ in range(2):
        state = d["state"].clone()
        out = linear_attention_step(state, d["q"], d["k"], d["v"], d["g"], state_indices=d["idx"])
        check({"out": out, "state": state}, dict(zip(("out", "state"), want)), dict(zip(("out", "state"), size)), 3 * (64 + 8))
        assert not out[1].any() and not out[4].any() and not out[6].any()
        assert torch.equal(state[[1, 2, 4]].cpu(), t["state"][[1, 2, 4]])
    if wide is torch.int64:
        state = d["state"].clone()
        far = torch.tensor([2 ** 32, 2 ** 32 + 3, -2 ** 33] + [-1] * 5, device="cuda")
        assert not linear_attention_step(state, d["q"], d["k"], d["v"], d["g"], state_indices=far).any() and torch.equal(state, d["state"])


def test_step_on_a_layer_of_a_pool_and_strided_inputs():
    t = step_inputs(3, 5, 4, 2, 64, 64, "token", torch.bfloat16)
    d = {n: x.cuda() for n, x in t.items()}
    layers = torch.randn(5, 3, 4, 64, 64, device="cuda")
    keep = layers.clone()
    layers[:, 1] = d["state"]
    fused = torch.cat([d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1)], 1)
    q, k, v = fused[:, :128].unflatten(1, (2, 64)), fused[:, 128:256].unflatten(1, (2, 64)), fused[:, 256:].unflatten(1, (4, 64))
    out = linear_attention_step(layers[:, 1], q, k, v, d["g"], state_indices=d["idx"])
    want = linear_attention_step(d["state"], d["q"], d["k"], d["v"], d["g"], state_indices=d["idx"])
    assert torch.equal(out, want) and torch.equal(layers[:, 1], d["state"])
    assert torch.equal(layers[:, 0], keep[:, 0]) and torch.equal(layers[:, 2], keep[:, 2])


def test_step_and_prompt_under_inference_mode():
    t = step_inputs(3, 0, 4, 2, 64, 64, "token", torch.bfloat16)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    want = d["state"].clone()
    out = linear_attention_step(want, d["q"], d["k"], d["v"], d["g"])
    with torch.inference_mode():
        state = d["state"].clone()
        assert torch.equal(linear_attention_step(state, d["q"], d["k"], d["v"], d["g"]), out) and torch.equal(state, want)
        assert linear_attention_fn(d["q"][:, None], d["k"][:, None], d["v"][:, None], d["g"][:, None], initial_state=d["state"]).shape == (3, 1, 4, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_prompt_then_tokens_equals_the_whole_sequence(dtype):
    """As a server uses them: packed prompts through linear_attention_fn into a pool, then tokens one by one, in a captured graph."""
    lens, H, G, dk, dv, new = [40, 65, 1], 4, 2, 64, 64, 6
    whole = make([max(lens) + new] * 3, False, H, G, dk, dv, dtype, init=False, seed=11, span=0.2)
    d = {n: None if x is None else x.cuda() for n, x in whole.items()}
    pick = lambda n: torch.cat([d[n][i, :m] for i, m in enumerate(lens)])[None]  # noqa: E731
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    with torch.no_grad():
        _, last = linear_attention_fn(pick("q"), pick("k"), pick("v"), pick("g"), cu_seqlens=cu, max_seqlen=max(lens), return_last_state=True)
    pool = torch.full((6, H, dk, dv), float("nan"), device="cuda")
    idx = torch.tensor([4, 0, 3], device="cuda", dtype=torch.int32)
    pool[idx.long()] = last
    tok = lambda n, s: torch.stack([d[n][i, m + s] for i, m in enumerate(lens)])  # noqa: E731
    bufs = [tok(n, 0).clone() for n in ("q", "k", "v", "g")]
    start = pool.clone()
    linear_attention_step(pool, *bufs, state_indices=idx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_attention_step(pool, *bufs, state_indices=idx)
    pool.copy_(start)
    size = reference(whole, [max(lens) + new] * 3, False, 0.125, True)["out"]
    ref = reference(whole, [max(lens) + new] * 3, False, 0.125)["out"]
    for s in range(new):
        for b, n in zip(bufs, ("q", "k", "v", "g")):
            b.copy_(tok(n, s))
        graph.replay()
        for i, m in enumerate(lens):
            err = (out[i].cpu().double() - ref[i, m + s]).abs()
            assert bool((err <= HALF[dtype] * ref[i, m + s].abs() + steps_of([max(lens) + new], dk, dv) * U * size[i, m + s]).all())
    assert torch.isnan(pool[1]).all() and torch.isnan(pool[2]).all()


# ---------------------------------------------------------------------------------------------------- refusals

def test_refusals():
    q, v, g = torch.zeros(1, 4, 2, 16).cuda(), torch.zeros(1, 4, 4, 16).cuda(), torch.zeros(4).cuda()
    cu = torch.tensor([0, 4], dtype=torch.int32).cuda()
    ok = dict(q=q, k=q, v=v, log_decay=g)
    for bad, word in ((dict(k=q[:, :3]), "equal"), (dict(v=v[:, :3]), "equal"), (dict(v=v[:, :, :3], log_decay=g[:3]), "multiple"), (dict(log_decay=g[:3]), "log_decay"),
                      (dict(log_decay=torch.zeros(1, 4, 1).cuda()), "log_decay"), (dict(q=torch.zeros(1, 4, 2, 129).cuda(), k=torch.zeros(1, 4, 2, 129).cuda()), "128"),
                      (dict(initial_state=torch.zeros(2, 4, 16, 16).cuda()), "initial_state"), (dict(cu_seqlens=cu.long()), "int32"), (dict(cu_seqlens=cu[:1]), "two"),
                      (dict(cu_seqlens=torch.zeros(4, dtype=torch.int32).cuda()[::2]), "contiguous"),
                      (dict(q=torch.zeros(2, 4, 2, 16).cuda(), k=torch.zeros(2, 4, 2, 16).cuda(), v=torch.zeros(2, 4, 4, 16).cuda(), cu_seqlens=cu), "batch must be 1"),
                      (dict(log_decay=g.int()), "floating")):
        with pytest.raises(ValueError, match=word):
            linear_attention_fn(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="GPU"):
        linear_attention_fn(**{**ok, "v": v.cpu()})
    state = torch.zeros(3, 4, 16, 16).cuda()
    ok = dict(state=state, q=q[0, :3], k=q[0, :3], v=v[0, :3], log_decay=g)
    for bad, word in ((dict(state=state.bfloat16()), "fp32"), (dict(state=state[:, :3]), "fp32"), (dict(state=state[:2]), "state_indices"),
                      (dict(state=state.transpose(2, 3)), "dense"), (dict(state=state[:1].expand(3, 4, 16, 16)), "overlap"),
                      (dict(state_indices=torch.zeros(2, dtype=torch.int32).cuda()), "state_indices"), (dict(state_indices=torch.zeros(3).cuda()), "state_indices"),
                      (dict(log_decay=torch.zeros(2, 4).cuda()), "log_decay"), (dict(k=q[0, :2]), "equal")):
        with pytest.raises(ValueError, match=word):
            linear_attention_step(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_attention_step(**{**ok, "q": q[0, :3].clone().requires_grad_()})
    version = state._version
    linear_attention_step(**ok)
    assert state._version > version


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(16, 64), (64, 32), (33, 100), (128, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_reach_later_rows_only(dtype, dk, dv, bad):
    t = {n: x.cuda() for n, x in make([300], False, 2, 2, dk, dv, dtype, seed=5).items()}
    call = lambda **kw: linear_attention_fn(*[kw.get(n, t[n]) for n in ("q", "k", "v", "g")], initial_state=t["s0"], return_last_state=True)  # noqa: E731
    out, last = call()
    v = t["v"].clone()
    v[0, 100, 0, 5], v[0, 37, 1, 7], v[0, 150, 1, 7] = bad, -bad, bad
    got, end = call(v=v)
    assert torch.equal(got[0, :100, 0], out[0, :100, 0]) and torch.equal(got[0, :37, 1], out[0, :37, 1])
    assert not torch.isfinite(got[0, 100:, 0, 5]).any() and not torch.isfinite(got[0, 37:, 1, 7]).any()
    assert not torch.isfinite(end[0, 0, :, 5]).any() and not torch.isfinite(end[0, 1, :, 7]).any()
    keep = torch.ones(2, dv, dtype=torch.bool, device="cuda")
    keep[0, 5] = keep[1, 7] = False
    assert torch.equal(got[0, :, keep], out[0, :, keep]) and torch.equal(end[0].transpose(1, 2)[keep], last[0].transpose(1, 2)[keep])
    for n in ("k", "q", "g"):
        x = t[n].clone()
        x[0, 90, 1] = float("nan")
        got, _ = call(**{n: x})
        assert torch.equal(got[0, :90], out[0, :90]) and torch.equal(got[0, :, 0], out[0, :, 0]) and torch.isnan(got[0, 90, 1]).all()
        assert n != "q" or torch.equal(got[0, 91:], out[0, 91:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hint", [None, 1, 900])
def test_many_packed_sequences_of_which_a_few_are_long(dtype, hint):
    lens = [0, 1, 2, 0, 63, 64, 65, 3] * 4 + [900] + [5, 0, 128] * 3 + [1500, 0, 0]
    t = make(lens, True, 2, 1, 32, 16, dtype, seed=11)
    scale = 32 ** -0.5
    want, size = reference(t, lens, True, scale), reference(t, lens, True, scale, absolute=True)
    check(run(t, lens, True, max_seqlen=hint), want, size, steps_of(lens, 32, 16))


def test_more_sequences_than_a_grid_axis_holds():
    """70000 sequences of one token and one that is split: the states' scratch holds a segment each, not the longest one's number of them."""
    n, L, dk, dv = 70000, 600, 4, 3
    r = torch.Generator().manual_seed(3)
    T = n + L
    q, k, v, g = (torch.randn(1, T, 2, d, generator=r).cuda() for d in (dk, dk, dv, 1))
    g = -g[..., 0].abs()
    cu = torch.cat([torch.arange(n // 2 + 1), torch.arange(n // 2, n + 1) + L]).to(torch.int32).cuda()       # the long one in the middle
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        out, last = linear_attention_fn(q, k, v, g, scale=1.0, cu_seqlens=cu, return_last_state=True)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 64 << 20
    one = torch.cat([torch.arange(n // 2), torch.arange(n // 2, n) + L]).cuda()
    d = lambda x: x[0, one].double()  # noqa: E731
    want = (d(q) * d(k)).sum(-1, keepdim=True) * d(v)
    assert bool(((out[0, one].double() - want).abs() <= (dk + 4) * U * (d(q) * d(k)).abs().sum(-1, keepdim=True) * d(v).abs() + 1e-30).all())
    lo = n // 2
    t = {"q": q[:, lo:lo + L], "k": k[:, lo:lo + L], "v": v[:, lo:lo + L], "g": g[:, lo:lo + L], "s0": None, "do": torch.zeros(1, L, 2, dv), "ds": torch.zeros(1, 2, dk, dv)}
    t = {m: None if x is None else x.cpu() for m, x in t.items()}
    ref, size = (reference(t, [L], False, 1.0, absolute=a) for a in (False, True))
    check({"out": out[:, lo:lo + L], "last": last[lo:lo + 1]}, ref, size, steps_of([L], dk, dv))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_expanded_and_single_row_views(dtype):
    """Tensors that repeat a row over tokens, batch or heads, and a row whose token stride means nothing, give what copies of them give."""
    t = {n: x.cuda() for n, x in make([70, 70], False, 4, 2, 16, 24, dtype, seed=9).items()}
    views = {"q": t["q"][:, :1].expand(-1, 70, -1, -1), "k": t["k"][:1].expand(2, -1, -1, -1), "v": t["v"][:, :, :1].expand(-1, -1, 4, -1), "g": t["g"][:, :, :1].expand(-1, -1, 4)}
    names = ("q", "k", "v", "g")
    dense = {n: x.contiguous() for n, x in views.items()}
    for use in ({"q"}, {"k"}, {"v"}, {"g"}, set(names)):
        res = []
        for d in (views, dense):
            leaves = [(d[n] if n in use else t[n]).detach().requires_grad_() for n in names]
            out = linear_attention_fn(*leaves, initial_state=t["s0"])
            res.append([out, *torch.autograd.grad(out, leaves, t["do"])])
        assert all(torch.equal(a, b) for a, b in zip(*res))
    still = t["g"][:, :1].expand(-1, 70, -1)                       # one decay for all tokens, but given (and differentiated) for each
    res = []
    for g in (still, still.contiguous()):
        g = g.detach().requires_grad_()
        res.append(torch.autograd.grad(linear_attention_fn(t["q"], t["k"], t["v"], g, initial_state=t["s0"]), g, t["do"])[0])
    assert torch.equal(*res) and bool((res[0] != 0).all())
    one = {n: t[n][:, :1] for n in names}
    odd = {n: x.as_strided(x.shape, (x.stride(0), 1, *x.stride()[2:])) for n, x in one.items()}
    want = linear_attention_fn(*[one[n].contiguous() for n in names], initial_state=t["s0"])
    assert torch.equal(linear_attention_fn(*[odd[n] for n in names], initial_state=t["s0"]), want)
    far = torch.empty_strided(t["v"].shape, (128, 1 << 23, 24, 1), device="cuda", dtype=dtype)[:, :3].copy_(t["v"][:, :3])
    q, k, g = (t[n][:, :3] for n in ("q", "k", "g"))
    assert torch.equal(linear_attention_fn(q, k, far, g), linear_attention_fn(q, k, t["v"][:, :3], g))


def test_differentiating_twice_raises():
    from mamba_unet_amd import norm_gate_residual
    t = {n: x.cuda() for n, x in make([5], False, 2, 2, 16, 16, torch.float32).items()}
    q = t["q"].requires_grad_()
    for out in (linear_attention_fn(q, t["k"], t["v"], t["g"]), norm_gate_residual(q, t["k"], torch.ones(16).cuda(), torch.ones(16).cuda())[1]):
        g, = torch.autograd.grad(out.sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            (g ** 2).sum().backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward(reentrant):
    from torch.utils.checkpoint import checkpoint
    t = {n: x.cuda() for n, x in make([130, 130], False, 4, 2, 32, 32, torch.bfloat16, seed=2).items()}
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    call = lambda *a: linear_attention_fn(*a)  # noqa: E731
    grads = []
    for out in (call(*leaves), checkpoint(call, *leaves, use_reentrant=reentrant)):
        for x in leaves:
            x.grad = None
        out.backward(t["do"])
        grads.append([x.grad.clone() for x in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_a_changed_input_is_noticed():
    t = {n: x.cuda() for n, x in make([40], False, 2, 2, 16, 16, torch.float32).items()}
    k = t["k"].clone().requires_grad_()
    out = linear_attention_fn(t["q"].requires_grad_(), k * 1.0, t["v"], t["g"])
    q2 = t["q"].detach()
    q2.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
