"""The gradient of linear_attention_fn's log_decay, for every token and as one decay for each head, against the recurrence in 64 bits.

    dg_t = exp(g_t) <D_t, S_{t-1}>,   D: gradient of the state behind token t,   S: the state in front of it

On positive inputs every term of it is positive, so no rounding is larger than its share of the result, and the limit is relative to the gradient itself,
however small a strong decay makes it: n roundings of u = 2^-24 with
    dk + dv          products and additions of q . k, do . v and of the products with a state
    2 * 200 a chunk  S and D: at most 64 additions of a chunk (in bf16 of three terms each), a decay and its addition
    2 * 128          the sums over the pairs of a chunk (at most 64 in a tile's rows and columns, ten tiles, sixteen waves, dk * dv / lanes of <D, S>)
    3 * sum |g|      a decay factor exp2(x) carries |x| u, x from sums of g, on both sides of t
and, for one decay for each head, one addition a token more.  On inputs of either sign the same count bounds the error relative to the gradient of the
inputs' magnitudes (the same formula on them), again without a term for a chunk's other pairs."""
import pytest
import torch

from mamba_unet_amd import linear_attention_fn

U = 2.0 ** -24
BAD = (1e-2, 1e-4, 1e-6, 1e-8, 1e-12)


def gradient(t, lens, packed, scale, state=True):
    """dg (rows, L, H), or (H,) for one decay a head, in 64 bits; without the last state's gradient if not `state`"""
    rows, L, G, dk = t["q"].shape
    H, dv = t["v"].shape[2:]
    q, k = (t[n].double().repeat_interleave(H // G, 2) for n in ("q", "k"))
    v, do, g = t["v"].double(), t["do"].double(), t["g"].double().expand(rows, L, H)
    out = torch.zeros(rows, L, H, dtype=torch.float64)
    at = 0
    for n, m in enumerate(lens):
        row, lo = (0, at) if packed else (n, 0)
        at += m
        S = [t["s0"][n].double() if t["s0"] is not None else torch.zeros(H, dk, dv, dtype=torch.float64)]
        f = g[row].exp()[:, :, None, None]
        for i in range(lo, lo + m):
            S.append(f[i] * S[-1] + k[row, i, :, :, None] * v[row, i, :, None, :])
        D = t["ds"][n].double() * state
        for i in range(lo + m - 1, lo - 1, -1):
            D = D + scale * q[row, i, :, :, None] * do[row, i, :, None, :]
            D = f[i] * D
            out[row, i] = (D * S[i - lo]).sum((1, 2))
    return out.sum((0, 1)) if t["g"].dim() == 1 else out


def make(case, dtype, decay, strong, positive=True, seed=0):
    lens, packed, H, G, dk, dv, init = case
    r = torch.Generator().manual_seed(seed)
    rows, L = (1, sum(lens)) if packed else (len(lens), lens[0])
    rnd = (lambda *s: 0.5 + torch.rand(*s, generator=r)) if positive else (lambda *s: torch.randn(*s, generator=r))
    t = {"q": rnd(rows, L, G, dk), "k": rnd(rows, L, G, dk), "v": rnd(rows, L, H, dv), "do": rnd(rows, L, H, dv)}
    t = {n: x.to(dtype) for n, x in t.items()}
    t["s0"], t["ds"] = rnd(len(lens), H, dk, dv) if init else None, rnd(len(lens), H, dk, dv)
    if decay == "head":
        t["g"] = -(torch.rand(H, generator=r) * (3.0 if strong else 0.05) + 0.005)
    else:
        t["g"] = -torch.rand(rows, L, H, generator=r) * 0.05
        if strong:                                  # every 29th token of a head and the first and the last of a chunk of 64
            for i in range(L):
                for h in range(H):
                    if (i + 7 * h) % 29 == 28 or (i + h) % 64 in (0, 63) and i > 70:
                        t["g"][:, i, h] = float(torch.tensor(BAD[(i + h) % len(BAD)], dtype=torch.float64).log())
    return t


def roundings(t, lens, dk, dv):
    n = dk + dv + 400 * (max(lens) // 32 + 1) + 256 + 3 * (float(t["g"].abs().max()) * max(lens) if t["g"].dim() == 1 else float(t["g"].double().abs().sum(1).max()))
    return n + (sum(lens) if t["g"].dim() == 1 else 0)


CASES = [
    ([64], False, 1, 1, 64, 64, True),
    ([65], False, 2, 1, 16, 64, False),
    ([33, 33], False, 4, 2, 33, 24, True),
    ([200], False, 4, 1, 128, 64, True),
    ([130], False, 2, 2, 128, 128, True),
    ([130], False, 2, 1, 32, 100, False),
    ([200], False, 2, 2, 64, 128, True),
    ([700], False, 2, 1, 64, 64, True),              # split into segments
    ([700], False, 2, 2, 16, 64, False),
    ([520], False, 2, 1, 128, 64, True),
    ([70, 0, 1, 5, 64, 600], True, 4, 2, 64, 64, True),
]


def limit(t, case, positive):
    lens, packed, _, _, dk, dv, _ = case
    want = gradient(t, lens, packed, 0.25)
    a = {n: None if x is None else x if n == "g" else x.abs() for n, x in t.items()}
    size = want if positive else gradient(a, lens, packed, 0.25)
    return want, roundings(t, lens, dk, dv) * U * size + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("positive", [True, False], ids=["positive", "signs"])
@pytest.mark.parametrize("strong", [False, True], ids=["mild", "strong"])
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_gradient_of_the_decays(case, dtype, decay, strong, positive):
    lens, packed = case[:2]
    t = make(case, dtype, decay, strong, positive)
    want, lim = limit(t, case, positive)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda() if packed else None
    g = d["g"].requires_grad_()
    out, last = linear_attention_fn(d["q"], d["k"], d["v"], g, scale=0.25, initial_state=d["s0"], cu_seqlens=cu, return_last_state=True)
    got, = torch.autograd.grad([out, last], g, [d["do"], d["ds"]])
    err = (got.cpu().double() - want).abs()
    assert bool((err <= lim).all()), f"{float((err / lim).max()):.2f} of the tolerance"
    if decay == "token" and not case[-1]:
        assert not got[:, 0].any()                  # nothing in front of the first token


@pytest.mark.parametrize("strong", [False, True], ids=["mild", "strong"])
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_the_limit_binds(case, decay, strong):
    """A gradient of zero, one that is off by 1 % and one that leaves out the last state's gradient do not pass."""
    t = make(case, torch.float32, decay, strong)
    want, lim = limit(t, case, True)
    some = want > 0
    assert bool((want[some] > lim[some]).all()) and bool((0.01 * want[some] > lim[some]).all())
    without = gradient(t, case[0], case[1], 0.25, state=False)
    assert bool(((want - without).abs() > lim)[some].any())


def test_the_formula_against_differences():
    case = ([9], False, 2, 1, 3, 2, True)
    t = {n: x.double() for n, x in make(case, torch.float32, "token", False, False, seed=4).items()}

    def value(g):
        S, total = t["s0"][0], 0.0
        for i in range(9):
            S = g[0, i].exp()[:, None, None] * S + t["k"][0, i].repeat_interleave(2, 0)[:, :, None] * t["v"][0, i][:, None, :]
            total = total + 0.25 * (t["q"][0, i].repeat_interleave(2, 0)[:, None, :] @ S)[:, 0].mul(t["do"][0, i]).sum()
        return float(total + (S * t["ds"][0]).sum())

    got = gradient(t, [9], False, 0.25)
    for i in range(9):
        for h in range(2):
            e = torch.zeros_like(t["g"])
            e[0, i, h] = 1e-5
            assert abs((value(t["g"] + e) - value(t["g"] - e)) / 2e-5 - float(got[0, i, h])) <= 1e-7 * (1 + abs(float(got[0, i, h])))
