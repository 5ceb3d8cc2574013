"""Nothing between linear_attention_fn's inputs and its rounded results has less than the 24 bits of fp32, in bf16 too.

The inputs are whole numbers and all decays are 1, so that every weight, state and partial sum is a whole number below 2^24 and fp32 arithmetic makes no error at
all: results equal the exact ones, rounded once to the type.  Weights and states have 18 and 19 bits and come in pairs that cancel: (s, 3 s) times (3 u, -u).  One
that has been cut to 16 or 17 bits on the way leaves a difference of a few units, where the exact result is 0."""
import pytest
import torch

from mamba_unet_amd import linear_attention_fn
from test_linear_attention_gpu import recurrence

pytestmark = pytest.mark.gpu
H, L = 2, 150


class Numbers:
    """Whole numbers of one seed: along axis `at`, neighbours are x, 3 x (thrice) or 3 x, -x (cancel)."""

    def __init__(self, seed):
        self.r = torch.Generator().manual_seed(seed)

    def draw(self, lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=self.r).double()

    def pairs(self, lo, hi, shape, at, thrice):
        half = list(shape)
        half[at] = (shape[at] + 1) // 2
        x = self.draw(lo, hi, *half)
        if not thrice:
            x = x * (2 * self.draw(0, 1, *half) - 1)
        both = torch.stack((x, 3 * x) if thrice else (3 * x, -x), at + 1)
        return both.flatten(at, at + 1).narrow(at, 0, shape[at])


def problem(kind, dk, dv, seed=0):
    n = Numbers(seed)
    z = {"q": torch.zeros(1, L, H, dk), "k": torch.zeros(1, L, H, dk), "v": torch.zeros(1, L, H, dv), "do": torch.zeros(1, L, H, dv),
         "s0": torch.zeros(1, H, dk, dv), "ds": torch.zeros(1, H, dk, dv)}
    z = {m: x.double() for m, x in z.items()}

    def scores(a, b, d):
        """a . b about 120000 over d numbers, b thrice along the tokens"""
        c = 27 if d >= 64 else 75
        e = 120000 // (d * c)
        z[a] = n.draw(max(1, e - e // 4), e + e // 4, 1, L, H, d)
        z[b] = n.pairs(c - c // 8, c + c // 8, (1, L, H, d), 1, True)

    def state(s, x, at, d):
        """a state of about 2^16 and 2^18, cancelling along its axis `at`, and a vector that is thrice along it"""
        z[s] = n.pairs(1 << 15, 1 << 16, (1, H, dk, dv), at, False)
        z[x] = n.pairs(1, 2, (1, L, H, d), 3, True)
        z[x][..., 2 * (d // 2):] = 0                       # (an odd last one has no partner)

    if kind == "scores in out":
        scores("q", "k", dk)
        z["v"] = n.pairs(1, 1, (1, L, H, dv), 1, False)
    elif kind == "state in out":
        state("s0", "q", 2, dk)
    elif kind == "scores in dq":
        scores("do", "v", dv)
        z["k"] = n.pairs(1, 1, (1, L, H, dk), 1, False)
    elif kind == "scores in dk":
        scores("v", "do", dv)
        z["q"] = n.pairs(1, 1, (1, L, H, dk), 1, False)
    elif kind == "scores in dv":
        scores("k", "q", dk)
        z["do"] = n.pairs(1, 1, (1, L, H, dv), 1, False)
    elif kind == "state in dq":
        state("s0", "do", 3, dv)
    elif kind == "state in dk":
        state("ds", "v", 3, dv)
    else:
        state("ds", "k", 2, dk)
    return z


KINDS = {"scores in out": "out", "state in out": "out", "scores in dq": "dq", "scores in dk": "dk", "scores in dv": "dv", "state in dq": "dq", "state in dk": "dk",
         "state in dv": "dv"}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk,dv", [(16, 64), (64, 64), (64, 128), (128, 64), (128, 128), (34, 66)])
def test_whole_numbers_are_exact(dk, dv, kind, dtype):
    t = problem(kind, dk, dv)
    out, _, dq, dk_, dv_, _, _ = recurrence(*(t[n][0] for n in ("q", "k", "v")), torch.zeros(L, H).double(), t["s0"][0], 1.0, t["do"][0], t["ds"][0])
    want = {"out": out, "dq": dq, "dk": dk_, "dv": dv_}[KINDS[kind]].reshape(L, H, -1)
    assert bool((want == 0).any())
    d = {n: x.to(dtype if n not in ("s0", "ds") else torch.float32) for n, x in t.items()}
    assert all(torch.equal(d[n].double(), t[n]) for n in t)                        # the inputs are held exactly
    leaves = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v")}
    o, last = linear_attention_fn(*leaves.values(), torch.zeros(1, L, H).cuda(), scale=1.0, initial_state=d["s0"].cuda(), return_last_state=True)
    grads = torch.autograd.grad([o, last], list(leaves.values()), [d["do"].cuda(), d["ds"].cuda()])
    got = dict(zip(("out", "dq", "dk", "dv"), (o.detach(), *grads)))[KINDS[kind]][0].cpu()
    assert torch.equal(got, want.to(dtype)), f"{int((got != want.to(dtype)).sum())} of {got.numel()} differ, by up to {float((got.double() - want).abs()[want == 0].max())} where 0 is exact"
