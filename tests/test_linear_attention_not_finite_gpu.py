"""A NaN or an infinity in one row of linear_attention_fn's inputs, or of the gradient that comes back, reaches the gradients that depend on that row
and no others (every other value keeps all its bits):

    dq_i: k_j, v_j of j <= i, dout_i          dk_j: q_i, dout_i of i >= j, v_j
    dv_j: q_i, dout_i of i >= j, k_j          dg_t: q_i, dout_i of i >= t, k_j, v_j of j < t

of the columns, a key's (query's) only its own in dq (dk), and a value's gradient only its own in dv."""
import pytest
import torch

from mamba_unet_amd import linear_attention_fn

pytestmark = pytest.mark.gpu
L, HIT = 300, (0, 37, 90, 127, 128, 200, 299)


def inputs(dtype, dk, dv):
    r = torch.Generator().manual_seed(3)
    t = {n: torch.randn(1, L, 2, d, generator=r).to(dtype) for n, d in (("q", dk), ("k", dk), ("v", dv), ("do", dv))}
    t["g"] = -0.2 * torch.rand(1, L, 2, generator=r)
    t["s0"] = torch.randn(1, 2, dk, dv, generator=r)
    return {n: x.cuda() for n, x in t.items()}


def gradients(t):
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    out = linear_attention_fn(*leaves, initial_state=t["s0"])
    return dict(zip(("dq", "dk", "dv", "dg"), torch.autograd.grad(out, leaves, t["do"])))


def reached(name, t, col, dk, dv):
    """what the value in row t, column col of `name` (head 1) may reach: (L, columns) masks"""
    m = {"dq": torch.zeros(L, dk, dtype=torch.bool), "dk": torch.zeros(L, dk, dtype=torch.bool), "dv": torch.zeros(L, dv, dtype=torch.bool),
         "dg": torch.zeros(L, 1, dtype=torch.bool)}
    if name == "q":
        m["dk"][:t + 1, col] = m["dv"][:t + 1] = m["dg"][:t + 1] = True
    elif name == "k":
        m["dq"][t:, col] = m["dv"][t] = m["dg"][t + 1:] = True
    elif name == "v":
        m["dq"][t:] = m["dk"][t] = m["dg"][t + 1:] = True
    else:
        m["dq"][t] = m["dk"][:t + 1] = m["dv"][:t + 1, col] = m["dg"][:t + 1] = True
    return m


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["q", "k", "v", "do"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(16, 64), (64, 64), (128, 64), (64, 100), (128, 128), (33, 7)])
def test_only_dependent_gradients_are_reached(dk, dv, dtype, name, bad):
    t = inputs(dtype, dk, dv)
    clean = gradients(t)
    for at in HIT:
        col = 3 + at % 4
        x = t[name].clone()
        x[0, at, 1, col] = bad
        got = gradients({**t, name: x})
        mask = {n: m.cuda() for n, m in reached(name, at, col, dk, dv).items()}
        for n, g in got.items():
            a, b = (v[0].reshape(L, 2, -1) for v in (g, clean[n]))
            assert torch.equal(a[:, 0], b[:, 0]), (n, at)
            wrong = (a[:, 1] != b[:, 1]) & ~mask[n]                      # (NaN differs from everything)
            assert not wrong.any(), f"{name}[{at}] reaches {n} of rows {wrong.any(1).nonzero().flatten().tolist()}"
        if bad != bad:
            for n, m in mask.items():
                assert torch.isnan(got[n][0].reshape(L, 2, -1)[:, 1][m]).all(), f"{name}[{at}] is lost in {n}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(16, 64), (64, 64), (128, 64), (128, 128)])
def test_an_infinity_keeps_its_sign_where_it_is_alone(dk, dv, dtype):
    """dq_i[c] = scale sum_j w_ij (do_i . v_j) k_j[c]: with one infinite k the sum is the infinity with the sign of its weight."""
    t = inputs(dtype, dk, dv)
    t["v"], t["do"], t["q"] = t["v"].abs() + 0.5, t["do"].abs() + 0.5, t["q"].abs() + 0.5
    for name, grad, rows in (("k", "dq", slice(90, L)), ("q", "dk", slice(0, 91)), ("do", "dv", slice(0, 91))):
        use = dict(t)
        if name == "do":
            use["k"] = t["k"].abs() + 0.5                                # weights q . k > 0
        x = use[name].clone()
        x[0, 90, 1, 5] = -float("inf")
        got = gradients({**use, name: x})[grad][0, rows, 1, 5]
        inside = got[:128 - 90] if name == "k" else got[64:]             # its own chunk: behind it, states carry NaN
        assert bool((inside == -float("inf")).all())
