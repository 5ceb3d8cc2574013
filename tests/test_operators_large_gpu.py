"""Linear attention, single tokens, the norms around a block and gradient clipping on tensors of more than 2^31 elements (and, bytes counted, past
2^32): their last rows against a call on a copy of those rows."""
import pytest
import torch

from mamba_unet_amd import clip_grad_norm, linear_attention_fn, linear_attention_step, norm_gate_residual

pytestmark = pytest.mark.gpu
BIG = (1 << 31) + (1 << 24)


def noise(*shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(len(shape) + shape[0] % 97)
    return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)


@pytest.fixture(autouse=True)
def enough_memory():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free GPU memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("packed", [False, True])
def test_attention_behind_two_to_the_31(packed):
    """With decays of exp(-1) a token, what lies 1024 tokens back weighs exp(-1024) = 0: both calls see the same numbers."""
    H, dv, dk, m = 64, 128, 16, 2048
    L = (BIG // (H * dv)) // 64 * 64
    q, k, v, g = noise(1, L, 1, dk), noise(1, L, 1, dk), noise(1, L, H, dv), torch.full((1, L, H), -1.0, device="cuda")
    do = torch.zeros_like(v)
    do[:, -256:] = noise(1, 256, H, dv)
    res = []
    for at in (0, L - m):
        t = [x[:, at:].detach().requires_grad_() for x in (q, k, v, g)]
        n = t[0].shape[1]
        cu = torch.tensor([0, n - 1500, n], device="cuda", dtype=torch.int32) if packed else None
        out = linear_attention_fn(*t, cu_seqlens=cu)
        grads = torch.autograd.grad(out, t, do[:, at:])
        res.append([x[0, -1024:].float() for x in (out.detach(), *grads)])
        if at == 0:
            assert not grads[2][0, 5000].any() and torch.isfinite(out[0, L // 2:L // 2 + 64]).all()
        del out, grads, t
    # the same terms in sums over other segments: fp32 sums differ by 300 roundings of 2^-24 of the largest value, a bf16 result by a step (2^-7) of itself
    for a, b in zip(*res):
        assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 300 * 2.0 ** -24 * b.abs().max()).all())
    assert res[0][3].abs().max() > 0


def test_token_in_a_pool_behind_two_to_the_31():
    H, dk, dv = 16, 64, 64
    slots = BIG // (H * dk * dv) + 2
    pool = torch.zeros(slots, H, dk, dv, device="cuda")
    idx = torch.tensor([slots - 1, 0, slots - 2], device="cuda")
    pool[idx] = noise(3, H, dk, dv, dtype=torch.float32)
    small = pool[idx].clone()
    q, k, v, g = noise(3, H, dk), noise(3, H, dk), noise(3, H, dv), -noise(3, H, dtype=torch.float32).abs()
    a = linear_attention_step(pool, q, k, v, g, state_indices=idx)
    b = linear_attention_step(small, q, k, v, g)
    assert torch.equal(a, b) and torch.equal(pool[idx], small) and not pool[1:slots - 2].any()


def test_norms_behind_two_to_the_31():
    D = 4096
    rows, m = BIG // D, 512
    x, y = noise(rows, D), noise(rows, D)
    w1, w2 = 1 + 0.1 * noise(D, dtype=torch.float32), 1 + 0.1 * noise(D, dtype=torch.float32)
    gx = torch.zeros_like(x)
    gx[-m:] = noise(m, D)
    res = []
    for at in (0, rows - m):
        t = [s[at:].detach().requires_grad_() for s in (x, y)] + [w.detach().requires_grad_() for w in (w1, w2)]
        xo, h = norm_gate_residual(t[0], t[1], t[2], t[3], rms=True)
        grads = torch.autograd.grad((xo, h), t, (gx[at:], gx[at:]))
        res.append([s[-m:] for s in (xo.detach(), h.detach(), grads[0], grads[1])] + [s.double() for s in grads[2:]])
        del xo, h, grads, t
    for a, b in zip(res[0][:4], res[1][:4]):
        assert torch.equal(a, b)
    for a, b in zip(res[0][4:], res[1][4:]):                       # sums of m terms in another order
        assert bool(((a - b).abs() <= m * 2.0 ** -24 * b.abs().max()).all())


def test_clip_behind_two_to_the_31():
    g = torch.full((BIG,), 2.0, device="cuda", dtype=torch.bfloat16)
    n = clip_grad_norm([g], 2.0 * BIG ** 0.5 / 8)
    assert abs(float(n) - 2.0 * BIG ** 0.5) <= 2.0 ** -23 * 2.0 * BIG ** 0.5
    assert bool((g[-1000:] == 0.25).all()) and bool((g[:1000] == 0.25).all()) and bool((g[1 << 31:] == 0.25).all())
