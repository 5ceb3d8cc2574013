"""Gradients of linear_attention_fn and norm_gate_residual when hooks on saved tensors hand the activations back in another layout, as offloading them to
host memory does: the same kernels run on the same values, so every gradient is equal to the last bit."""
import pytest
import torch

from mamba_unet_amd import linear_attention_fn, norm_gate_residual

pytestmark = pytest.mark.gpu


def spread(x):
    """The same values, every axis with a gap behind it (for vectors: every second element)."""
    wide = torch.full([2 * n + 1 for n in x.shape], -7, device=x.device, dtype=x.dtype)
    out = wide[tuple(slice(0, 2 * n, 2) for n in x.shape)]
    out.copy_(x)
    return out


def turned(x):
    """The same values with the axes laid out in the reverse order."""
    order = list(range(x.dim()))[::-1]
    return x.permute(order).contiguous().permute(order)


HOOKS = {"dense": lambda x: x.detach().clone(memory_format=torch.contiguous_format), "spread": lambda x: spread(x.detach()), "turned": lambda x: turned(x.detach())}


def rnd(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def both(call, grads, leaves, hook):
    """gradients without hooks, and with `hook` giving saved tensors back (cu_seqlens, int32, stays as it is)"""
    want = torch.autograd.grad(call(), leaves, grads)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: hook(x) if x.is_floating_point() else x):
        out = call()
    return want, torch.autograd.grad(out, leaves, grads)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
def test_norms_of_slices_of_a_wider_tensor(D, dtype, hook):
    fused = rnd(0, 3, 9, 3 * D, dtype=dtype).requires_grad_()
    w1, b1, a, w2, b2 = (rnd(i, D).requires_grad_() for i in range(1, 6))
    drop = torch.tensor([0.0, 1.5, 1.5]).cuda()

    def call():
        x, y, z = fused.split(D, -1)
        return norm_gate_residual(x, y, w1, w2, post_bias=b1, pre_bias=b2, z=z, res_scale=a, drop_scale=drop)

    want, got = both(call, [rnd(6, 3, 9, D, dtype=dtype), rnd(7, 3, 9, D, dtype=dtype)], [fused, w1, b1, a, w2, b2], HOOKS[hook])
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (33, 24)])
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("packed", [False, True])
def test_attention_on_views_of_a_fused_projection(dk, dv, decay, packed, dtype, hook):
    H, G, L, B = 4, 2, 150, 1 if packed else 2
    fused = rnd(0, B, L, 2 * G * dk + H * dv, dtype=dtype).requires_grad_()
    g = (-rnd(1, H).abs() if decay == "head" else -rnd(1, B, L, H).abs()).requires_grad_()
    cu = torch.tensor([0, 70, 70, 150], dtype=torch.int32).cuda() if packed else None
    s0 = rnd(2, 3 if packed else B, H, dk, dv).requires_grad_()

    def call():
        q, k, v = fused.split([G * dk, G * dk, H * dv], -1)
        return linear_attention_fn(q.unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv)), g, initial_state=s0, cu_seqlens=cu,
                                   return_last_state=True)

    want, got = both(call, [rnd(3, B, L, H, dv, dtype=dtype), rnd(4, *s0.shape)], [fused, g, s0], HOOKS[hook])
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_offloaded_to_host_memory():
    D = 64
    fused, w = rnd(0, 4, 50, 3 * D).requires_grad_(), rnd(1, D).requires_grad_()

    def call():
        x, y, z = fused.split(D, -1)
        x, h = norm_gate_residual(x, y, w, w, z=z, rms=True)
        q, k, v = (t.unflatten(-1, (4, 16)) for t in (h, y, z))
        return linear_attention_fn(q, k, v, -0.1 * torch.ones(4, device="cuda")).sum() + x.sum()

    want = torch.autograd.grad(call(), [fused, w])
    for pinned in (False, True):
        with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
            out = call()
        assert all(torch.equal(x, y) for x, y in zip(want, torch.autograd.grad(out, [fused, w])))


def test_saved_tensors_of_another_shape_or_place_are_refused():
    x, w = rnd(0, 4, 32).requires_grad_(), rnd(1, 32)
    q, g = rnd(2, 1, 20, 2, 16).requires_grad_(), -torch.ones(2, device="cuda")
    calls = (lambda: norm_gate_residual(x, x, w, w)[1], lambda: linear_attention_fn(q, q, q, g))
    for call, leaf in zip(calls, (x, q)):
        for hook, error in ((lambda t: t[:1] if t.dim() else t, ValueError), (lambda t: t.detach().cpu(), RuntimeError)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
                out = call()
            with pytest.raises(error):
                torch.autograd.grad(out.sum(), leaf)


def test_offsets_of_packed_sequences_come_back_with_gaps():
    q, v = rnd(0, 1, 100, 2, 16).requires_grad_(), rnd(1, 1, 100, 4, 24)
    g, cu = -rnd(2, 1, 100, 4).abs(), torch.tensor([0, 30, 30, 100], dtype=torch.int32).cuda()
    call = lambda: linear_attention_fn(q, q, v, g, cu_seqlens=cu).sum()  # noqa: E731
    want, = torch.autograd.grad(call(), q)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: spread(x.detach())):
        out = call()
    assert torch.equal(torch.autograd.grad(out, q)[0], want)
