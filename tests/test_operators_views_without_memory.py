"""Tensors that do not hold their values in memory: the negated view that the imaginary part of a conjugate is, and torch's zero tensors without memory.  As
inputs they are refused (before the check for the GPU, so that the CPU sees it); as gradients that come back they are read for what they stand for."""
import pytest
import torch

from mamba_unet_amd import clip_grad_norm, linear_attention_fn, linear_attention_step, norm_gate_residual


def negated(x):
    """A view with the values of x whose memory holds -x."""
    v = torch.complex(torch.zeros_like(x), -x).conj().imag
    assert v.is_neg() and torch.equal(v.resolve_neg(), x)
    return v


def calls(dev="cpu"):
    r = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=r).to(dev)  # noqa: E731
    attn = {"q": rnd(1, 5, 2, 16), "k": rnd(1, 5, 2, 16), "v": rnd(1, 5, 2, 16), "log_decay": -rnd(2).abs(), "initial_state": rnd(1, 2, 16, 16)}
    norm = {"x": rnd(3, 8), "y": rnd(3, 8), "post_weight": rnd(8), "pre_weight": rnd(8), "z": rnd(3, 8), "res_scale": rnd(8)}
    step = {"state": rnd(1, 2, 16, 16), "q": rnd(1, 2, 16), "k": rnd(1, 2, 16), "v": rnd(1, 2, 16), "log_decay": -rnd(1, 2).abs()}
    return [(linear_attention_fn, attn), (norm_gate_residual, norm), (linear_attention_step, step)]


@pytest.mark.parametrize("kind", ["negated", "no memory"])
def test_inputs_are_refused(kind):
    view = negated if kind == "negated" else lambda x: torch._efficientzerotensor(x.shape)
    for f, args in calls():
        for name, x in args.items():
            with pytest.raises(ValueError, match="negated view"):
                f(**{**args, name: view(x)})
    with pytest.raises(ValueError, match="negated view"):
        clip_grad_norm([view(torch.ones(3))], 1.0)


@pytest.mark.gpu
def test_gradients_are_read_for_what_they_stand_for():
    for f, args in calls("cuda")[:2]:
        leaves = [x.requires_grad_() for x in args.values()]
        out = f(**args)
        out = out if torch.is_tensor(out) else out[0]
        back = lambda g: torch.autograd.grad(out, leaves, g, retain_graph=True, allow_unused=True)  # noqa: E731,B023
        g = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).cuda()
        for a, b in ((negated(g), g), (torch._efficientzerotensor(g.shape, device="cuda"), torch.zeros_like(g))):
            for x, y in zip(back(a), back(b)):
                assert (x is None and y is None) or torch.equal(x, y)
