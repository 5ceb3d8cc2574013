"""Forward-mode derivatives (torch.autograd.forward_ad) of the operators whose kernels carry no tangents: a call with a dual tensor raises instead of
returning a result without a tangent.  The check comes before the one for the GPU, so all but the backward's is tested on the CPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from mamba_unet_amd import clip_grad_norm, linear_attention_fn, linear_attention_step, norm_gate_residual


def inputs(dev):
    t = {"q": torch.ones(1, 4, 2, 16), "k": torch.ones(1, 4, 2, 16), "v": torch.ones(1, 4, 2, 16), "log_decay": -torch.ones(2), "initial_state": torch.ones(1, 2, 16, 16)}
    n = {"x": torch.ones(3, 8), "y": torch.ones(3, 8), "post_weight": torch.ones(8), "pre_weight": torch.ones(8), "post_bias": torch.ones(8), "pre_bias": torch.ones(8),
         "z": torch.ones(3, 8), "res_scale": torch.ones(8), "drop_scale": torch.ones(3)}
    s = {"state": torch.ones(1, 2, 16, 16), "q": torch.ones(1, 2, 16), "k": torch.ones(1, 2, 16), "v": torch.ones(1, 2, 16), "log_decay": -torch.ones(1, 2)}
    return [(f, {m: x.to(dev) for m, x in a.items()}) for f, a in ((linear_attention_fn, t), (norm_gate_residual, n), (linear_attention_step, s))]


def raise_for_every_argument(dev):
    for f, args in inputs(dev):
        for name, x in args.items():
            with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(**{**args, name: fwad.make_dual(x, torch.ones_like(x))})
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        clip_grad_norm([torch.ones(3, device=dev), fwad.make_dual(torch.ones(3, device=dev), torch.ones(3, device=dev))][::-1], 1.0)


def test_tangents_are_refused():
    raise_for_every_argument("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu():
    raise_for_every_argument("cuda")
    for f, args in inputs("cuda")[:2]:
        leaf = next(iter(args.values())).requires_grad_()
        out = f(**args)
        out = out if torch.is_tensor(out) else out[0]
        with fwad.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):      # a dual gradient: forward over reverse
                torch.autograd.grad(out, leaf, fwad.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
        assert torch.isfinite(torch.autograd.grad(out, leaf, torch.ones_like(out))[0]).all()
