"""clip_grad_norm on gradients with gaps (slices of a wider tensor): the same one twice, or one inside another, is refused as dense ones are; neighbours are clipped."""
import pytest
import torch

from mamba_unet_amd import clip_grad_norm

pytestmark = pytest.mark.gpu


def test_slices_that_share_memory_are_refused():
    w = torch.randn(10, 16).cuda()
    keep = w.clone()
    pairs = [(w[:, 3:9], w[:, 3:9]), (w, w[:, 3:9]), (w[:, 3:9], w), (w[:, 3:9], w[2:, 5:7]), (w[4:, 5:7], w[:, 3:9]), (w[:, 3:9], w[5, 4:6]), (w.t()[3:9], w[:, 8:])]
    for a, b in pairs:
        with pytest.raises(ValueError, match="shares memory"):
            clip_grad_norm([a, b], 0.1)
        assert torch.equal(w, keep)


def test_neighbouring_slices_are_clipped_together():
    w = torch.randn(10, 16).cuda()
    keep, parts = w.cpu().double(), [w[:, :3], w[:, 3:9], w[:7, 9:], w[8, 9:], w[9, 9:12]]
    n = torch.cat([p.flatten() for p in parts]).cpu().double().norm()
    got = clip_grad_norm(parts, 0.1)
    assert abs(float(got) - float(n)) <= 2.0 ** -23 * float(n)
    want = keep * (0.1 / (n + 1e-6))
    want[7, 9:], want[9, 12:] = keep[7, 9:], keep[9, 12:]
    # the factor's rounding and the product's
    assert bool(((w.cpu().double() - want).abs() <= 5 * 2.0 ** -24 * want.abs()).all())
