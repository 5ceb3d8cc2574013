"""clip_grad_norm against its formula in 64 bits.  The norm is one rounding of a 64-bit sum (2^-23 covers the final conversion and the square root); a
scaled gradient carries the factor's rounding, the product's and, in bf16, half a step of the type (2^-8)."""
import math

import pytest
import torch

from mamba_unet_amd import clip_grad_norm

pytestmark = pytest.mark.gpu


def tensors(sizes, dtype, seed=0, scale=1.0):
    r = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=r) * scale).to(dtype) for s in sizes]


def expect(ts, max_norm, inf=False):
    flat = torch.cat([t.double().flatten() for t in ts]) if ts else torch.zeros(1)
    n = float(flat.abs().max()) if inf else float(flat.norm())
    f = max_norm / (n + 1e-6)
    return n, [t.double() * f if not f >= 1 else t.double() for t in ts], f


def check(ts, max_norm, inf=False):
    n, want, f = expect(ts, max_norm, inf)
    gpu = [t.cuda() for t in ts]
    got = clip_grad_norm(gpu, max_norm, float("inf") if inf else 2.0)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - n) <= 2.0 ** -23 * n
    for g, w, t in zip(gpu, want, ts):
        if f >= 1:
            assert torch.equal(g.cpu(), t)
        else:
            half = 2.0 ** -8 if t.dtype == torch.bfloat16 else 2.0 ** -24
            assert bool(((g.cpu().double() - w).abs() <= (half + 4 * 2.0 ** -24) * w.abs() + 1e-44).all())


SIZES = [[1], [3, 1, 7], [16384], [16385, 16383], [(5, 7), (64, 33), 0, 1], [100003, 5, 70000], [11] * 500]


@pytest.mark.parametrize("inf", [False, True], ids=["two", "inf"])
@pytest.mark.parametrize("max_norm", [0.0, 0.3, 1e6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("sizes", SIZES, ids=[str(i) for i in range(len(SIZES))])
def test_norm_and_scaled_gradients(sizes, dtype, max_norm, inf):
    check(tensors(sizes, dtype), max_norm, inf)


def test_mixed_types_and_many_tensors():
    check(tensors([100, 200, 300], torch.float32) + tensors([5, 5000], torch.bfloat16) + tensors([17] * 600, torch.float32, 3), 0.7)


def test_pieces_of_one_buffer_at_any_offset():
    for dtype in (torch.float32, torch.bfloat16):
        sizes = [1, 2, 3, 40001, 5, 17000, 33, 8]
        flat = tensors([sum(sizes) + 2], dtype)[0]
        gpu = flat.cuda()
        n, want, _ = expect([flat[1:-1]], 0.5)
        got = clip_grad_norm(gpu[1:-1].split(sizes), 0.5)
        assert abs(float(got) - n) <= 2.0 ** -23 * n
        assert gpu[0].cpu() == flat[0] and gpu[-1].cpu() == flat[-1]
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert bool(((gpu[1:-1].cpu().double() - want[0]).abs() <= (half + 4 * 2.0 ** -24) * want[0].abs()).all())


def test_other_layouts():
    """Channels-last and transposed gradients are scaled where they are; a gradient with gaps leaves the gaps alone."""
    base = torch.randn(6, 8, 5, 3)
    cl = base.cuda().contiguous(memory_format=torch.channels_last)
    tr = torch.randn(30, 20).cuda().t()
    wide = torch.randn(10, 16).cuda()
    keep = wide.clone()
    want = [t.cpu().clone() for t in (cl, tr, wide[:, 3:9])]
    n, exp, _ = expect(want, 0.1)
    got = clip_grad_norm([cl, tr, wide[:, 3:9]], 0.1)
    assert abs(float(got) - n) <= 2.0 ** -23 * n
    for g, w in zip((cl, tr, wide[:, 3:9]), exp):
        assert bool(((g.cpu().double() - w).abs() <= 5 * 2.0 ** -24 * w.abs()).all())
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 9:], keep[:, 9:])


def test_large_values_do_not_overflow_and_non_finite_ones_spread():
    g = [torch.full((1000,), 1e30).cuda(), torch.full((7,), -2e30).cuda()]
    n = math.sqrt(1000 * 1e60 + 7 * 4e60)
    assert abs(float(clip_grad_norm(g, 1.0)) - n) <= 2.0 ** -22 * n and abs(float(g[0][0]) - 1e30 / n) <= 1e-6
    for bad in (float("nan"), float("inf")):
        for inf in (2.0, float("inf")):
            g = [torch.ones(5000).cuda(), torch.ones(40, dtype=torch.bfloat16).cuda()]
            g[0][4321] = bad
            ref = [t.cpu().clone() for t in g]
            got = clip_grad_norm(g, 1.0, inf)
            want = torch.nn.utils.clip_grad_norm_([p for p in (torch.nn.Parameter(t) for t in ref) if setattr(p, "grad", p.data) is None], 1.0, inf)
            assert torch.equal(got.cpu().isnan(), want.float().isnan()) and torch.equal(got.cpu().isinf(), want.float().isinf())
            for a, b in zip(g, ref):
                assert torch.equal(a.cpu().isnan(), b.isnan())


def test_parameters_and_measuring_only():
    p = [torch.nn.Parameter(torch.randn(4, 5).cuda()) for _ in range(3)]
    p[0].grad, p[2].grad = torch.full((4, 5), 3.0).cuda(), torch.full((4, 5), 4.0).cuda()
    n = math.sqrt(20 * 25)
    assert abs(float(clip_grad_norm(p, float("inf"))) - n) <= 1e-6 * n and torch.equal(p[0].grad, torch.full((4, 5), 3.0).cuda())
    v = p[0].grad._version
    assert abs(float(clip_grad_norm(iter(p), 1.0)) - n) <= 1e-6 * n and p[1].grad is None and p[0].grad._version > v
    assert abs(float(torch.cat([p[0].grad.flatten(), p[2].grad.flatten()]).norm()) - 1.0) <= 1e-5
    assert float(clip_grad_norm([], 1.0)) == 0.0
    assert float(clip_grad_norm([torch.empty(0).cuda()], 1.0)) == 0.0


def test_leaves_that_are_no_parameters_keep_their_values():
    a, b = (torch.full((6,), x, device="cuda", requires_grad=True) for x in (7.0, 9.0))
    a.grad = torch.full((6,), 2.0, device="cuda")
    n = math.sqrt(24)
    assert abs(float(clip_grad_norm([a, b, None], 1.0)) - n) <= 1e-6 * n
    assert bool((a == 7.0).all()) and bool((b == 9.0).all()) and b.grad is None and abs(float(a.grad.norm()) - 1.0) <= 1e-5
    with pytest.raises(ValueError, match="no leaf"):
        clip_grad_norm([a * 2], 1.0)


def test_refusals():
    a = torch.randn(10).cuda()
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm([a, a], 1.0)
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm([a[:6], a[5:]], 1.0)
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm([a[5:], a[:6]], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm([a], bad)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm([a], 1.0, 1.0)
    with pytest.raises(ValueError, match="fp32 or bf16"):
        clip_grad_norm([a.half()], 1.0)


def test_captured_clip_replays_and_does_not_depend_on_the_run():
    ts = tensors([50000, 3, 1000], torch.float32, 1) + tensors([20001], torch.bfloat16, 2)
    buf = [t.cuda() for t in ts]
    clip_grad_norm(buf, 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(buf, 0.5)
    for seed in range(3):
        new = [t.cuda() for t in tensors([50000, 3, 1000], torch.float32, 5 + seed, 2.0 ** seed) + tensors([20001], torch.bfloat16, 9 + seed)]
        for b, t in zip(buf, new):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = clip_grad_norm(new, 0.5)
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(buf, new))


def test_training_step_clips():
    """supervised_step(max_grad_norm=...) takes the same step as clipping by hand between backward and update, captured as well."""
    from mamba_unet_amd import VSSM
    from mamba_unet_amd.train import GraphedSupervisedStep, ce_dice_loss, make_sgd, poly_lr, set_lr, supervised_step
    r = torch.Generator().manual_seed(3)
    images, labels = torch.randn(2, 3, 32, 32, generator=r).cuda(), torch.randint(0, 4, (2, 32, 32), generator=r).cuda()
    nets = []
    for _ in range(3):
        torch.manual_seed(5)
        nets.append(VSSM(patch_size=4, in_chans=3, num_classes=4, depths=[1, 1, 1, 1], dims=[16, 32, 64, 128], drop_path_rate=0.0).cuda().train())
    flat = lambda n: torch.cat([p.detach().flatten() for p in n.parameters()])  # noqa: E731
    start = flat(nets[0])
    opts = [make_sgd(n.parameters(), tensor_lr_device="cuda") for n in nets]
    graphed = GraphedSupervisedStep(nets[2], opts[2], images, labels, 4, 100, warmup=2, max_grad_norm=0.05)     # two eager steps, then the capture
    for it in range(3):
        supervised_step(nets[0], opts[0], images, labels, 4, it, 100, max_grad_norm=0.05)
        opts[1].zero_grad()
        ce, dice = ce_dice_loss(nets[1](images), labels, 4)
        (0.5 * (dice + ce)).backward()
        assert float(torch.nn.utils.clip_grad_norm_(nets[1].parameters(), 0.05)) > 0.5
        opts[1].step()
        set_lr(opts[1], poly_lr(0.01, it, 100))
        if it == 2:
            graphed(images, labels, it)
        if it:
            moved = float((flat(nets[0]) - start).norm())
            # the backward's float atomics change gradients in their last digits (1e-5 of them); a step without the clip would be 10 times as long
            for other in nets[1:]:
                assert float((flat(nets[0]) - flat(other)).norm()) <= 1e-2 * moved


def test_cross_supervised_step_clips_each_network():
    import copy
    from mamba_unet_amd.train import semi_step
    torch.manual_seed(7)
    nets = [torch.nn.Conv2d(1, 4, 3, padding=1).cuda() for _ in range(2)]
    images, labels = torch.randn(4, 1, 32, 32, device="cuda"), torch.randint(0, 4, (4, 32, 32), device="cuda")
    grads = []
    for max_norm in (None, 0.02):
        two = [copy.deepcopy(n) for n in nets]
        opts = [torch.optim.SGD(n.parameters(), lr=0.5) for n in two]
        semi_step(*two, *opts, images, labels, 2, 4, 0, 30000, 0.1, max_grad_norm=max_norm)
        grads.append([[p.grad.double() for p in n.parameters()] for n in two])
    for plain, clipped in zip(*grads):
        norm = torch.stack([g.norm() for g in plain]).norm()
        assert norm > 0.02
        for a, b in zip(plain, clipped):      # the two runs' gradients come from the same kernels; a factor and a product: 2 roundings, the norm's own half step
            assert float((b - a * (0.02 / (norm + 1e-6))).abs().max()) <= 3 * 2.0 ** -24 * float(a.abs().max()) + 1e-12
