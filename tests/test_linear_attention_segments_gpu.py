"""Sequences cut into segments against the same sequences in one walk, forward and backward, through the C entry points (where the caller says how many
segments there are): contributions, joins and walks from a segment's state against the plain walk.

Both sides carry the roundings that tests/test_linear_attention_gpu.py counts (steps * 2^-24 of the sum of the terms' magnitudes, half a step of the output's type), so
they differ by at most twice that; the decays' gradients as tests/test_linear_attention_decay.py counts."""
import ctypes

import pytest
import torch

import test_linear_attention_decay as decay
from mamba_unet_amd import _lib
from test_linear_attention_gpu import HALF, U, make, reference, steps_of

pytestmark = pytest.mark.gpu


def run(t, lens, packed, plan, scale):
    lib = _lib.load()
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    rows, L, G, dk = d["q"].shape
    H, dv = d["v"].shape[2:]
    N, dtype = len(lens), d["q"].dtype
    code = 1 if dtype == torch.bfloat16 else 0
    nseg, segc = plan >> 32, plan & 0xffffffff
    C = lib.ss2d_linattn_chunk(code, dk, dv)
    new = lambda *s, dtype=torch.float32: torch.full(s, float("nan"), device="cuda", dtype=dtype)  # noqa: E731
    walks = N if nseg == 1 else L // (segc * C) + N if packed else N * nseg
    chunks = L // C + N if packed else N * -(-L // C)
    cu = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda() if packed else None
    b = {"out": new(rows, L, H, dv, dtype=dtype), "last": new(N, H, dk, dv), "dq": new(rows, L, G, dk, dtype=dtype), "dk": new(rows, L, G, dk, dtype=dtype),
         "dv": new(rows, L, H, dv, dtype=dtype), "dg": new(rows, L, H), "ds0": new(N, H, dk, dv)}
    states, seg, segd = new(chunks, H, lib.ss2d_linattn_state_floats(code, dk, dv)), new(walks, H, dk, dv), new(walks, H, dtype=torch.float64)
    heads = [new(rows, L, H, dk) for _ in range(2)] if H > G else [None, None]
    st = (ctypes.c_longlong * 12)(*[x.stride(i) for x in (d["q"], d["k"], d["v"]) for i in range(3)], *d["g"].stride())
    p = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    sizes = (N, L, H, G, dk, dv, scale, nseg, segc, stream)
    _lib.check(lib.ss2d_linattn_fwd(code, p(d["q"]), p(d["k"]), p(d["v"]), p(d["g"]), st, p(cu), p(d["s0"]), p(b["out"]), p(b["last"]), p(states), p(seg), p(segd),
                                    *sizes), "fwd")
    _lib.check(lib.ss2d_linattn_bwd(code, p(d["q"]), p(d["k"]), p(d["v"]), p(d["g"]), st, p(cu), p(d["do"]), p(d["ds"]), p(states), p(b["dq"]), p(b["dk"]), p(b["dv"]),
                                    p(b["dg"]), p(b["ds0"]), p(heads[0]), p(heads[1]), p(seg), p(segd), *sizes), "bwd")
    torch.cuda.synchronize()
    return {n: x.cpu() for n, x in b.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("packed", [False, True], ids=["batch", "packed"])
@pytest.mark.parametrize("H,G,dk,dv", [(2, 1, 64, 64), (2, 2, 16, 64), (1, 1, 128, 128), (2, 1, 33, 100)])
def test_segments_equal_one_walk(H, G, dk, dv, packed, dtype):
    lens = [1100, 0, 3, 700, 64] if packed else [1300]
    t = make(lens, packed, H, G, dk, dv, dtype, seed=3, span=0.05)
    scale = dk ** -0.5
    lib = _lib.load()
    code = 1 if dtype == torch.bfloat16 else 0
    plans = [lib.ss2d_linattn_segments(code, sum(lens), max(lens), H, dk, dv, back) for back in (0, 1)]
    assert all(plan >> 32 > 1 for plan in plans)                  # what the operator does with this call
    one = run(t, lens, packed, 1 << 32 | 1, scale)
    want, size = reference(t, lens, packed, scale), reference(t, lens, packed, scale, absolute=True)
    a = {n: x if n == "g" or x is None else x.abs() for n, x in t.items()}
    size["dg"] = decay.gradient(a, lens, packed, scale) * (decay.roundings(t, lens, dk, dv) / steps_of(lens, dk, dv))
    for plan in {*plans, 3 << 32 | -(-max(lens) // 32 // 3)}:
        got = run(t, lens, packed, plan, scale)
        for n, x in got.items():
            assert torch.isfinite(x).all(), n
            lim = HALF[x.dtype] * want[n].abs() + steps_of(lens, dk, dv) * U * size[n] + 1e-30
            for y in (x, one[n]):
                assert bool(((y.double() - want[n]).abs() <= lim).all()), n
            assert bool(((x.double() - one[n].double()).abs() <= 2 * lim).all()), n
