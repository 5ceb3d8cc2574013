"""What the linear-attention, block-norm and clipping operators refuse, without a GPU: CPU tensors in Python, bad arguments at the C boundary
(checked on the host before any launch)."""
import array
import ctypes

import pytest
import torch


def test_cpu_tensors_are_rejected():
    from mamba_unet_amd import clip_grad_norm, linear_attention_fn, linear_attention_step, norm_gate_residual
    q, v = torch.zeros(1, 4, 2, 16), torch.zeros(1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_attention_fn(q, q, v, torch.zeros(2))
    with pytest.raises(RuntimeError, match="GPU"):
        linear_attention_step(torch.zeros(1, 2, 16, 16), q[:, 0], q[:, 0], v[:, 0], torch.zeros(2))
    with pytest.raises(RuntimeError, match="GPU"):
        norm_gate_residual(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), torch.ones(8))
    with pytest.raises(RuntimeError, match="GPU"):
        clip_grad_norm([torch.zeros(4)], 1.0)


def _fwd(lib, **kw):
    a = dict(dtype=0, q=16, k=16, v=16, g=16, st=(ctypes.c_longlong * 12)(*[128] * 12), cu=None, s0=None, out=16, last=None, chunks=None, ws=None, wd=None, N=1, L=8,
             H=2, G=2, dk=16, dv=16, nseg=1, segc=1)
    a.update(kw)
    return lib.ss2d_linattn_fwd(a["dtype"], a["q"], a["k"], a["v"], a["g"], a["st"], a["cu"], a["s0"], a["out"], a["last"], a["chunks"], a["ws"], a["wd"], a["N"],
                                a["L"], a["H"], a["G"], a["dk"], a["dv"], 1.0, a["nseg"], a["segc"], None)


@pytest.mark.parametrize("kw,rc,word", [(dict(dtype=3), -1, b"dtype"), (dict(q=None), -2, b"null"), (dict(st=None), -2, b"null"), (dict(out=None), -2, b"null"),
                                        (dict(N=0), -3, b"size"), (dict(L=0), -3, b"size"), (dict(L=1 << 31), -3, b"size"), (dict(nseg=0), -3, b"size"),
                                        (dict(H=3), -4, b"multiple"), (dict(dk=129), -5, b"128"), (dict(dv=0), -5, b"128"),
                                        (dict(N=1 << 30, H=8, G=8), -6, b"many"), (dict(nseg=2), -2, b"workspace"),
                                        (dict(st=(ctypes.c_longlong * 12)(*[15] * 12)), -4, b"strides"),
                                        (dict(st=(ctypes.c_longlong * 12)(*[1 << 22] * 12)), -4, b"strides")])
def test_linattn_fwd_refuses(kw, rc, word):
    from mamba_unet_amd import _lib
    lib = _lib.load()
    assert _fwd(lib, **kw) == rc and word in lib.ss2d_last_error()


def test_linattn_bwd_and_step_refuse():
    from mamba_unet_amd import _lib
    lib = _lib.load()
    st = (ctypes.c_longlong * 12)(*[128] * 12)
    bwd = lambda dout=16, H=2, heads=None: lib.ss2d_linattn_bwd(0, 16, 16, 16, 16, st, None, dout, None, 16, 16, 16, 16, 16, None, heads, heads, None, None,  # noqa: E731
                                                                1, 8, H, 2, 16, 16, 1.0, 1, 1, None)
    assert bwd(dout=None) == -2 and bwd(H=4) == -2 and b"shared key heads" in lib.ss2d_last_error()
    step = lambda dtype=0, B=1, G=1, dk=16, pool=4, stride=512, slots=None: lib.ss2d_linattn_step(dtype, 16, 16, 16, 16, 16, st, slots, 0, 16, pool, stride, B, 2,  # noqa: E731
                                                                                                 G, dk, 16, 1.0, None)
    assert step(dtype=2) == -1 and step(B=0) == -3 and step(G=3) == -4 and step(dk=200) == -5
    assert step(stride=511) == -4 and b"overlap" in lib.ss2d_last_error()
    assert step(B=5) == -3 and b"states" in lib.ss2d_last_error()
    assert step(B=1 << 28, slots=16) == -6


def test_block_norm_refuses():
    from mamba_unet_amd import _lib
    lib = _lib.load()
    fwd = lambda rt=0, io=0, x=16, drop=None, rps=0, rows=4, D=64, ld=64: lib.ss2d_block_norm_fwd(rt, io, x, 16, None, 16, None, 16, None, None, drop, rps, 16, 16,  # noqa: E731
                                                                                                 None, rows, D, ld, ld, ld, 1e-5, 0, None)
    assert fwd(rt=2) == -1 and fwd(io=-1) == -1 and fwd(x=None) == -2 and fwd(rows=0) == -3 and fwd(D=8193, ld=8193) == -4 and fwd(ld=63) == -4
    assert fwd(drop=16, rps=0) == -3 and fwd(drop=16, rps=5) == -3
    assert lib.ss2d_block_norm_bwd(0, 0, 16, 16, 16, 16, 16, 16, None, 16, None, None, 0, 16, 16, 16, None, 16, 16, 4, 64, 64, 64, 64, 0, None) == -2


def test_grad_clip_refuses():
    from mamba_unet_amd import _lib
    lib = _lib.load()

    def clip(ptrs, sizes, kinds=None, max_norm=1.0, nbytes=1 << 20):
        p, s = array.array("Q", ptrs), array.array("q", sizes)
        return lib.ss2d_grad_clip(kinds or bytes(len(ptrs)), p.buffer_info()[0], s.buffer_info()[0], len(ptrs), 0, max_norm, 1, 16, 16, nbytes, None)
    assert clip([4096, 4096], [4, 4]) == -4 and b"shares memory" in lib.ss2d_last_error()
    assert clip([4096, 8192, 4108], [4, 4, 4]) == -4 and clip([8192, 4096], [4, 1025]) == -4
    assert clip([4097], [4]) == -3 and clip([0], [4]) == -3 and clip([4096], [-1]) == -3 and clip([4098], [4], bytes([1]), -1.0) == -3
    assert clip([4096], [4], max_norm=float("nan")) == -3 and clip([4096], [4], nbytes=8) == -8
    assert lib.ss2d_grad_clip(None, None, None, 0, 0, 1.0, 1, 16, 16, 1 << 20, None) == -2
