"""Linear attention with a decay for each head: the matrix-state neighbour of the selective scan.

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        o_t = scale * S_t^T q_t        (S: dk x dv per sequence and head, fp32)

`linear_attention_fn` runs whole sequences (chunked, forward and backward), `linear_attention_step` one new token for each of
many requests whose states lie in a pool.  Both run on the HIP kernels of libss2d_hip.so; CPU tensors are rejected."""
from __future__ import annotations

import struct

import torch

from . import _lib
from .ss2d_ops import _dense16, colsum

_F32, _BF16 = 0, 1          # include/ss2d.h: SS2D_DTYPE_F32 / SS2D_DTYPE_BF16
_MAX_DIM = 128


def _operand(t, io):
    """t in the storage type, its last axis dense and its tokens apart by less than 2^22 elements and not overlapping (an expanded or far-flung view is
    copied; a slice of a fused projection is used in place).  bf16 heads made of 16-byte pieces that begin inside a 32-bit word are copied, too."""
    if t.dtype is not io:
        t = t.to(io)
    n, s = t.shape[-1], t.stride()
    if (n > 1 and s[3] != 1) or not n <= s[1] < 1 << 22 or (n % 8 == 0 and io is torch.bfloat16 and (t.data_ptr() % 4 or (s[0] | s[1] | s[2]) % 2)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _storage(q, k, v):
    return torch.bfloat16 if q.dtype is torch.bfloat16 and k.dtype is torch.bfloat16 and v.dtype is torch.bfloat16 else torch.float32


def _fp32(t):
    return t if t is None or t.dtype is torch.float32 else t.float()


def _check_devices(name, **tensors):
    """Raises for the first tensor that is not on the GPU, or on another one than the first."""
    first = None
    for n, t in tensors.items():
        if t is not None:
            if not t.is_cuda:
                raise RuntimeError(f"{name}: `{n}` must be a GPU tensor (no CPU path in mamba_unet_amd)")
            first = first or (n, t.device)
            if t.device != first[1]:
                raise ValueError(f"{name}: `{n}` is on {t.device}, {first[0]} on {first[1]}")


def _check(q, k, v, log_decay, initial_state, cu_seqlens):
    d = q.get_device()
    if d < 0 or k.get_device() != d or v.get_device() != d or log_decay.get_device() != d or (initial_state is not None and initial_state.get_device() != d) \
            or (cu_seqlens is not None and cu_seqlens.get_device() != d):
        _check_devices("linear_attention_fn", q=q, k=k, v=v, log_decay=log_decay, initial_state=initial_state, cu_seqlens=cu_seqlens)
    if not (q.is_floating_point() and k.is_floating_point() and v.is_floating_point() and log_decay.is_floating_point()) \
            or (initial_state is not None and not initial_state.is_floating_point()):
        raise ValueError("linear_attention_fn: q, k, v, log_decay and initial_state must be floating-point tensors")
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"q/k must be (batch, L, groups, dk) and equal, v (batch, L, heads, dv): {tuple(q.shape)} / {tuple(k.shape)} / {tuple(v.shape)}")
    B, L, G, dk = q.shape
    H, dv = v.shape[2], v.shape[3]
    if G == 0 or H == 0 or H % G:
        raise ValueError(f"{H} heads are not a multiple of {G} key heads")
    if not (1 <= dk <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise ValueError(f"dk {dk} and dv {dv} must lie in 1 ... {_MAX_DIM}")
    if log_decay.shape not in ((H,), (B, L, H)):
        raise ValueError(f"log_decay must be ({H},) or {(B, L, H)}, got {tuple(log_decay.shape)}")
    N = B
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous int32 tensor of at least two offsets")
        if B != 1:
            raise ValueError(f"packed sequences lie in one row: batch must be 1 with cu_seqlens, got {B}")
        N = cu_seqlens.numel() - 1
    if initial_state is not None and initial_state.shape != (N, H, dk, dv):
        raise ValueError(f"initial_state must be {(N, H, dk, dv)}, got {tuple(initial_state.shape)}")
    return B, L, G, dk, H, dv, N


_TWELVE, _EIGHT = struct.Struct("12q").pack, struct.Struct("8q").pack


def _strides(q, k, v, g):
    """The host array of twelve strides (batch, token, head of q, k, v, g); a decay for each head only has stride 0 over tokens."""
    gs = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return _TWELVE(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *gs)


def _segments(lib, dev, code, N, rows, L, H, longest, dk, dv, packed, backward):
    """(segments, chunks a segment, state scratch, decay scratch)"""
    plan = lib.ss2d_linattn_segments(code, rows * L, longest, H, dk, dv, backward)
    nseg, segc = plan >> 32, plan & 0xffffffff
    if nseg == 1:
        return 1, segc, None, None
    slots = L // (segc * lib.ss2d_linattn_chunk(code, dk, dv)) + N if packed else N * nseg
    return (nseg, segc, torch.empty((slots, H, dk, dv), device=dev, dtype=torch.float32), torch.empty((slots, H), device=dev, dtype=torch.float64))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, g, s0, cu, scale, dims, longest, want_last, want_chunks):
    B, L, G, dk, H, dv, N = dims
    io = q.dtype
    dev = q.device
    out = torch.empty((B, L, H, dv), device=dev, dtype=io)
    last = torch.empty((N, H, dk, dv), device=dev, dtype=torch.float32) if want_last else None
    if L == 0:
        if want_last:
            last.zero_() if s0 is None else last.copy_(s0)
        return out, last, None
    lib = _lib.load()
    code = _BF16 if io is torch.bfloat16 else _F32
    chunks = None
    if want_chunks:
        C = lib.ss2d_linattn_chunk(code, dk, dv)
        slots = N * -(-L // C) if cu is None else L // C + N
        chunks = torch.empty((slots, H, lib.ss2d_linattn_state_floats(code, dk, dv)), device=dev, dtype=torch.float32)
    nseg, segc, ws, wd = _segments(lib, dev, code, N, B, L, H, longest, dk, dv, cu is not None, 0)
    args = (code, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), _strides(q, k, v, g), _ptr(cu), _ptr(s0), out.data_ptr(), _ptr(last), _ptr(chunks),
            _ptr(ws), _ptr(wd), N, L, H, G, dk, dv, scale, nseg, segc)
    stream = _lib.stream_of(dev.index)
    if stream is None:
        with torch.cuda.device(dev):
            rc = lib.ss2d_linattn_fwd(*args, _lib.stream())
    else:
        rc = lib.ss2d_linattn_fwd(*args, stream)
    if rc:
        _lib.check(rc, "ss2d_linattn_fwd")
    return out, last, chunks


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, cu_seqlens, scale, dims, longest, want_last):
        io = _storage(q, k, v)
        q_, k_, v_, g_ = _operand(q, io), _operand(k, io), _operand(v, io), _fp32(log_decay)
        s0 = None if initial_state is None else initial_state.float().contiguous()
        ctx.set_materialize_grads(False)
        out, last, chunks = _forward(q_, k_, v_, g_, s0, cu_seqlens, scale, dims, longest, want_last, True)
        ctx.save_for_backward(q_, k_, v_, g_, cu_seqlens, chunks)
        ctx.meta = (dims, longest, scale, io, q.dtype, k.dtype, v.dtype, log_decay.dtype, None if initial_state is None else initial_state.dtype)
        out = out.to(v.dtype)
        return (out, last) if want_last else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlast=None):
        q, k, v, g, cu, chunks = ctx.saved_tensors
        (B, L, G, dk, H, dv, N), longest, scale, io, q_dt, k_dt, v_dt, g_dt, s_dt = ctx.meta
        dev = q.device
        if dout is None and dlast is None:
            return (None,) * 10
        want_s0 = s_dt is not None and ctx.needs_input_grad[4]
        if L == 0:
            z = lambda *sh, dt: torch.zeros(sh, device=dev, dtype=dt)  # noqa: E731
            ds0 = None if not want_s0 else (z(N, H, dk, dv, dt=s_dt) if dlast is None else dlast.to(s_dt))
            return z(B, L, G, dk, dt=q_dt), z(B, L, G, dk, dt=k_dt), z(B, L, H, dv, dt=v_dt), z(*g.shape, dt=g_dt), ds0, None, None, None, None, None
        go = torch.zeros((B, L, H, dv), device=dev, dtype=io) if dout is None else _dense16(dout, io)
        gl = None if dlast is None else _dense16(dlast, torch.float32)
        dq, dk_ = torch.empty((B, L, G, dk), device=dev, dtype=io), torch.empty((B, L, G, dk), device=dev, dtype=io)
        dv_ = torch.empty((B, L, H, dv), device=dev, dtype=io)
        dg = torch.empty((B, L, H), device=dev, dtype=torch.float32)
        ds0 = torch.empty((N, H, dk, dv), device=dev, dtype=torch.float32) if want_s0 else None
        hq, hk = [torch.empty((B, L, H, dk), device=dev, dtype=torch.float32) for _ in range(2)] if H > G else (None, None)
        lib = _lib.load()
        code = _BF16 if io is torch.bfloat16 else _F32
        nseg, segc, ws, wd = _segments(lib, dev, code, N, B, L, H, longest, dk, dv, cu is not None, 1)
        args = (code, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), _strides(q, k, v, g), _ptr(cu), go.data_ptr(), _ptr(gl), chunks.data_ptr(),
                dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(), dg.data_ptr(), _ptr(ds0), _ptr(hq), _ptr(hk), _ptr(ws), _ptr(wd), N, L, H, G, dk, dv, scale, nseg, segc)
        stream = _lib.stream_of(dev.index)
        if stream is None:
            with torch.cuda.device(dev):
                rc = lib.ss2d_linattn_bwd(*args, _lib.stream())
        else:
            rc = lib.ss2d_linattn_bwd(*args, stream)
        if rc:
            _lib.check(rc, "ss2d_linattn_bwd")
        if g.dim() == 1:        # a decay for each head: the sum over all tokens (in a fixed order, and right in a replayed graph)
            dg = colsum(dg.view(B * L, H)) if ctx.needs_input_grad[3] else None
        cast = lambda t, d: t if t is None or t.dtype is d else t.to(d)  # noqa: E731
        return cast(dq, q_dt), cast(dk_, k_dt), cast(dv_, v_dt), cast(dg, g_dt), cast(ds0, s_dt), None, None, None, None, None


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, cu_seqlens=None, max_seqlen=None, return_last_state=False):
    """q, k (b, l, g, dk); v (b, l, h, dv), h a multiple of g: value head j uses key head j // (h // g); log_decay (h,) or
    (b, l, h), normally <= 0 (a decay below -150, -inf included, resets the state); scale defaults to dk ** -0.5; initial_state (n, h, dk, dv).
    Returns out (b, l, h, dv) in v's dtype [, last_state (n, h, dk, dv) fp32, differentiable].  dk, dv <= 128.

    bf16 tensors (all of q, k, v) stay bf16 in memory, everything else is fp32; states, decays and sums are fp32 or wider.
    cu_seqlens (n + 1 int32 offsets, non-decreasing): l tokens of one row (b = 1) hold n sequences, some possibly empty; rows that
    belong to none give zeros.  max_seqlen: an estimate of the longest of them (a hint whether to split any, default l).
    Without cu_seqlens n = b."""
    dims = _check(q, k, v, log_decay, initial_state, cu_seqlens)
    B, L, G, dk, H, dv, N = dims
    scale = float(dk ** -0.5 if scale is None else scale)
    longest = L if cu_seqlens is None or max_seqlen is None else min(L, max(1, int(max_seqlen)))
    if N == 0:
        raise ValueError("linear_attention_fn: empty batch")
    want_last = bool(return_last_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or (initial_state is not None and initial_state.requires_grad)):
        return LinearAttentionFn.apply(q, k, v, log_decay, initial_state, cu_seqlens, scale, dims, longest, want_last)
    io = _storage(q, k, v)
    s0 = None if initial_state is None else _fp32(initial_state).contiguous()
    out, last, _ = _forward(_operand(q, io), _operand(k, io), _operand(v, io), _fp32(log_decay), s0, cu_seqlens, scale, dims, longest, want_last, False)
    if out.dtype is not v.dtype:
        out = out.to(v.dtype)
    return (out, last) if want_last else out


def linear_attention_step(state, q, k, v, log_decay, scale=None, state_indices=None):
    """One new token for each of b requests: S <- exp(log_decay) S + k v^T in place, out = scale * S^T q (b, h, dv) in v's dtype.

    state (slots, h, dk, dv) fp32, its slots dense (a layer's part of a larger pool is fine); q, k (b, g, dk), v (b, h, dv), log_decay (h,) or
    (b, h); scale defaults to dk ** -0.5.  state_indices (b,) int32 or int64: the slot of each request (default: slot = request).  An index outside the
    pool, -1 for instance, marks a padded request: it gives zeros and changes no state.  Requests that name the same slot are applied in
    their order.  States as linear_attention_fn returns them.  For serving: no gradients."""
    d = state.get_device()
    if d < 0 or q.get_device() != d or k.get_device() != d or v.get_device() != d or log_decay.get_device() != d \
            or (state_indices is not None and state_indices.get_device() != d):
        _check_devices("linear_attention_step", state=state, q=q, k=k, v=v, log_decay=log_decay, state_indices=state_indices)
    if torch.is_grad_enabled() and (state.requires_grad or q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad):
        raise RuntimeError("linear_attention_step updates its state in place and has no gradient: call it under torch.no_grad(), or linear_attention_fn")
    qs, vs, ss = q.shape, v.shape, state.shape
    if len(qs) != 3 or k.shape != qs or len(vs) != 3 or vs[0] != qs[0]:
        raise ValueError(f"q/k must be (b, groups, dk) and equal, v (b, heads, dv): {tuple(qs)} / {tuple(k.shape)} / {tuple(vs)}")
    B, G, dk = qs
    _, H, dv = vs
    if G == 0 or H == 0 or H % G:
        raise ValueError(f"{H} heads are not a multiple of {G} key heads")
    if not (1 <= dk <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise ValueError(f"dk {dk} and dv {dv} must lie in 1 ... {_MAX_DIM}")
    if state.dtype is not torch.float32 or len(ss) != 4 or ss[1] != H or ss[2] != dk or ss[3] != dv:
        raise ValueError(f"state must be fp32 (slots, {H}, {dk}, {dv}), got {state.dtype} {tuple(ss)}")
    pool, n = ss[0], H * dk * dv
    pitch, *inner = state.stride()
    if pool and (inner != [dk * dv, dv, 1] and not state[0].is_contiguous() or pool > 1 and pitch < n):
        raise ValueError("the slots of state must be dense and must not overlap: it is updated in place")
    gs = log_decay.shape
    if gs != (H,) and gs != (B, H):
        raise ValueError(f"log_decay must be ({H},) or {(B, H)}, got {tuple(gs)}")
    slots, wide = None, 0
    if state_indices is None:
        if pool != B:
            raise ValueError(f"{B} requests and {pool} states: give state_indices")
    else:
        wide = int(state_indices.dtype is torch.int64)
        if state_indices.shape != (B,) or not (wide or state_indices.dtype is torch.int32):
            raise ValueError(f"state_indices must be ({B},) int32 or int64, got {state_indices.dtype} {tuple(state_indices.shape)}")
        slots = state_indices.contiguous()
    io = _storage(q, k, v)
    q_, k_, v_, g_ = _token(q, io), _token(k, io), _token(v, io), _fp32(log_decay)
    dev = state.device
    out = torch.empty((B, H, dv), device=dev, dtype=io)
    if B == 0 or pool == 0:
        return out.zero_().to(v.dtype)
    strides = _EIGHT(*q_.stride()[:2], *k_.stride()[:2], *v_.stride()[:2], *((0, g_.stride(0)) if len(gs) == 1 else g_.stride()))
    lib = _lib.load()
    args = (_BF16 if io is torch.bfloat16 else _F32, state.data_ptr(), q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), g_.data_ptr(), strides, _ptr(slots), wide,
            out.data_ptr(), pool, max(n, pitch), B, H, G, dk, dv, float(dk ** -0.5 if scale is None else scale))
    stream = _lib.stream_of(d)
    if stream is None:
        with torch.cuda.device(dev):
            rc = lib.ss2d_linattn_step(*args, _lib.stream())
    else:
        rc = lib.ss2d_linattn_step(*args, stream)
    if rc:
        _lib.check(rc, "ss2d_linattn_step")
    if not state.is_inference():                # (tensors made under inference_mode have no version)
        torch._C._increment_version((state,))
    return out if io is v.dtype else out.to(v.dtype)


def _token(t, io):
    """t in the storage type with a dense last axis"""
    if t.dtype is not io:
        t = t.to(io)
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()
