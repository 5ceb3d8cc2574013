"""Linear attention with a decay for each head: the matrix-state neighbour of the selective scan.

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        o_t = scale * S_t^T q_t        (S: dk x dv per sequence and head, fp32)

`linear_attention_fn` runs whole sequences (chunked, forward and backward), `linear_attention_step` one new token for each of
many requests whose states lie in a pool.  Both run on the HIP kernels of libss2d_hip.so; CPU tensors are rejected."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ss2d_ops import colsum

_F32, _BF16 = 0, 1          # include/ss2d.h: SS2D_DTYPE_F32 / SS2D_DTYPE_BF16
_MAX_DIM = 128


def _operand(t, io):
    """t in the storage type, its last axis dense and, where the head size allows 16-byte accesses, everything aligned for them
    (a slice of a fused projection is used in place; a view at an odd offset is copied)."""
    if t.dtype != io:
        t = t.to(io)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.contiguous()
    if t.shape[-1] % 8 == 0 and (t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:-1])):
        return t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _check(q, k, v, log_decay, initial_state, cu_seqlens):
    for name, t in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("initial_state", initial_state), ("cu_seqlens", cu_seqlens)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"linear_attention_fn: `{name}` must be a GPU tensor (no CPU path in mamba_unet_amd)")
        if t.device != q.device:
            raise ValueError(f"linear_attention_fn: `{name}` is on {t.device}, q on {q.device}")
        if name != "cu_seqlens" and not t.is_floating_point():
            raise ValueError(f"linear_attention_fn: `{name}` must be a floating-point tensor, got {t.dtype}")
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


def _strides(q, k, v, g):
    """The host array of twelve strides (batch, token, head of q, k, v, g); a decay for each head only has stride 0 over tokens."""
    gs = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return (ctypes.c_longlong * 12)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *gs)


def _segments(lib, dev, code, N, tokens, H, longest, dk, dv, backward):
    """(segments, chunks a segment, state scratch, decay scratch)"""
    C = lib.ss2d_linattn_chunk(code, dk, dv)
    segc = lib.ss2d_linattn_segment_chunks(code, tokens, longest, H, dk, dv, backward)
    nseg = max(1, -(-(-(-longest // C)) // segc))
    if nseg == 1:
        return 1, segc, None, None
    return (nseg, segc, torch.empty((N, H, nseg, dk, dv), device=dev, dtype=torch.float32),
            torch.empty((N, H, nseg), device=dev, dtype=torch.float64))


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
    code = _BF16 if io == torch.bfloat16 else _F32
    chunks = None
    if want_chunks:
        C = lib.ss2d_linattn_chunk(code, dk, dv)
        slots = N * -(-L // C) if cu is None else L // C + N
        chunks = torch.empty((slots, H, lib.ss2d_linattn_state_floats(code, dk, dv)), device=dev, dtype=torch.float32)
    nseg, segc, ws, wd = _segments(lib, dev, code, N, B * L, H, longest, dk, dv, 0)
    p = _lib.ptr
    with _lib.on_device(dev):
        rc = lib.ss2d_linattn_fwd(code, p(q), p(k), p(v), p(g), _strides(q, k, v, g), p(cu), p(s0), p(out), p(last),
                                  p(chunks), p(ws), p(wd), N, L, H, G, dk, dv, scale, nseg, segc, _lib.stream())
    _lib.check(rc, "ss2d_linattn_fwd")
    return out, last, chunks


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, cu_seqlens, scale, dims, longest, want_last):
        io = torch.bfloat16 if q.dtype == k.dtype == v.dtype == torch.bfloat16 else torch.float32
        q_, k_, v_, g_ = _operand(q, io), _operand(k, io), _operand(v, io), log_decay.float()
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
        go = torch.zeros((B, L, H, dv), device=dev, dtype=io) if dout is None else dout.to(io).contiguous()
        if go.data_ptr() % 16:
            go = go.clone()
        gl = None if dlast is None else dlast.float().contiguous()
        dq, dk_ = torch.empty((B, L, G, dk), device=dev, dtype=io), torch.empty((B, L, G, dk), device=dev, dtype=io)
        dv_ = torch.empty((B, L, H, dv), device=dev, dtype=io)
        dg = torch.empty((B, L, H), device=dev, dtype=torch.float32)
        ds0 = torch.empty((N, H, dk, dv), device=dev, dtype=torch.float32) if want_s0 else None
        heads = [torch.empty((B, L, H, dk), device=dev, dtype=torch.float32) for _ in range(2)] if H > G else (None, None)
        lib = _lib.load()
        code = _BF16 if io == torch.bfloat16 else _F32
        nseg, segc, ws, wd = _segments(lib, dev, code, N, B * L, H, longest, dk, dv, 1)
        p = _lib.ptr
        with _lib.on_device(dev):
            rc = lib.ss2d_linattn_bwd(code, p(q), p(k), p(v), p(g), _strides(q, k, v, g), p(cu), p(go), p(gl), p(chunks),
                                      p(dq), p(dk_), p(dv_), p(dg), p(ds0), p(heads[0]), p(heads[1]), p(ws), p(wd), N, L, H, G, dk, dv, scale, nseg,
                                      segc, _lib.stream())
        _lib.check(rc, "ss2d_linattn_bwd")
        if g.dim() == 1:        # a decay for each head: the sum over all tokens (in a fixed order, and right in a replayed graph)
            dg = colsum(dg.view(B * L, H)) if ctx.needs_input_grad[3] else None
        cast = lambda t, d: None if t is None else t.to(d)  # noqa: E731
        return cast(dq, q_dt), cast(dk_, k_dt), cast(dv_, v_dt), cast(dg, g_dt), cast(ds0, s_dt), None, None, None, None, None


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, cu_seqlens=None, max_seqlen=None, return_last_state=False):
    """q, k (b, l, g, dk); v (b, l, h, dv), h a multiple of g: value head j uses key head j // (h // g); log_decay (h,) or
    (b, l, h), normally <= 0 (a decay below -150, -inf included, resets the state); scale defaults to dk ** -0.5; initial_state (n, h, dk, dv).
    Returns out (b, l, h, dv) in v's dtype [, last_state (n, h, dk, dv) fp32, differentiable].  dk, dv <= 128.

    bf16 tensors (all of q, k, v) stay bf16 in memory, everything else is fp32; states, decays and sums are fp32 or wider.
    cu_seqlens (n + 1 int32 offsets, non-decreasing): l tokens of one row (b = 1) hold n sequences, some possibly empty; rows that
    belong to none give zeros.  max_seqlen: an upper estimate of the longest of them (a hint for splitting the work, default l).
    Without cu_seqlens n = b."""
    dims = _check(q, k, v, log_decay, initial_state, cu_seqlens)
    B, L, G, dk, H, dv, N = dims
    scale = float(dk ** -0.5 if scale is None else scale)
    longest = L if cu_seqlens is None or max_seqlen is None else min(L, max(1, int(max_seqlen)))
    if N == 0:
        raise ValueError("linear_attention_fn: empty batch")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        return LinearAttentionFn.apply(q, k, v, log_decay, initial_state, cu_seqlens, scale, dims, longest, bool(return_last_state))
    io = torch.bfloat16 if q.dtype == k.dtype == v.dtype == torch.bfloat16 else torch.float32
    s0 = None if initial_state is None else initial_state.float().contiguous()
    out, last, _ = _forward(_operand(q, io), _operand(k, io), _operand(v, io), log_decay.float(), s0, cu_seqlens, scale, dims, longest,
                            bool(return_last_state), False)
    out = out.to(v.dtype)
    return (out, last) if return_last_state else out


def linear_attention_step(state, q, k, v, log_decay, scale=None, state_indices=None):
    """One new token for each of b requests: S <- exp(log_decay) S + k v^T in place, out = scale * S^T q (b, h, dv) in v's dtype.

    state (slots, h, dk, dv) fp32, its slots dense (a layer's part of a larger pool is fine); q, k (b, g, dk), v (b, h, dv), log_decay (h,) or
    (b, h); scale defaults to dk ** -0.5.  state_indices (b,) int32 or int64: the slot of each request (default: slot = request).  An index outside the
    pool, -1 for instance, marks a padded request: it gives zeros and changes no state.  Requests that name the same slot are applied in
    their order.  States as linear_attention_fn returns them.  For serving: no gradients."""
    for name, t in (("state", state), ("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("state_indices", state_indices)):
        if t is not None:
            if not t.is_cuda:
                raise RuntimeError(f"linear_attention_step: `{name}` must be a GPU tensor (no CPU path in mamba_unet_amd)")
            if t.device != state.device:
                raise ValueError(f"linear_attention_step: `{name}` is on {t.device}, state on {state.device}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (state, q, k, v, log_decay)):
        raise RuntimeError("linear_attention_step updates its state in place and has no gradient: call it under torch.no_grad(), or linear_attention_fn")
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise ValueError(f"q/k must be (b, groups, dk) and equal, v (b, heads, dv): {tuple(q.shape)} / {tuple(k.shape)} / {tuple(v.shape)}")
    B, G, dk = q.shape
    H, dv = v.shape[1:]
    if G == 0 or H == 0 or H % G:
        raise ValueError(f"{H} heads are not a multiple of {G} key heads")
    if not (1 <= dk <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise ValueError(f"dk {dk} and dv {dv} must lie in 1 ... {_MAX_DIM}")
    if state.dtype != torch.float32 or state.dim() != 4 or state.shape[1:] != (H, dk, dv):
        raise ValueError(f"state must be fp32 (slots, {H}, {dk}, {dv}), got {state.dtype} {tuple(state.shape)}")
    pool = state.shape[0]
    n = H * dk * dv
    if pool and not (state[0].is_contiguous() and (pool == 1 or state.stride(0) >= n)):
        raise ValueError("the slots of state must be dense and must not overlap: it is updated in place")
    if log_decay.shape not in ((H,), (B, H)):
        raise ValueError(f"log_decay must be ({H},) or {(B, H)}, got {tuple(log_decay.shape)}")
    if state_indices is None:
        if pool != B:
            raise ValueError(f"{B} requests and {pool} states: give state_indices")
    elif state_indices.shape != (B,) or state_indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"state_indices must be ({B},) int32 or int64, got {state_indices.dtype} {tuple(state_indices.shape)}")
    io = torch.bfloat16 if q.dtype == k.dtype == v.dtype == torch.bfloat16 else torch.float32
    dense = lambda t: t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()  # noqa: E731
    q_, k_, v_, g_ = dense(q.to(io)), dense(k.to(io)), dense(v.to(io)), log_decay.float()
    out = torch.empty((B, H, dv), device=state.device, dtype=io)
    if B == 0 or pool == 0:
        return out.zero_().to(v.dtype)
    idx = None if state_indices is None else state_indices.contiguous()
    strides = (ctypes.c_longlong * 8)(q_.stride(0), q_.stride(1), k_.stride(0), k_.stride(1), v_.stride(0), v_.stride(1),
                                      *((0, g_.stride(0)) if g_.dim() == 1 else g_.stride()))
    lib, p = _lib.load(), _lib.ptr
    with _lib.on_device(state.device):
        rc = lib.ss2d_linattn_step(_BF16 if io == torch.bfloat16 else _F32, p(state), p(q_), p(k_), p(v_), p(g_), strides, p(idx),
                                   int(idx is not None and idx.dtype == torch.int64), p(out), pool, max(n, state.stride(0)), B, H, G, dk, dv,
                                   float(dk ** -0.5 if scale is None else scale), _lib.stream())
    _lib.check(rc, "ss2d_linattn_step")
    torch.autograd.graph.increment_version(state)
    return out if out.dtype == v.dtype else out.to(v.dtype)
