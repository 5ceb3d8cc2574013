"""Linear attention with a decay for each head: the matrix-state neighbour of the selective scan.

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        o_t = scale * S_t^T q_t        (S: dk x dv per sequence and head, fp32)

`linear_attention_fn` runs whole sequences (chunked, forward and backward), `linear_attention_step` one new token for each of
many requests whose states lie in a pool.  Both run on the HIP kernels of libss2d_hip.so (checks, outputs and autograd: csrc/host_ops.cpp); CPU tensors are
rejected."""
from __future__ import annotations

from . import _lib


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, cu_seqlens=None, max_seqlen=None, return_last_state=False):
    """q, k (b, l, g, dk); v (b, l, h, dv), h a multiple of g: value head j uses key head j // (h // g); log_decay (h,) or
    (b, l, h), normally <= 0 (a decay below -150, -inf included, is a factor of 0: it resets a finite state); scale defaults to dk ** -0.5; initial_state (n, h, dk, dv).
    Returns out (b, l, h, dv) in v's dtype [, last_state (n, h, dk, dv) fp32, differentiable].  dk, dv <= 128.

    bf16 tensors (all of q, k, v) stay bf16 in memory, everything else is fp32: states, weights, decays and sums keep at least 24 bits, also as factors on the
    bf16 matrix units, and results are rounded once.  Gradients once; forward-mode derivatives and differentiating twice raise.
    cu_seqlens (n + 1 int32 offsets, non-decreasing): l tokens of one row (b = 1) hold n sequences, some possibly empty; rows that
    belong to none give zeros.  max_seqlen: an estimate of the longest of them (a hint whether to split any, default l).
    Without cu_seqlens n = b."""
    return _lib.host().attention(q, k, v, log_decay, scale, initial_state, cu_seqlens, max_seqlen, bool(return_last_state))


def linear_attention_step(state, q, k, v, log_decay, scale=None, state_indices=None):
    """One new token for each of b requests: S <- exp(log_decay) S + k v^T in place, out = scale * S^T q (b, h, dv) in v's dtype.

    state (slots, h, dk, dv) fp32, its slots dense (a layer's part of a larger pool is fine); q, k (b, g, dk), v (b, h, dv), log_decay (h,) or
    (b, h); scale defaults to dk ** -0.5.  state_indices (b,) int32 or int64: the slot of each request (default: slot = request).  An index outside the
    pool, -1 for instance, marks a padded request: it gives zeros and changes no state.  Requests that name the same slot are applied in
    their order.  States as linear_attention_fn returns them.  For serving: no gradients."""
    return _lib.host().attention_step(state, q, k, v, log_decay, scale, state_indices)
