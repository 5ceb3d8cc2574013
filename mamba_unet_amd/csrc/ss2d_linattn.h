// Shared pieces of the linear-attention kernels (ss2d_linattn_fwd.hip, ss2d_linattn_bwd.hip): the problem description, the
// walk over a sequence in chunks, the decays of a chunk and the tile loads.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t        (S: dk x dv per sequence and value head, fp32)
//
// With b_i = g_1 + ... + g_i counted from a chunk's start and S the state in front of it
//   o_i   = scale * ( exp(b_i) S^T q_i + sum_{j <= i} exp(b_i - b_j) (q_i . k_j) v_j )
//   S_end = exp(b_C) S + sum_j exp(b_C - b_j) k_j v_j^T
// so a chunk costs four matrix products and one state.  No exponent is positive for g <= 0: decays of any size are safe.
#pragma once
#include "ss2d_common.h"

namespace linattn {

struct Problem {
    const void *q, *k, *v;
    const float *g;
    long long qb, ql, qh, kb, kl, kh, vb, vl, vh, gb, gl, gh;   // element strides: batch, token, head (the last axis is dense)
    const int *cu;                // packed sequences: N + 1 row offsets into one row of `tokens` tokens; null: a batch
    long long tokens;             // tokens of a row (batch: the length of every sequence)
    int N, H, G, dk, dv;
    float scale;
    int nseg, segc;               // segments of a sequence, chunks a segment
    int vec;                      // all rows start on 16-byte boundaries and dk, dv are multiples of 8
};

// A workgroup's sequence: token rows [start, start + len) of batch row `row`.  The offsets of a packed batch come from device
// memory: they are clamped to the row, so no value of theirs can lead outside the tensors.
struct Seq {
    long long start;
    int len, row;
};
__device__ __forceinline__ Seq get_seq(const Problem &p, int n) {
    Seq s;
    if (p.cu) {
        const long long T = p.tokens;
        long long a = p.cu[n], e = p.cu[n + 1];
        a = a < 0 ? 0 : a > T ? T : a;
        e = e < a ? a : e > T ? T : e;
        s.start = a;
        s.len = (int)(e - a);
        s.row = 0;
    } else {
        s.start = 0;
        s.len = (int)p.tokens;
        s.row = n;
    }
    return s;
}
// a sequence's last segment takes whatever is left: the number of segments comes from a hint of the longest sequence
__device__ __forceinline__ int segment_end(const Problem &p, int seg, int nch) {
    const long long e = (long long)(seg + 1) * p.segc;
    return seg + 1 == p.nseg || e > nch ? nch : (int)e;
}
__device__ __forceinline__ int segments_of(const Problem &p, int nch) {
    const int n = (nch + p.segc - 1) / p.segc;
    return n < p.nseg ? n : p.nseg;
}
// slot of a sequence's chunk 0 in the chunk-state buffer: floor(start / C) + n leaves room for every earlier sequence's last,
// partly filled chunk
__device__ __forceinline__ long long chunk_base(const Problem &p, const Seq &s, int n, int C) {
    return p.cu ? s.start / C + n : (long long)n * ((p.tokens + C - 1) / C);
}

// A decay below exp(-150) is 0 in fp32: g is limited there, which keeps -inf and the type's lowest value (a state reset)
// out of the differences b_i - b_j.  NaN passes.
__device__ __forceinline__ float limit_decay(float g) { return g < -150.0f ? -150.0f : g; }

// Inclusive prefix sums of log2(e) * g over the lanes of a wave (C <= 64 tokens), in 64 bits: the sum over a chunk that holds a
// reset is ~200 per reset, and the decays behind the reset must not lose their last bits to it.  A pair's decay is
// exp2((hi_i - hi_j) + (lo_i - lo_j)) with hi + lo = b.
__device__ __forceinline__ double chunk_decay_scan(float g, int lane) {
    double b = (double)g * 1.4426950408889634074;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(b, d, 64);
        if (lane >= d) b += o;
    }
    return b;
}

// rows [0, C) of `src` (row stride ld, D columns, rows >= n read as zero) -> fp32 tile in LDS, PITCH floats a row, columns
// D .. DP-1 zero
template <int C, int DP, int PITCH, int NT, typename IO>
__device__ __forceinline__ void load_tile(float *dst, const IO *src, long long ld, int n, int D, bool vec) {
    constexpr int Q = DP / 4;
    for (int e = threadIdx.x; e < C * Q; e += NT) {
        const int r = e / Q, c = 4 * (e % Q);
        f4 v = f4{0, 0, 0, 0};
        if (r < n) {
            const IO *s = src + (long long)r * ld + c;
            if (vec) {
                if (c < D) v = ld4(s);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (c + t < D) v[t] = ld1(s + t);
            }
        }
        *reinterpret_cast<f4 *>(dst + r * PITCH + c) = v;
    }
}

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// tokens of a chunk: the backward holds q, k, v, dout, a dk x dv state and two C x C matrices in 160 KB of LDS
inline int linattn_chunk(int dk, int dv) { return dk <= 64 && dv <= 64 ? 64 : 32; }

// Chunks a segment.  One workgroup walks a segment; fewer than about two workgroups a CU leave the card idle, and a segment costs
// a second pass over k and v (q and dout in the backward) and a state's round trip, so it is at least four chunks long.
inline int linattn_segment_chunks(int N, long long max_len, int H, int dk, int dv, int backward) {
    const int C = linattn_chunk(dk, dv);
    const long long nch = (max_len + C - 1) / C, walks = (long long)N * H * (backward ? 1 : (dv + 63) / 64);
    const long long want = (512 + walks - 1) / walks;
    long long segc = (nch + want - 1) / want;
    if (segc < 4) segc = 4;
    return (int)(segc < nch ? segc : nch > 0 ? nch : 1);
}

inline int linattn_problem(Problem &p, int dtype, const void *q, const void *k, const void *v, const float *g, const long long *st, const int *cu,
                           int N, long long tokens, int H, int G, int dk, int dv, float scale, int nseg, int segc, const char *name) {
    if (dtype != 0 && dtype != 1) { ss2d_set_error("%s: unknown dtype %d", name, dtype); return -1; }
    if (!q || !k || !v || !g || !st) { ss2d_set_error("%s: null pointer", name); return -2; }
    if (N <= 0 || tokens <= 0 || tokens > 0x7fffff00LL || H <= 0 || G <= 0 || nseg <= 0 || segc <= 0) { ss2d_set_error("%s: size out of range", name); return -3; }
    if (H % G) { ss2d_set_error("%s: %d heads are not a multiple of %d key heads", name, H, G); return -4; }
    if (dk < 1 || dk > 128 || dv < 1 || dv > 128) { ss2d_set_error("%s: dk %d and dv %d must be 1 ... 128", name, dk, dv); return -5; }
    if ((long long)N * H * nseg * 2 > 0x7ffffff0LL || (long long)N * H > 65535LL * 32) { ss2d_set_error("%s: too many sequences and heads", name); return -6; }
    p.q = q; p.k = k; p.v = v; p.g = g; p.cu = cu; p.tokens = tokens; p.N = N; p.H = H; p.G = G; p.dk = dk; p.dv = dv; p.scale = scale; p.nseg = nseg; p.segc = segc;
    p.qb = st[0]; p.ql = st[1]; p.qh = st[2]; p.kb = st[3]; p.kl = st[4]; p.kh = st[5];
    p.vb = st[6]; p.vl = st[7]; p.vh = st[8]; p.gb = st[9]; p.gl = st[10]; p.gh = st[11];
    const int m = 8;                                            // 16 bytes of bf16, 32 of fp32
    bool vec = dk % m == 0 && dv % m == 0 && ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0;
    for (int i = 0; i < 9; ++i) vec = vec && st[i] % m == 0;
    p.vec = vec;
    return 0;
}

}  // namespace linattn
