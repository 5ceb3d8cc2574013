// Linear attention with a decay for each head, forward, for gfx950 (formulas: ss2d_linattn.h).  Beside the selective scan
// (ss2d_scan_fwd.hip), whose decay is per channel and state: here one decay per head and token, a dk x dv state, and the work
// inside a chunk is matrix products.
//
// A workgroup walks one segment of one sequence and value head with the state in accumulator registers; a wave owns 16
// columns of dv.  A sequence is cut into segments when there are too few (sequence, head) pairs to fill the card: a first pass
// leaves every segment's own contribution, a small pass joins them in order, and the main pass starts each segment from its
// true state.
#include <type_traits>
#include "ss2d_linattn.h"
#include "../../include/ss2d.h"

namespace {
using namespace linattn;

constexpr int NT = 256;

struct FwdArgs {
    Problem p;
    void *o;                      // (rows, tokens, H, dv) dense
    const float *s0;              // (N, H, dk, dv) or null
    float *last;                  // (N, H, dk, dv) or null
    float *chunk_states;          // (slots, H, dk, dv): the state in front of every chunk, or null
    float *seg_states;            // (N, H, nseg, dk, dv): contributions, then the states in front of the segments; null with nseg == 1
    double *seg_decay;            // (N, H, nseg): log2 of a segment's decay
};

constexpr int GAP_WGS = 16;
template <typename IO>
__device__ void zero_gaps(const Problem &p, IO *o, long long row, int w) {
    const long long lo = p.cu[0] < 0 ? 0 : p.cu[0] < p.tokens ? p.cu[0] : p.tokens;
    long long hi = p.cu[p.N];
    hi = hi < lo ? lo : hi < p.tokens ? hi : p.tokens;
    const long long step = (long long)GAP_WGS * NT;
    for (long long e = (long long)w * NT + threadIdx.x; e < lo * row; e += step) st1(o + e, 0.0f);
    for (long long e = hi * row + (long long)w * NT + threadIdx.x; e < p.tokens * row; e += step) st1(o + e, 0.0f);
}

// mode 0: the whole walk; mode 1: only a segment's own contribution to the state
template <int DK, int C, int MODE, typename IO>
__global__ __launch_bounds__(NT) void la_fwd_kernel(const FwdArgs a) {
    constexpr int PK = DK + 4, PV = 64 + 4, PP = C + 4, KT = DK / 16, CT = C / 16;
    __shared__ __attribute__((aligned(16))) float lds[C * PK + C * PV + 256 + (MODE == 0 ? C * PK + C * PP : 0)];
    float *Ks = lds, *Vs = Ks + C * PK, *bh = Vs + C * PV, *bl = bh + 64, *eb = bl + 64, *wt = eb + 64, *Qs = wt + 64, *Ps = Qs + C * PK;
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, gq = lane >> 4;
    const int dvt = (p.dv + 63) / 64;
    int id = blockIdx.x;
    if (id >= p.N * p.H * p.nseg * dvt) {        // packed rows that belong to no sequence: their output is zero
        if (MODE == 0) zero_gaps(p, static_cast<IO *>(a.o), (long long)p.H * p.dv, id - p.N * p.H * p.nseg * dvt);
        return;
    }
    const int vt = id % dvt; id /= dvt;
    const int seg = id % p.nseg; id /= p.nseg;
    const int h = id % p.H, n = id / p.H;
    const Seq s = get_seq(p, n);
    const int c0 = seg * p.segc, nch = (s.len + C - 1) / C;
    const int c1 = segment_end(p, seg, nch);
    const bool empty = s.len == 0;
    if (c0 >= c1 && !(empty && seg == 0)) return;
    if (MODE == 1 && c1 == nch && !empty && !a.last) return;     // nothing starts from the last segment's end
    const int hk = h / (p.H / p.G), col = 64 * vt + 16 * wave + l16;
    const bool cok = col < p.dv;
    const IO *Q = static_cast<const IO *>(p.q) + s.row * p.qb + s.start * p.ql + hk * p.qh;
    const IO *K = static_cast<const IO *>(p.k) + s.row * p.kb + s.start * p.kl + hk * p.kh;
    const IO *V = static_cast<const IO *>(p.v) + s.row * p.vb + s.start * p.vl + h * p.vh + 64 * vt;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    IO *O = static_cast<IO *>(a.o) + ((s.row * p.tokens + s.start) * p.H + h) * (long long)p.dv;
    const long long ldo = (long long)p.H * p.dv, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    f4 S[KT];
    const float *init = MODE == 1 ? nullptr : p.nseg > 1 ? a.seg_states + (nh * p.nseg + seg) * sz : a.s0 ? a.s0 + nh * sz : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * t + 4 * gq + r;
            S[t][r] = init && cok && k < p.dk ? init[(long long)k * p.dv + col] : 0.0f;
        }
    double total = 0.0;
    const long long cb = chunk_base(p, s, n, C);
    for (int c = c0; c < c1; ++c) {
        const long long r0 = (long long)c * C;
        const int nr = s.len - r0 < C ? (int)(s.len - r0) : C;
        if (MODE == 0 && a.chunk_states) {
            float *d = a.chunk_states + ((cb + c) * p.H + h) * sz;
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int k = 16 * t + 4 * gq + r;
                    if (cok && k < p.dk) d[(long long)k * p.dv + col] = S[t][r];
                }
        }
        __syncthreads();
        if (MODE == 0) load_tile<C, DK, PK, NT>(Qs, Q + r0 * p.ql, p.ql, nr, p.dk, p.vec);
        load_tile<C, DK, PK, NT>(Ks, K + r0 * p.kl, p.kl, nr, p.dk, p.vec);
        load_tile<C, 64, PV, NT>(Vs, V + r0 * p.vl, p.vl, nr, p.dv - 64 * vt, p.vec);
        const float gv = lane < nr ? limit_decay(g[(r0 + lane) * p.gl]) : 0.0f;
        const double b = chunk_decay_scan(gv, lane), bend = __shfl(b, 63, 64);
        total += bend;
        const float eend = exp2f((float)bend);
        if (wave == 0) {
            const float hi = (float)b;
            bh[lane] = hi;
            bl[lane] = (float)(b - hi);
            eb[lane] = exp2f(hi) * p.scale;
            wt[lane] = exp2f((float)(bend - b));
        }
        __syncthreads();
        if (MODE == 0) {
            // P[i][j] = scale exp(b_i - b_j) q_i . k_j, j <= i: tiles (it, jt) dealt to the waves
            for (int t = wave; t < CT * CT; t += 4) {
                const int it = t / CT, jt = t % CT;
                if (jt > it) continue;
                f4 acc = f4{0, 0, 0, 0};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const f4 x = *reinterpret_cast<const f4 *>(Qs + (16 * it + l16) * PK + 16 * kt + 4 * gq);
                    const f4 y = *reinterpret_cast<const f4 *>(Ks + (16 * jt + l16) * PK + 16 * kt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc = mfma4(x[r], y[r], acc);
                }
                const int j = 16 * jt + l16;
                const float hj = bh[j], lj = bl[j];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    Ps[i * PP + j] = j <= i ? acc[r] * p.scale * exp2f((bh[i] - hj) + (bl[i] - lj)) : 0.0f;
                }
            }
            __syncthreads();
#pragma unroll
            for (int it = 0; it < CT; ++it) {
                f4 acc = f4{0, 0, 0, 0};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const f4 x = *reinterpret_cast<const f4 *>(Qs + (16 * it + l16) * PK + 16 * kt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc = mfma4(x[r], S[kt][r], acc);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] *= eb[16 * it + 4 * gq + r];
                for (int jt = 0; jt <= it; ++jt) {
                    const f4 x = *reinterpret_cast<const f4 *>(Ps + (16 * it + l16) * PP + 16 * jt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc = mfma4(x[r], Vs[(16 * jt + 4 * gq + r) * PV + 16 * wave + l16], acc);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    if (i < nr && cok) st1(O + (r0 + i) * ldo + col, acc[r]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] *= eend;
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * jt + 4 * gq + r;
                y[r] = Vs[j * PV + 16 * wave + l16] * wt[j];
            }
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t] = mfma4(Ks[(16 * jt + 4 * gq + r) * PK + 16 * t + l16], y[r], S[t]);
        }
    }
    float *dst = MODE == 1 ? a.seg_states + (nh * p.nseg + seg) * sz : (a.last && p.nseg == 1) ? a.last + nh * sz : nullptr;
    if (dst) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = 16 * t + 4 * gq + r;
                if (cok && k < p.dk) dst[(long long)k * p.dv + col] = S[t][r];
            }
        if (MODE == 1 && tid == 0 && vt == 0) a.seg_decay[nh * p.nseg + seg] = total;
    }
}

// joins the segments of a (sequence, head): seg_states[s] = state in front of segment s; one thread per state element
__global__ __launch_bounds__(NT) void la_join_fwd_kernel(const FwdArgs a, int C) {
    const Problem &p = a.p;
    const long long sz = (long long)p.dk * p.dv;
    const long long e = (long long)blockIdx.x * NT + threadIdx.x;
    const long long nh = blockIdx.y;
    if (e >= sz) return;
    const Seq s = get_seq(p, (int)(nh / p.H));
    const int nch = (s.len + C - 1) / C, ns = segments_of(p, nch);
    float v = a.s0 ? a.s0[nh * sz + e] : 0.0f;
    for (int i = 0; i < ns; ++i) {
        float *u = a.seg_states + (nh * p.nseg + i) * sz + e;
        if (i + 1 == ns && !a.last) { *u = v; break; }
        const float own = *u;
        *u = v;
        v = v * exp2f((float)a.seg_decay[nh * p.nseg + i]) + own;
    }
    if (a.last) a.last[nh * sz + e] = v;
}

template <int DK, int C, typename IO>
void launch_fwd(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    const Problem &p = a.p;
    const unsigned grid = (unsigned)((long long)p.N * p.H * p.nseg * ((p.dv + 63) / 64));
    if (p.nseg > 1) {
        ss2d_launch((la_fwd_kernel<DK, C, 1, IO>), dim3(grid), dim3(NT), 0, s, a);
        const long long sz = (long long)p.dk * p.dv;
        ss2d_launch(la_join_fwd_kernel, dim3((unsigned)((sz + NT - 1) / NT), (unsigned)(p.N * p.H)), dim3(NT), 0, s, a, C);
    }
    ss2d_launch((la_fwd_kernel<DK, C, 0, IO>), dim3(grid + gaps), dim3(NT), 0, s, a);
}

template <typename IO>
void dispatch_fwd(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    const int dk = a.p.dk;
    const bool c64 = linattn_chunk(a.p.dk, a.p.dv) == 64;
    if (dk <= 16) c64 ? launch_fwd<16, 64, IO>(a, gaps, s) : launch_fwd<16, 32, IO>(a, gaps, s);
    else if (dk <= 64) c64 ? launch_fwd<64, 64, IO>(a, gaps, s) : launch_fwd<64, 32, IO>(a, gaps, s);
    else launch_fwd<128, 32, IO>(a, gaps, s);
}

}  // namespace

extern "C" int ss2d_linattn_chunk(int dk, int dv) { return linattn_chunk(dk, dv); }
extern "C" int ss2d_linattn_segment_chunks(int N, long long max_len, int H, int dk, int dv, int backward) {
    return N > 0 && max_len >= 0 && H > 0 ? linattn_segment_chunks(N, max_len, H, dk, dv, backward) : 1;
}

extern "C" int ss2d_linattn_fwd(int dtype, const void *q, const void *k, const void *v, const float *g, const long long *strides,
                                const int *cu_seqlens, const float *s0, void *out, float *last, float *chunk_states,
                                float *seg_states, double *seg_decay, int N, long long tokens, int H, int G, int dk, int dv, float scale,
                                int nseg, int seg_chunks, void *stream) {
    FwdArgs a{};
    int rc = linattn_problem(a.p, dtype, q, k, v, g, strides, cu_seqlens, N, tokens, H, G, dk, dv, scale, nseg, seg_chunks, "linattn_fwd");
    if (rc) return rc;
    if (!out) { ss2d_set_error("linattn_fwd: null pointer"); return -2; }
    if (nseg > 1 && (!seg_states || !seg_decay)) { ss2d_set_error("linattn_fwd: segments without a workspace"); return -2; }
    a.o = out; a.s0 = s0; a.last = last; a.chunk_states = chunk_states; a.seg_states = seg_states; a.seg_decay = seg_decay;
    const unsigned gaps = cu_seqlens ? GAP_WGS : 0;
    if (dtype == SS2D_DTYPE_BF16) dispatch_fwd<bf16>(a, gaps, (hipStream_t)stream); else dispatch_fwd<float>(a, gaps, (hipStream_t)stream);
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("linattn_fwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
