// Linear attention with a decay for each head, backward, for gfx950 (forward: ss2d_linattn_fwd.hip, formulas: ss2d_linattn.h).
//
// With D the gradient of the state behind a chunk, S the state in front of it (left by the forward), w_ij = scale exp(b_i - b_j) for
// j <= i (else 0), X_ij = w_ij q_i . k_j and Y_ij = w_ij do_i . v_j:
//   dq_i = sum_j Y_ij k_j + scale exp(b_i) S do_i          dk_j = sum_i Y_ij q_i + exp(b_C - b_j) D v_j
//   dv_j = sum_i X_ij do_i + exp(b_C - b_j) D^T k_j        D_prev = exp(b_C) D + sum_i scale exp(b_i) q_i do_i^T
// A decay g_t scales every path that crosses it, so its gradient is the sum over the pairs on both sides of it,
//   dg_t = sum_{i >= t > j} M_ij,  M_ij = w_ij (q_i . k_j)(do_i . v_j),
// with the state in front of the chunk as one more column, D as one more row.  It is taken as row sums minus column sums, added
// up from the chunk's end; pairs that do not cross t cancel there, but only pairs of ONE chunk, and the diagonal, whose terms
// are the largest and cross nothing, never enters.
//
// A workgroup walks one segment of one sequence and value head from its end to its start with D in accumulator registers (a wave owns
// 16-column slices of dv).  Segments as in the forward: own contributions, a join in order, the walk.
#include "ss2d_linattn.h"
#include "../../include/ss2d.h"

namespace {
using namespace linattn;

constexpr int NT = 256;

struct BwdArgs {
    Problem p;
    const void *dout;             // (rows, tokens, H, dv) dense
    const float *dlast;           // (N, H, dk, dv) or null
    const float *chunk_states;    // as the forward left them
    void *dq, *dk_, *dv_;         // dq, dk: (rows, tokens, G, dk) in the storage type, or (rows, tokens, H, dk) fp32 with H > G; dv (rows, tokens, H, dv)
    float *dg;                    // (rows, tokens, H)
    float *ds0;                   // (N, H, dk, dv) or null
    float *seg_states;            // as in the forward, for D
    double *seg_decay;
};

template <int TP, typename F>
__device__ __forceinline__ void each_tile_element(F f) {      // (row, column) of this thread's elements of D: tile t, register r
#pragma unroll
    for (int t = 0; t < TP; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) f(t, r);
}

// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_mov<DPP_ROW_ROR(8), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(4), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(2), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(1), 0xf, false>(0.0f, v);
    return v;
}

// a segment's own contribution to D: sum over its tokens of scale exp(b) q do^T
template <int DK, int C, typename IO>
__global__ __launch_bounds__(NT) void la_bwd_seg_kernel(const BwdArgs a) {
    constexpr int PK = DK + 4, PV = 64 + 4, KT = DK / 16, CT = C / 16;
    __shared__ __attribute__((aligned(16))) float lds[C * PK + C * PV + 64];
    float *Qs = lds, *Os = Qs + C * PK, *eb = Os + C * PV;
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, gq = lane >> 4;
    const int dvt = (p.dv + 63) / 64;
    int id = blockIdx.x;
    const int vt = id % dvt; id /= dvt;
    const int seg = id % p.nseg; id /= p.nseg;
    const int h = id % p.H, n = id / p.H;
    const Seq s = get_seq(p, n);
    const int c0 = seg * p.segc, nch = (s.len + C - 1) / C;
    const int c1 = segment_end(p, seg, nch);
    if (c0 >= c1) return;
    const int hk = h / (p.H / p.G), col = 64 * vt + 16 * wave + l16;
    const bool cok = col < p.dv;
    const IO *Q = static_cast<const IO *>(p.q) + s.row * p.qb + s.start * p.ql + hk * p.qh;
    const long long ldo = (long long)p.H * p.dv, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    const IO *DO = static_cast<const IO *>(a.dout) + ((s.row * p.tokens + s.start) * p.H + h) * (long long)p.dv + 64 * vt;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    f4 D[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) D[t] = f4{0, 0, 0, 0};
    double total = 0.0;
    for (int c = c1 - 1; c >= c0; --c) {
        const long long r0 = (long long)c * C;
        const int nr = s.len - r0 < C ? (int)(s.len - r0) : C;
        __syncthreads();
        load_tile<C, DK, PK, NT>(Qs, Q + r0 * p.ql, p.ql, nr, p.dk, p.vec);
        load_tile<C, 64, PV, NT>(Os, DO + r0 * ldo, ldo, nr, p.dv - 64 * vt, p.vec);
        const float gv = lane < nr ? limit_decay(g[(r0 + lane) * p.gl]) : 0.0f;
        const double b = chunk_decay_scan(gv, lane), bend = __shfl(b, 63, 64);
        total += bend;
        const float eend = exp2f((float)bend);
        if (wave == 0) eb[lane] = exp2f((float)b) * p.scale;
        __syncthreads();
#pragma unroll
        for (int t = 0; t < KT; ++t) D[t] *= eend;
#pragma unroll
        for (int it = 0; it < CT; ++it) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * gq + r;
                y[r] = Os[i * PV + 16 * wave + l16] * eb[i];
            }
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) D[t] = mfma4(Qs[(16 * it + 4 * gq + r) * PK + 16 * t + l16], y[r], D[t]);
        }
    }
    float *dst = a.seg_states + (nh * p.nseg + seg) * sz;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * t + 4 * gq + r;
            if (cok && k < p.dk) dst[(long long)k * p.dv + col] = D[t][r];
        }
    if (tid == 0 && vt == 0) a.seg_decay[nh * p.nseg + seg] = total;
}

// seg_states[s] = D behind segment s
__global__ __launch_bounds__(NT) void la_join_bwd_kernel(const BwdArgs a, int C) {
    const Problem &p = a.p;
    const long long sz = (long long)p.dk * p.dv;
    const long long e = (long long)blockIdx.x * NT + threadIdx.x;
    const long long nh = blockIdx.y;
    if (e >= sz) return;
    const Seq s = get_seq(p, (int)(nh / p.H));
    const int nch = (s.len + C - 1) / C, ns = segments_of(p, nch);
    float v = a.dlast ? a.dlast[nh * sz + e] : 0.0f;
    for (int i = ns - 1; i >= 0; --i) {
        float *u = a.seg_states + (nh * p.nseg + i) * sz + e;
        const float own = *u;
        *u = v;
        v = v * exp2f((float)a.seg_decay[nh * p.nseg + i]) + own;
    }
    if (a.ds0) a.ds0[nh * sz + e] = v;
}

template <typename IO>
__device__ void zero_rows(const Problem &p, IO *o, long long row, int w, int nw) {
    const long long lo = p.cu[0] < 0 ? 0 : p.cu[0] < p.tokens ? p.cu[0] : p.tokens;
    long long hi = p.cu[p.N];
    hi = hi < lo ? lo : hi < p.tokens ? hi : p.tokens;
    for (long long e = (long long)w * NT + threadIdx.x; e < lo * row; e += (long long)nw * NT) st1(o + e, 0.0f);
    for (long long e = hi * row + (long long)w * NT + threadIdx.x; e < p.tokens * row; e += (long long)nw * NT) st1(o + e, 0.0f);
}
constexpr int GAP_WGS = 16;

// QT: storage type of dq / dk (fp32 per value head when heads share keys, then summed)
template <int DK, int DV, int C, typename IO, typename QT>
__global__ __launch_bounds__(NT) void la_bwd_kernel(const BwdArgs a) {
    constexpr int PK = DK + 4, PV = DV + 4, PP = C + 4, KT = DK / 16, VT = DV / 16, CT = C / 16;
    constexpr int VW = (VT + 3) / 4, KW = (KT + 3) / 4;              // tiles of dv / of dk that a wave owns: wave + 4 m
    __shared__ __attribute__((aligned(16))) float lds[2 * C * PK + 2 * C * PV + DK * PV + 2 * C * PP + 8 * 64 + 4];
    float *Qs = lds, *Ks = Qs + C * PK, *Vs = Ks + C * PK, *Os = Vs + C * PV, *Ds = Os + C * PV, *Xs = Ds + DK * PV, *Ys = Xs + C * PP;
    float *bh = Ys + C * PP, *bl = bh + 64, *eb = bl + 64, *wt = eb + 64, *parts = wt + 64, *corners = parts + 256;
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, gq = lane >> 4;
    int id = blockIdx.x;
    const int main_wgs = p.N * p.H * p.nseg;
    const int hq = p.H > p.G ? p.H : p.G;                            // heads of dq / dk as written
    if (id >= main_wgs) {                                            // packed rows that belong to no sequence
        zero_rows(p, static_cast<QT *>(a.dq), (long long)hq * p.dk, id - main_wgs, GAP_WGS);
        zero_rows(p, static_cast<QT *>(a.dk_), (long long)hq * p.dk, id - main_wgs, GAP_WGS);
        zero_rows(p, static_cast<IO *>(a.dv_), (long long)p.H * p.dv, id - main_wgs, GAP_WGS);
        zero_rows(p, a.dg, p.H, id - main_wgs, GAP_WGS);
        return;
    }
    const int seg = id % p.nseg; id /= p.nseg;
    const int h = id % p.H, n = id / p.H;
    const Seq s = get_seq(p, n);
    const int c0 = seg * p.segc, nch = (s.len + C - 1) / C;
    const int c1 = segment_end(p, seg, nch);
    const bool empty = s.len == 0;
    if (c0 >= c1 && !(empty && seg == 0)) return;
    const int hk = h / (p.H / p.G);
    const long long ldv = (long long)p.H * p.dv, ldq = (long long)hq * p.dk, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    const IO *Q = static_cast<const IO *>(p.q) + s.row * p.qb + s.start * p.ql + hk * p.qh;
    const IO *K = static_cast<const IO *>(p.k) + s.row * p.kb + s.start * p.kl + hk * p.kh;
    const IO *V = static_cast<const IO *>(p.v) + s.row * p.vb + s.start * p.vl + h * p.vh;
    const long long t0 = s.row * p.tokens + s.start;
    const IO *DO = static_cast<const IO *>(a.dout) + (t0 * p.H + h) * (long long)p.dv;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    QT *DQ = static_cast<QT *>(a.dq) + (t0 * hq + h) * (long long)p.dk;
    QT *DKp = static_cast<QT *>(a.dk_) + (t0 * hq + h) * (long long)p.dk;
    IO *DVp = static_cast<IO *>(a.dv_) + (t0 * p.H + h) * (long long)p.dv;
    float *DG = a.dg + t0 * p.H + h;
    f4 D[VW][KT];
    const float *init = p.nseg > 1 ? a.seg_states + (nh * p.nseg + seg) * sz : a.dlast ? a.dlast + nh * sz : nullptr;
#pragma unroll
    for (int m = 0; m < VW; ++m)
        each_tile_element<KT>([&](int t, int r) {
            const int k = 16 * t + 4 * gq + r, col = 16 * (wave + 4 * m) + l16;
            D[m][t][r] = init && col < p.dv && k < p.dk ? init[(long long)k * p.dv + col] : 0.0f;
        });
    const long long cb = chunk_base(p, s, n, C);
    for (int c = c1 - 1; c >= c0; --c) {
        const long long r0 = (long long)c * C;
        const int nr = s.len - r0 < C ? (int)(s.len - r0) : C;
        __syncthreads();
        load_tile<C, DK, PK, NT>(Qs, Q + r0 * p.ql, p.ql, nr, p.dk, p.vec);
        load_tile<C, DK, PK, NT>(Ks, K + r0 * p.kl, p.kl, nr, p.dk, p.vec);
        load_tile<C, DV, PV, NT>(Vs, V + r0 * p.vl, p.vl, nr, p.dv, p.vec);
        load_tile<C, DV, PV, NT>(Os, DO + r0 * ldv, ldv, nr, p.dv, p.vec);
#pragma unroll
        for (int m = 0; m < VW; ++m)
            if (wave + 4 * m < VT)
                each_tile_element<KT>([&](int t, int r) { Ds[(16 * t + 4 * gq + r) * PV + 16 * (wave + 4 * m) + l16] = D[m][t][r]; });
        const float gv = lane < nr ? limit_decay(g[(r0 + lane) * p.gl]) : 0.0f;
        const double b = chunk_decay_scan(gv, lane), bend = __shfl(b, 63, 64);
        const float eend = exp2f((float)bend);
        if (wave == 0) {
            const float hi = (float)b;
            bh[lane] = hi;
            bl[lane] = (float)(b - hi);
            eb[lane] = exp2f(hi) * p.scale;
            wt[lane] = exp2f((float)(bend - b));
        }
        parts[wave * 64 + lane] = 0.0f;                                  // gradient of b_i, a partial sum of every wave
        __syncthreads();
        // X, Y and the sums of M below the diagonal
        for (int t = wave; t < CT * CT; t += 4) {
            const int it = t / CT, jt = t % CT;
            if (jt > it) continue;
            f4 x = f4{0, 0, 0, 0}, y = f4{0, 0, 0, 0};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const f4 u = *reinterpret_cast<const f4 *>(Qs + (16 * it + l16) * PK + 16 * kt + 4 * gq);
                const f4 w = *reinterpret_cast<const f4 *>(Ks + (16 * jt + l16) * PK + 16 * kt + 4 * gq);
#pragma unroll
                for (int r = 0; r < 4; ++r) x = mfma4(u[r], w[r], x);
            }
#pragma unroll
            for (int vt = 0; vt < VT; ++vt) {
                const f4 u = *reinterpret_cast<const f4 *>(Os + (16 * it + l16) * PV + 16 * vt + 4 * gq);
                const f4 w = *reinterpret_cast<const f4 *>(Vs + (16 * jt + l16) * PV + 16 * vt + 4 * gq);
#pragma unroll
                for (int r = 0; r < 4; ++r) y = mfma4(u[r], w[r], y);
            }
            const int j = 16 * jt + l16;
            const float hj = bh[j], lj = bl[j];
            float colsum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * gq + r;
                const float w = j <= i ? p.scale * exp2f((bh[i] - hj) + (bl[i] - lj)) : 0.0f;
                const float yw = j <= i ? y[r] * w : 0.0f, xw = j <= i ? x[r] * w : 0.0f;
                const float m = j < i ? x[r] * yw : 0.0f;
                Xs[i * PP + j] = xw;
                Ys[i * PP + j] = yw;
                colsum += m;
                const float rs = row16_sum(m);
                if (l16 == 0) parts[wave * 64 + i] += rs;
            }
            colsum += __shfl_xor(colsum, 16, 64);
            colsum += __shfl_xor(colsum, 32, 64);
            if (gq == 0) parts[wave * 64 + j] -= colsum;
        }
        __syncthreads();
        // dq and dk: a wave owns 16-column slices of dk.  The corner <D, S_end> = exp(b_C) <D, S> + sum_j k_j . exp(b_C - b_j) D v_j.
        const float *Sc = a.chunk_states + ((cb + c) * p.H + h) * sz;
        float corner_s = 0.0f, corner_k = 0.0f;
#pragma unroll 1
        for (int m = 0; m < KW; ++m) {
            const int kt = wave + 4 * m;
            if (kt >= KT) break;
            const int k = 16 * kt + l16;                              // this lane's column
            const bool kok = k < p.dk;
            f4 sf[VT], df[VT];
#pragma unroll
            for (int vt = 0; vt < VT; ++vt) {
                const int v0 = 16 * vt + 4 * gq;
                sf[vt] = f4{0, 0, 0, 0};
                if (kok) {
                    if (p.vec) {
                        if (v0 < p.dv) sf[vt] = ld4(Sc + (long long)k * p.dv + v0);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (v0 + r < p.dv) sf[vt][r] = Sc[(long long)k * p.dv + v0 + r];
                    }
                }
                df[vt] = *reinterpret_cast<const f4 *>(Ds + k * PV + v0);
#pragma unroll
                for (int r = 0; r < 4; ++r) corner_s += sf[vt][r] * df[vt][r];
            }
#pragma unroll 1
            for (int it = 0; it < CT; ++it) {
                f4 dq = f4{0, 0, 0, 0}, dk = f4{0, 0, 0, 0};
#pragma unroll
                for (int vt = 0; vt < VT; ++vt) {
                    const f4 u = *reinterpret_cast<const f4 *>(Os + (16 * it + l16) * PV + 16 * vt + 4 * gq);
                    const f4 w = *reinterpret_cast<const f4 *>(Vs + (16 * it + l16) * PV + 16 * vt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) { dq = mfma4(u[r], sf[vt][r], dq); dk = mfma4(w[r], df[vt][r], dk); }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    dq[r] *= eb[i];
                    dk[r] *= wt[i];
                    const float qq = dq[r] * Qs[i * PK + k], kk = dk[r] * Ks[i * PK + k];
                    corner_k += kk;
                    const float rs = row16_sum(qq - kk);
                    if (l16 == 0) parts[wave * 64 + i] += rs;
                }
                for (int jt = 0; jt <= it; ++jt) {
                    const f4 u = *reinterpret_cast<const f4 *>(Ys + (16 * it + l16) * PP + 16 * jt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) dq = mfma4(u[r], Ks[(16 * jt + 4 * gq + r) * PK + k], dq);
                }
                for (int jt = it; jt < CT; ++jt)                      // rows of tile `it` of dk: sums over the later tokens
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        dk = mfma4(Ys[(16 * jt + 4 * gq + r) * PP + 16 * it + l16], Qs[(16 * jt + 4 * gq + r) * PK + k], dk);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    if (i < nr && kok) {
                        st1(DQ + (r0 + i) * ldq + k, dq[r]);
                        st1(DKp + (r0 + i) * ldq + k, dk[r]);
                    }
                }
            }
        }
        const float corner = lanes_sum<64>(corner_s) * eend + lanes_sum<64>(corner_k);
        if (lane == 0) corners[wave] = corner;
        // dv and the state: a wave owns 16-column slices of dv
#pragma unroll
        for (int m = 0; m < VW; ++m) {
            if (wave + 4 * m >= VT) break;
            const int col = 16 * (wave + 4 * m) + l16;
            const bool cok = col < p.dv;
#pragma unroll 1
            for (int jt = 0; jt < CT; ++jt) {
                f4 acc = f4{0, 0, 0, 0};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const f4 u = *reinterpret_cast<const f4 *>(Ks + (16 * jt + l16) * PK + 16 * kt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc = mfma4(u[r], D[m][kt][r], acc);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] *= wt[16 * jt + 4 * gq + r];
                for (int it = jt; it < CT; ++it)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc = mfma4(Xs[(16 * it + 4 * gq + r) * PP + 16 * jt + l16], Os[(16 * it + 4 * gq + r) * PV + col], acc);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * jt + 4 * gq + r;
                    if (j < nr && cok) st1(DVp + (r0 + j) * ldv + col, acc[r]);
                }
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) D[m][t] *= eend;
#pragma unroll
            for (int it = 0; it < CT; ++it) {
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    y[r] = Os[i * PV + col] * eb[i];
                }
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) D[m][t] = mfma4(Qs[(16 * it + 4 * gq + r) * PK + 16 * t + l16], y[r], D[m][t]);
            }
        }
        __syncthreads();
        if (wave == 0) {
            double x = 0.0;                                           // gradient of b_lane inside the chunk, then its sums from the end
#pragma unroll
            for (int w = 0; w < 4; ++w) x += (double)parts[w * 64 + lane];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_down(x, d, 64);
                if (lane + d < 64) x += o;
            }
            const float e = (corners[0] + corners[1]) + (corners[2] + corners[3]);
            if (lane < nr) DG[(r0 + lane) * p.H] = (float)(x + (double)e);
        }
    }
    if (a.ds0 && p.nseg == 1) {
        float *d = a.ds0 + nh * sz;
#pragma unroll
        for (int m = 0; m < VW; ++m)
            each_tile_element<KT>([&](int t, int r) {
                const int k = 16 * t + 4 * gq + r, col = 16 * (wave + 4 * m) + l16;
                if (col < p.dv && k < p.dk) d[(long long)k * p.dv + col] = D[m][t][r];
            });
    }
}

// dq / dk of the value heads that share a key head, summed: (rows, G, rep, dk) fp32 -> (rows, G, dk)
template <typename IO>
__global__ __launch_bounds__(NT) void la_head_sum_kernel(const float *a, const float *b, IO *oa, IO *ob, long long total, int rep, int dk) {
    const long long e = (long long)blockIdx.x * NT + threadIdx.x;
    if (e >= total) return;
    const long long rg = e / dk;
    const float *src = (blockIdx.y ? b : a) + rg * rep * dk + (e - rg * dk);
    float v = src[0];
    for (int i = 1; i < rep; ++i) v += src[(long long)i * dk];
    st1((blockIdx.y ? ob : oa) + e, v);
}

template <int DK, int DV, int C, typename IO>
void launch_bwd(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const Problem &p = a.p;
    const unsigned walks = (unsigned)((long long)p.N * p.H * p.nseg);
    if (p.nseg > 1) {
        ss2d_launch((la_bwd_seg_kernel<DK, C, IO>), dim3(walks * ((p.dv + 63) / 64)), dim3(NT), 0, s, a);
        const long long sz = (long long)p.dk * p.dv;
        ss2d_launch(la_join_bwd_kernel, dim3((unsigned)((sz + NT - 1) / NT), (unsigned)(p.N * p.H)), dim3(NT), 0, s, a, C);
    }
    if (p.H > p.G) ss2d_launch((la_bwd_kernel<DK, DV, C, IO, float>), dim3(walks + gaps), dim3(NT), 0, s, a);
    else ss2d_launch((la_bwd_kernel<DK, DV, C, IO, IO>), dim3(walks + gaps), dim3(NT), 0, s, a);
}

template <typename IO>
void dispatch_bwd(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const int dk = a.p.dk, dv = a.p.dv;
    if (dv <= 64) {
        if (dk <= 16) launch_bwd<16, 64, 64, IO>(a, gaps, s);
        else if (dk <= 64) launch_bwd<64, 64, 64, IO>(a, gaps, s);
        else launch_bwd<128, 64, 32, IO>(a, gaps, s);
    } else {
        if (dk <= 16) launch_bwd<16, 128, 32, IO>(a, gaps, s);
        else if (dk <= 64) launch_bwd<64, 128, 32, IO>(a, gaps, s);
        else launch_bwd<128, 128, 32, IO>(a, gaps, s);
    }
}

}  // namespace

extern "C" int ss2d_linattn_bwd(int dtype, const void *q, const void *k, const void *v, const float *g, const long long *strides,
                                const int *cu_seqlens, const void *dout, const float *dlast, const float *chunk_states, void *dq,
                                void *dk_out, void *dv_out, float *dg, float *ds0, float *dq_heads, float *dk_heads, float *seg_states,
                                double *seg_decay, int N, long long tokens, int H, int G, int dk, int dv, float scale, int nseg,
                                int seg_chunks, void *stream) {
    BwdArgs a{};
    int rc = linattn_problem(a.p, dtype, q, k, v, g, strides, cu_seqlens, N, tokens, H, G, dk, dv, scale, nseg, seg_chunks, "linattn_bwd");
    if (rc) return rc;
    if (!dout || !chunk_states || !dq || !dk_out || !dv_out || !dg) { ss2d_set_error("linattn_bwd: null pointer"); return -2; }
    if (H > G && (!dq_heads || !dk_heads)) { ss2d_set_error("linattn_bwd: shared key heads need dq_heads and dk_heads"); return -2; }
    if (nseg > 1 && (!seg_states || !seg_decay)) { ss2d_set_error("linattn_bwd: segments without a workspace"); return -2; }
    a.dout = dout; a.dlast = dlast; a.chunk_states = chunk_states; a.dq = H > G ? dq_heads : dq; a.dk_ = H > G ? dk_heads : dk_out;
    a.dv_ = dv_out; a.dg = dg; a.ds0 = ds0; a.seg_states = seg_states; a.seg_decay = seg_decay;
    a.p.vec = a.p.vec && (uintptr_t)dout % 16 == 0;
    const unsigned gaps = cu_seqlens ? GAP_WGS : 0;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == SS2D_DTYPE_BF16) dispatch_bwd<bf16>(a, gaps, s); else dispatch_bwd<float>(a, gaps, s);
    if (H > G) {
        const long long rows = (cu_seqlens ? 1 : N) * tokens, total = rows * G * dk;
        const dim3 grid((unsigned)((total + NT - 1) / NT), 2);
        if (dtype == SS2D_DTYPE_BF16) ss2d_launch((la_head_sum_kernel<bf16>), grid, dim3(NT), 0, s, dq_heads, dk_heads, (bf16 *)dq, (bf16 *)dk_out, total, H / G, dk);
        else ss2d_launch((la_head_sum_kernel<float>), grid, dim3(NT), 0, s, dq_heads, dk_heads, (float *)dq, (float *)dk_out, total, H / G, dk);
    }
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("linattn_bwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
