// Linear attention with a decay for each head, forward, for gfx950 (formulas: ss2d_linattn.h).  Beside the selective scan
// (ss2d_scan_fwd.hip), whose decay is per channel and state: here one decay per head and token, a dk x dv state, and the work
// inside a chunk is matrix products.
//
// A workgroup walks one segment of one sequence and value head with the state in accumulator registers; a wave owns 16
// columns of dv.  A sequence is cut into segments when there are too few (sequence, head) pairs to fill the card: a first pass
// leaves every segment's own contribution, a small pass joins them in order, and the main pass starts each segment from its
// true state.
//
// Measured (a 1 GB copy reaches 5.0 TB/s).  65536 tokens, 8 heads of 128 x 128 bf16: contributions 70 us (268 MB, 3.8 TB/s), join 15, walk 182 (537 MB, 2.9
// TB/s): the walk keeps the matrix units busy 38% of its time and LDS 42% (a quarter of that bank conflicts of 8-byte writes); the rest is the splitting of
// fp32 factors and the wait at three barriers a chunk (about 11,000 cycles a workgroup, two workgroups a CU).  24 x 3136 tokens, 3 heads of 16 x 64 fp32 with the
// states for the backward: 15 + 5 + 42 us (159 MB, 3.8 TB/s).  One prompt of 17 tokens: 7.7 us, of which 4 are a launch.
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
    float *seg_states;            // (slots, H, dk, dv): contributions, then the states in front of the segments; null with nseg == 1
    double *seg_decay;            // (slots, H): log2 of a segment's decay
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

// mode 0: the whole walk; mode 1: only a segment's own contribution to the state; mode 2: the backward's, sum of scale exp(b) q dout^T from the
// segment's end, with q in the place of k and dout in that of v
// fp32 on v_mfma_f32_16x16x4_f32, 64 columns of dv a workgroup: a lane holds row / column l16 of an operand and contracted indices 4 gq + r of a
// 16-block in step r, so a state tile in accumulators is an operand; direct operands are 16-byte LDS reads, transposed ones 4-byte reads, both free of
// bank conflicts at a pitch of 4 mod 16 floats.  The next chunk is in flight in registers.
template <int DK, int C, int MODE, bool VEC>
__global__ __launch_bounds__(NT) void la_fwd_kernel(const FwdArgs a) {
    constexpr int PK = DK + 4, PV = 64 + 4, PP = C + 4, KT = DK / 16, CT = C / 16;
    __shared__ __attribute__((aligned(16))) float lds[C * PK + C * PV + 640 + (MODE == 0 ? C * PK + C * PP : 0)];
    float *Ks = lds, *Vs = Ks + C * PK, *decays = Vs + C * PV, *Qs = decays + 640, *Ps = Qs + C * PK;
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, gq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int dvt = (p.dv + 63) / 64, walks = p.slots * p.H * dvt;
    if ((int)blockIdx.x >= walks) {              // packed rows that belong to no sequence: their output is zero
        if (MODE == 0) zero_gaps(p, static_cast<float *>(a.o), (long long)p.H * p.dv, blockIdx.x - walks);
        return;
    }
    int id = xcd_remap(blockIdx.x, walks);
    const int vt = id % dvt; id /= dvt;
    const int h = id % p.H; id /= p.H;
    const int slot = id;
    int n, seg;
    walk_of(p, slot, C, n, seg);
    if (seg < 0) return;
    const Seq s = get_seq(p, n);
    const int c0 = seg * p.segc, nch = (s.len + C - 1) / C;
    const int c1 = segment_end(p, seg, nch);
    const bool empty = s.len == 0;
    if (c0 >= c1 && !(empty && seg == 0)) return;
    if (MODE == 1 && c1 == nch) return;          // no segment starts from the last one's end
    if (MODE == 2 && c0 == 0) return;            // (here: from the first one's)
    const int hk = h / (p.H / p.G), col = 64 * vt + 16 * wave + l16, first = MODE == 2 ? c1 - 1 : c0, dvc = p.dv - 64 * vt;
    const bool cok = col < p.dv;
    const float *Q = static_cast<const float *>(p.q) + s.row * p.qb + (s.start + (long long)c0 * C) * p.ql + hk * p.qh;
    const float *K = static_cast<const float *>(p.k) + s.row * p.kb + (s.start + (long long)first * C) * p.kl + hk * p.kh;
    const float *V = static_cast<const float *>(p.v) + s.row * p.vb + (s.start + (long long)first * C) * p.vl + h * p.vh + 64 * vt;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    const long long ldo = (long long)p.H * p.dv, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    float *O = static_cast<float *>(a.o) + ((s.row * p.tokens + s.start + (long long)c0 * C) * p.H + h) * (long long)p.dv;
    f4 S[KT];
    const float *init = MODE >= 1 ? nullptr : segments_of(p, nch) > 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.s0 ? a.s0 + nh * sz : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * t + 4 * gq + r;
            S[t][r] = init && cok && k < p.dk ? init[k * p.dv + col] : 0.0f;
        }
    double total = 0.0;
    float *saved = MODE == 0 && a.chunk_states ? a.chunk_states + ((chunk_base(p, s, n, C) + c0) * p.H + h) * sz : nullptr;
    TileRegsF<C, DK, PK, NT, VEC> qr, kr;
    TileRegsF<C, 64, PV, NT, VEC> vr;
    qr.init(p.ql, p.dk);
    kr.init(p.kl, p.dk);
    vr.init(p.vl, dvc);
    auto rows_of = [&](int c) { const int left = s.len - c * C; return left < C ? left : C; };
    constexpr int STEP = MODE == 2 ? -1 : 1;
    auto fetch = [&](int c) {                    // chunk c, the tensors' pointers at chunk c
        const int nr = rows_of(c);
        if (MODE == 0) qr.load(Q, p.ql, nr, p.dk);
        kr.load(K, p.kl, nr, p.dk);
        vr.load(V, p.vl, nr, dvc);
        Q += C * p.ql; K += STEP * C * p.kl; V += STEP * C * p.vl;
    };
    float gr = 0.0f;                             // wave 0: decays, a chunk ahead of the tiles
    auto fetch_g = [&](int c) {
        if (wave == 0 && c >= c0 && c < c1) gr = lane < rows_of(c) ? limit_decay(g[((long long)c * C + lane) * p.gl]) : 0.0f;
    };
    auto scan = [&](int c) {                     // two chunks of: b (two terms), scale exp(b), exp(b_C - b), exp(b_C)
        if (wave == 0 && c >= c0 && c < c1) {
            float *d = decays + (c & 1) * 320;
            const double b = chunk_decay_scan(gr), bend = lane63(b);
            const float hi = (float)b;
            if (MODE >= 1) total += bend;
            d[lane] = hi;
            d[64 + lane] = (float)(b - hi);
            d[128 + lane] = hw_exp2(hi) * p.scale;
            d[192 + lane] = hw_exp2((float)(bend - b));
            if (lane == 63) d[256] = hw_exp2((float)bend);
        }
    };
    fetch_g(first);
    scan(first);
    fetch_g(first + STEP);
    if (c0 < c1) fetch(first);
    // A NaN or an infinity in v_j times the zero weight of an earlier row would reach that row.  Once one has been met, such values stay out of the
    // products and are added to the rows from j on alone, and their columns of the state become NaN.
    int *poison = reinterpret_cast<int *>(decays + 300);                // (the first chunk's set of decays ends at 257)
    if (MODE == 0 && tid == 0) *poison = 0;
#pragma unroll 1
    for (int c = first; c >= c0 && c < c1; c += STEP) {
        const int nr = rows_of(c);
        if (MODE == 0 && saved) {
            float *d = saved + (4 * gq) * p.dv + col;
            int step = p.dv;
            asm volatile("" : "+s"(step));       // (else the offsets of all rows live in registers across the loop)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (cok && 16 * t + 4 * gq + r < p.dk) *d = S[t][r];
                    d += step;
                }
                d += 12 * step;
            }
            saved += p.H * sz;
        }
        __syncthreads();
        if (MODE == 0) qr.put(Qs, p.dk);
        kr.put(Ks, p.dk);
        vr.put(Vs, dvc);
        if (MODE == 0 && vr.not_finite()) *poison = 1;
        if (c + STEP >= c0 && c + STEP < c1) fetch(c + STEP);
        __syncthreads();
        const float *bh = decays + (c & 1) * 320, *bl = bh + 64, *eb = bl + 64, *wt = eb + 64, *tail = wt + 64;
        const bool poisoned = MODE == 0 && __builtin_amdgcn_readfirstlane(*poison);
        if (MODE == 0) {
            // P[i][j] = scale exp(b_i - b_j) q_i . k_j, j <= i: tiles (it, jt) dealt to the waves
#pragma unroll 1
            for (int t = wave; t < CT * (CT + 1) / 2; t += 4) {
                const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
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
                const f4 hi = *reinterpret_cast<const f4 *>(bh + 16 * it + 4 * gq), li = *reinterpret_cast<const f4 *>(bl + 16 * it + 4 * gq);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * gq + r;
                    Ps[i * PP + j] = j <= i ? acc[r] * p.scale * hw_exp2((hi[r] - hj) + (li[r] - lj)) : 0.0f;
                }
            }
            __syncthreads();
        }
        float vv[CT][4];                         // this wave's columns of v: rows 16 jt + 4 gq + r
#pragma unroll
        for (int jt = 0; jt < CT; ++jt)
#pragma unroll
            for (int r = 0; r < 4; ++r) vv[jt][r] = Vs[(16 * jt + 4 * gq + r) * PV + 16 * wave + l16];
        float eend = tail[0];
        if (MODE == 0) {
            f4 acc[CT];
#pragma unroll
            for (int it = 0; it < CT; ++it) acc[it] = f4{0, 0, 0, 0};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int it = 0; it < CT; ++it) {
                    const f4 x = *reinterpret_cast<const f4 *>(Qs + (16 * it + l16) * PK + 16 * kt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[it] = mfma4(x[r], S[kt][r], acc[it]);
                }
#pragma unroll
            for (int it = 0; it < CT; ++it) acc[it] *= *reinterpret_cast<const f4 *>(eb + 16 * it + 4 * gq);
            if (poisoned) {
                int bad = 0;
#pragma unroll
                for (int jt = 0; jt < CT; ++jt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!__builtin_isfinite(vv[jt][r])) { vv[jt][r] = 0.0f; bad = 1; }
                bad |= __shfl_xor(bad, 16, 64);
                bad |= __shfl_xor(bad, 32, 64);
                if (bad) eend = __builtin_nanf("");
            }
#pragma unroll
            for (int it = 0; it < CT; ++it) {
#pragma unroll
                for (int jt = 0; jt <= it; ++jt) {
                    const f4 x = *reinterpret_cast<const f4 *>(Ps + (16 * it + l16) * PP + 16 * jt + 4 * gq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[it] = mfma4(x[r], vv[jt][r], acc[it]);
                }
            }
            if (poisoned) {
#pragma unroll 1
                for (int j = 0; j < C; ++j) {
                    const float x = Vs[j * PV + 16 * wave + l16];
                    if (__builtin_isfinite(x)) continue;
#pragma unroll
                    for (int it = 0; it < CT; ++it)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j <= 16 * it + 4 * gq + r) acc[it][r] += Ps[(16 * it + 4 * gq + r) * PP + j] * x;
                }
            }
            const RowsOut out(O, nr, ldo);
#pragma unroll
            for (int it = 0; it < CT; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) out.put1(acc[it][r], 16 * it + 4 * gq + r, col, ldo, p.dv);
            O += C * ldo;
        }
        scan(c + STEP);
        fetch_g(c + 2 * STEP);
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] *= eend;
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
            const f4 w = *reinterpret_cast<const f4 *>((MODE == 2 ? eb : wt) + 16 * jt + 4 * gq);
#pragma unroll
            for (int r = 0; r < 4; ++r) vv[jt][r] *= w[r];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t] = mfma4(Ks[(16 * jt + 4 * gq + r) * PK + 16 * t + l16], vv[jt][r], S[t]);
        }
    }
    float *dst = MODE >= 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.last && c1 == nch ? a.last + nh * sz : nullptr;
    if (dst) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = 16 * t + 4 * gq + r;
                if (cok && k < p.dk) dst[k * p.dv + col] = S[t][r];
            }
        if (MODE >= 1 && tid == 0 && vt == 0) a.seg_decay[(long long)slot * p.H + h] = total;
    }
}

// The same walk for bf16 tensors on the bf16 matrix instruction; a workgroup owns all of dv (a wave 16 columns: NW = 4 or 8 waves), the next chunk is in
// flight in registers during the products.  Per chunk: P (weights, to LDS), then for all rows i  O^T = S^T Q^T, scaled by exp(b_i), plus V^T P^T, then
// S += K^T (exp(b_C - b_j) V), with P, S and the weighted V in three bf16 terms: nothing between the inputs and the rounded results has less than 24
// bits.  (Two terms of P and S, which leave 2^-17 of a term, took 245 us for 65536 tokens, 8 heads of 128 x 128, three take 263; 9 prompts of 7121 tokens, 16 heads of
// 64 x 64, 38 and 40.)
// LDS rows are an odd number of 32-byte pieces long: 16-byte direct reads (4 cycles) and transposed ones (2) are then free of bank conflicts (measured
// over pitches of 128 ... 320 bytes); q and P lie in operand order, so a lane's eight values are one read.  P is packed below the diagonal (and q's rows at 64 wide
// keys are half a piece shorter), so that as many workgroups share a CU as with two terms.
template <int DK, int NW, int MODE, bool VEC>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 4 : DK <= 64 ? 3 : 2) void la_fwd_bf16_kernel(const FwdArgs a) {
    constexpr int NT = 64 * NW, C = 64, DV = 16 * NW, KT = DK / 16, KS = DK / 32, QP = 2 * DK + (DK == 64 && NW == 4 ? 16 : 32), KP = 2 * DK + 32,
                  VP = 2 * DV + 32;
    __shared__ __attribute__((aligned(16))) unsigned char lds[C * (KP + VP) + (MODE == 0 ? C * QP + 3 * PAIRS : 0) + 10 * C * 4];
    unsigned char *Ks = lds, *Vs = Ks + C * KP, *Qs = Vs + C * VP, *Ps = Qs + C * QP;
    float *decays = reinterpret_cast<float *>(MODE == 0 ? Ps + 3 * PAIRS : Qs);     // two chunks of: b (two terms), scale exp(b), exp(b_C - b), exp(b_C)
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane0 = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int walks = p.slots * p.H;
    if ((int)blockIdx.x >= walks) {              // packed rows that belong to no sequence: their output is zero
        if (MODE == 0) zero_gaps(p, static_cast<bf16 *>(a.o), (long long)p.H * p.dv, blockIdx.x - walks);
        return;
    }
    int id = xcd_remap(blockIdx.x, walks);       // heads of a group run next to each other on one XCD: they read the same q and k
    const int h = id % p.H; id /= p.H;
    const int slot = id;
    int n, seg;
    walk_of(p, slot, C, n, seg);
    if (seg < 0) return;
    const Seq s = get_seq(p, n);
    const int c0 = seg * p.segc, nch = (s.len + C - 1) / C;
    const int c1 = segment_end(p, seg, nch);
    const bool empty = s.len == 0;
    if (c0 >= c1 && !(empty && seg == 0)) return;
    if (MODE == 1 && c1 == nch) return;          // no segment starts from the last one's end
    if (MODE == 2 && c0 == 0) return;            // (here: from the first one's)
    const int hk = h / (p.H / p.G), first = MODE == 2 ? c1 - 1 : c0;
    const bf16 *Q = static_cast<const bf16 *>(p.q) + s.row * p.qb + (s.start + (long long)c0 * C) * p.ql + hk * p.qh;
    const bf16 *K = static_cast<const bf16 *>(p.k) + s.row * p.kb + (s.start + (long long)first * C) * p.kl + hk * p.kh;
    const bf16 *V = static_cast<const bf16 *>(p.v) + s.row * p.vb + (s.start + (long long)first * C) * p.vl + h * p.vh;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    const long long ldo = (long long)p.H * p.dv, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    bf16 *O = static_cast<bf16 *>(a.o) + ((s.row * p.tokens + s.start + (long long)c0 * C) * p.H + h) * (long long)p.dv;
    const int col = 16 * wave + (lane0 & 15);
    f4 S[KT];
    TileRegs<C, DK, NT, VEC> qr, kr;
    TileRegs<C, DV, NT, VEC> vr;
    qr.init(Q, p.ql, p.dk);
    kr.init(K, p.kl, p.dk);
    vr.init(V, p.vl, p.dv);
    auto rows_of = [&](int c) { const int left = s.len - c * C; return left < C ? left : C; };
    auto fetch = [&](int c) {                    // chunk c, the tensors' pointers at chunk c
        const int nr = rows_of(c);
        if (MODE == 0) qr.load(Q, p.ql, nr, p.dk);
        kr.load(K, p.kl, nr, p.dk);
        vr.load(V, p.vl, nr, p.dv);
    };
    float gr = 0.0f;                             // wave 0: decays, a chunk ahead of the tiles
    auto fetch_g = [&](int c) {
        if (wave == 0 && c >= c0 && c < c1) gr = lane0 < rows_of(c) ? limit_decay(g[((long long)c * C + lane0) * p.gl]) : 0.0f;
    };
    fetch_g(first);
    if (c0 < c1) fetch(first);
    const float *init = MODE >= 1 ? nullptr : segments_of(p, nch) > 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.s0 ? a.s0 + nh * sz : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * t + 4 * (lane0 >> 4) + r;
            S[t][r] = init && col < p.dv && k < p.dk ? init[k * p.dv + col] : 0.0f;
        }
    double total = 0.0;
    f4 *saved = MODE == 0 && a.chunk_states ? reinterpret_cast<f4 *>(a.chunk_states) + ((chunk_base(p, s, n, C) + c0) * p.H + h) * (DK * DV / 4) + wave * KT * 64 + lane0 : nullptr;
    auto scan = [&](int c) {
        if (wave == 0 && c >= c0 && c < c1) {
            float *d = decays + (c & 1) * 5 * C;
            const double b = chunk_decay_scan(gr), bend = lane63(b);
            const float hi = (float)b;
            if (MODE >= 1) total += bend;
            d[lane0] = hi;
            d[C + lane0] = (float)(b - hi);
            d[2 * C + lane0] = hw_exp2(hi) * p.scale;
            d[3 * C + lane0] = hw_exp2((float)(bend - b));
            if (lane0 == 63) d[4 * C] = hw_exp2((float)bend);
        }
    };
    constexpr int STEP = MODE == 2 ? -1 : 1;
    scan(first);
    fetch_g(first + STEP);
    if (MODE == 0 && tid < 128) {                // the tiles of P behind the diagonal that are read with it (32 columns at a time): zero for good
        const int half = tid >> 6, at = pair_row(half, 32 * half + (tid & 15)) + 2 * operand_pos(32 * half + 16 + 4 * ((tid >> 4) & 3));
#pragma unroll
        for (int u = 0; u < 3; ++u) *reinterpret_cast<u32x2 *>(Ps + u * PAIRS + at) = u32x2{0, 0};
    }
    // A NaN or an infinity in v_j times the zero weight of an earlier row would reach that row.  Once one has been met, such values stay out of the
    // products and are added to the rows from j on alone, and their columns of the state become NaN.
    int *poison = reinterpret_cast<int *>(decays + 300);                // (the first chunk's set of decays ends at 257)
    if (MODE == 0 && tid == 0) *poison = 0;
#pragma unroll 1
    for (int c = first; c >= c0 && c < c1; c += STEP) {
        const int nr = rows_of(c);
        if (MODE == 0 && saved) {
#pragma unroll
            for (int t = 0; t < KT; ++t) saved[64 * t] = S[t];
            saved += (long long)p.H * (DK * DV / 4);
        }
        __syncthreads();
        if (MODE == 0) qr.template put<true>(Qs, QP, p.dk);
        kr.put(Ks, KP, p.dk);
        vr.put(Vs, VP, p.dv);
        if (MODE == 0 && vr.not_finite()) *poison = 1;
        Q += C * p.ql; K += STEP * C * p.kl; V += STEP * C * p.vl;
        if (MODE >= 1 && c + STEP >= c0 && c + STEP < c1) fetch(c + STEP);
        const float *bh = decays + (c & 1) * 5 * C, *bl = bh + C, *eb = bl + C, *wt = eb + C, *tail = wt + C;
        __syncthreads();
        const bool poisoned = MODE == 0 && __builtin_amdgcn_readfirstlane(*poison);
        if (MODE == 0) {
            // P[i][j] = scale exp(b_i - b_j) q_i . k_j, j <= i: the ten 16 x 16 tiles are dealt to the waves and worked on side by side (a wave with one
            // less repeats the last one: the same values)
            const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
            constexpr int NTL = (10 + NW - 1) / NW;
            f4 acc[NTL];
#pragma unroll
            for (int n = 0; n < NTL; ++n) {
                const int t = wave + n * NW < 10 ? wave + n * NW : 9, it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
                acc[n] = f4{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) acc[n] = mfma8(frag(Ks, KP, 16 * jt + l16, ks, gq), frag_p(Qs, QP, 16 * it + l16, ks, gq), acc[n]);
            }
#pragma unroll
            for (int n = 0; n < NTL; ++n) {
                const int t = wave + n * NW < 10 ? wave + n * NW : 9, it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
                const int i = 16 * it + l16, j = 16 * jt + 4 * gq;
                const float hi = bh[i], li = bl[i];
                const f4 h4 = *reinterpret_cast<const f4 *>(bh + j), l4 = *reinterpret_cast<const f4 *>(bl + j);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[n][r] = j + r <= i ? acc[n][r] * p.scale * hw_exp2((hi - h4[r]) + (li - l4[r])) : 0.0f;
                put_pairs(Ps + pair_row(it / 2, i) + 2 * operand_pos(j), acc[n]);
            }
            __syncthreads();
        }
        const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
        bf16x8 vf[2];
#pragma unroll
        for (int js = 0; js < 2; ++js) vf[js] = frag_t(Vs, VP, wave, js, lane);
        float eend = tail[0];
        if (MODE == 0) {
            f4 acc[4];
#pragma unroll
            for (int it = 0; it < 4; ++it) acc[it] = f4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 sf[3];
                split8<3>(S[2 * ks], S[2 * ks + 1], sf);
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const bf16x8 q = frag_p(Qs, QP, 16 * it + l16, ks, gq);
#pragma unroll
                    for (int u = 0; u < 3; ++u) acc[it] = mfma8(sf[u], q, acc[it]);
                }
                if (NW == 8) __builtin_amdgcn_sched_barrier(0);
            }
            const RowsOut out(O, nr, ldo);
#pragma unroll
            for (int it = 0; it < 4; ++it) acc[it] *= eb[16 * it + l16];
            if (poisoned) {
                int bad = 0;
#pragma unroll
                for (int js = 0; js < 2; ++js) bad |= finite_only(vf[js]);
                bad |= __shfl_xor(bad, 16, 64);
                bad |= __shfl_xor(bad, 32, 64);
                if (bad) eend = __builtin_nanf("");
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
#pragma unroll
                for (int js = 0; js <= it / 2; ++js) {
#pragma unroll
                    for (int u = 0; u < 3; ++u)
                        acc[it] = mfma8(vf[js], frag_p(Ps + u * PAIRS + pair_row(it / 2, 0), pair_pitch(it / 2), 16 * it + l16, js, gq), acc[it]);
                }
            }
            if (poisoned) {
#pragma unroll 1
                for (int j = 0; j < C; ++j) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(Vs + j * VP + 2 * (16 * wave + 4 * gq));
                    const f2 x0 = bf16pair_to_f2(x.x), x1 = bf16pair_to_f2(x.y);
                    const float v[4] = {x0.x, x0.y, x1.x, x1.y};
                    const int at = 2 * (operand_pos(j & ~3) + (j & 3));
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        if (j > 16 * it + l16) continue;
                        const float w = get_pair(Ps + pair_row(it / 2, 16 * it + l16) + at);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!__builtin_isfinite(v[r])) acc[it][r] += w * v[r];
                    }
                }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) out.template put4<VEC>(O, 16 * it + l16, 16 * wave + 4 * gq, ldo, p.dv, acc[it]);
            O += C * ldo;
        }
        __builtin_amdgcn_sched_barrier(0);
        if (MODE == 0 && c + 1 < c1) fetch(c + 1);   // in flight during the state's products; earlier, its registers would cost a workgroup a CU
        scan(c + STEP);
        fetch_g(c + 2 * STEP);
        bf16x8 vw[2][3];
#pragma unroll
        for (int js = 0; js < 2; ++js) {
            const float *w = MODE == 2 ? eb : wt;
            const f4 w0 = *reinterpret_cast<const f4 *>(w + 32 * js + 4 * gq), w1 = *reinterpret_cast<const f4 *>(w + 32 * js + 16 + 4 * gq);
            f4 x, y;
            widen8(vf[js], x, y);
            split8<3>(x * w0, y * w1, vw[js]);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            S[t] *= eend;
#pragma unroll
            for (int js = 0; js < 2; ++js) {
                const bf16x8 k = frag_t(Ks, KP, t, js, lane);
#pragma unroll
                for (int u = 0; u < 3; ++u) S[t] = mfma8(k, vw[js][u], S[t]);
            }
        }
    }
    float *dst = MODE >= 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.last && c1 == nch ? a.last + nh * sz : nullptr;
    if (dst) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = 16 * t + 4 * (lane0 >> 4) + r;
                if (col < p.dv && k < p.dk) dst[k * p.dv + col] = S[t][r];
            }
        if (MODE >= 1 && tid == 0) a.seg_decay[(long long)slot * p.H + h] = total;
    }
}

// joins the segments of a (sequence, head): seg_states[slot] = state in front of the segment; one thread W state elements
template <int W>
__global__ __launch_bounds__(NT) void la_join_fwd_kernel(const FwdArgs a, int C) {
    typedef typename Elements<W>::type V;
    const Problem &p = a.p;
    const long long sz = (long long)p.dk * p.dv;
    const int tiles = (int)((sz + NT * W - 1) / (NT * W)), nh = blockIdx.x / tiles, n = nh / p.H;
    const long long e = ((long long)(blockIdx.x % tiles) * NT + threadIdx.x) * W;
    const Seq s = get_seq(p, n);
    const int ns = segments_of(p, (s.len + C - 1) / C);
    if (e >= sz || ns <= 1) return;
    const auto at = [](float *q) -> V & { return *reinterpret_cast<V *>(q); };
    V v = V{};
    if (a.s0) v = *reinterpret_cast<const V *>(a.s0 + nh * sz + e);
    const long long first = (long long)first_slot(p, n, C) * p.H + nh % p.H, step = p.H * sz;
    float *u = a.seg_states + first * sz + e;
    const double *d = a.seg_decay + first;
    for (int i = 0; i < ns; i += 8) {                       // eight segments' loads are in flight at once
        V own[8];
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = i + j < ns - 1 ? i + j : ns - 2;  // (the last segment's contribution is not there, and not used)
            own[j] = at(u + k * step);
            f[j] = hw_exp2((float)d[(long long)k * p.H]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i + j < ns) {
                at(u + (i + j) * step) = v;
                v = v * f[j] + own[j];
            }
        }
    }
}

template <int MODE, bool VEC, int DK, int C>
void launch_f32(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    const unsigned walks = (unsigned)((long long)a.p.slots * a.p.H * ((a.p.dv + 63) / 64));
    ss2d_launch((la_fwd_kernel<DK, C, MODE, VEC>), dim3(walks + gaps), dim3(NT), 0, s, a);
}
template <int MODE, bool VEC>
void dispatch_f32(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    const int dk = a.p.dk;
    const bool c64 = linattn_chunk(SS2D_DTYPE_F32, a.p.dk, a.p.dv) == 64;
    if (dk <= 16) c64 ? launch_f32<MODE, VEC, 16, 64>(a, gaps, s) : launch_f32<MODE, VEC, 16, 32>(a, gaps, s);
    else if (dk <= 64) c64 ? launch_f32<MODE, VEC, 64, 64>(a, gaps, s) : launch_f32<MODE, VEC, 64, 32>(a, gaps, s);
    else launch_f32<MODE, VEC, 128, 32>(a, gaps, s);
}
template <int MODE, bool VEC, int DK, int NW>
void launch_bf16(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    ss2d_launch((la_fwd_bf16_kernel<DK, NW, MODE, VEC>), dim3((unsigned)((long long)a.p.slots * a.p.H) + gaps), dim3(64 * NW), 0, s, a);
}
template <int MODE, bool VEC>
void dispatch_bf16(const FwdArgs &a, unsigned gaps, hipStream_t s) {
    const int dk = a.p.dk;
    if (a.p.dv <= 64) {
        if (dk <= 32) launch_bf16<MODE, VEC, 32, 4>(a, gaps, s);
        else if (dk <= 64) launch_bf16<MODE, VEC, 64, 4>(a, gaps, s);
        else launch_bf16<MODE, VEC, 128, 4>(a, gaps, s);
    } else {
        if (dk <= 32) launch_bf16<MODE, VEC, 32, 8>(a, gaps, s);
        else if (dk <= 64) launch_bf16<MODE, VEC, 64, 8>(a, gaps, s);
        else launch_bf16<MODE, VEC, 128, 8>(a, gaps, s);
    }
}
template <int MODE>
void dispatch(int dtype, const FwdArgs &a, unsigned gaps, hipStream_t s) {
    if (dtype == SS2D_DTYPE_F32) a.p.vec ? dispatch_f32<MODE, true>(a, gaps, s) : dispatch_f32<MODE, false>(a, gaps, s);
    else a.p.vec ? dispatch_bf16<MODE, true>(a, gaps, s) : dispatch_bf16<MODE, false>(a, gaps, s);
}

}  // namespace

void linattn_segment_pass(int dtype, const linattn::Problem &p, float *seg_states, double *seg_decay, bool reverse, hipStream_t s) {
    FwdArgs a{};
    a.p = p; a.seg_states = seg_states; a.seg_decay = seg_decay;
    reverse ? dispatch<2>(dtype, a, 0, s) : dispatch<1>(dtype, a, 0, s);
}

extern "C" int ss2d_linattn_chunk(int dtype, int dk, int dv) { return linattn_chunk(dtype, dk, dv); }
extern "C" long long ss2d_linattn_state_floats(int dtype, int dk, int dv) { return linattn_state_floats(dtype, dk, dv); }
extern "C" long long ss2d_linattn_segments(int dtype, long long all_tokens, long long max_len, int H, int dk, int dv, int backward) {
    return all_tokens >= 0 && max_len >= 0 && H > 0 ? linattn_segments(dtype, all_tokens, max_len, H, dk, dv, backward) : 1LL << 32 | 1;
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
    hipStream_t s = (hipStream_t)stream;
    if (nseg > 1) {
        linattn_segment_pass(dtype, a.p, seg_states, seg_decay, false, s);
        const int C = linattn_chunk(dtype, dk, dv), w = dk * dv % 4 == 0 ? 4 : 1;
        const dim3 grid((unsigned)((dk * dv + NT * w - 1) / (NT * w) * N * H));
        if (w == 4) ss2d_launch(la_join_fwd_kernel<4>, grid, dim3(NT), 0, s, a, C);
        else ss2d_launch(la_join_fwd_kernel<1>, grid, dim3(NT), 0, s, a, C);
    }
    dispatch<0>(dtype, a, gaps, s);
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("linattn_fwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
