// Linear attention with a decay for each head, backward, for gfx950 (forward: ss2d_linattn_fwd.hip, formulas: ss2d_linattn.h).
//
// With D the gradient of the state behind a chunk, S the state in front of it (left by the forward), w_ij = scale exp(b_i - b_j) for
// j <= i (else 0), X_ij = w_ij q_i . k_j and Y_ij = w_ij do_i . v_j:
//   dq_i = sum_j Y_ij k_j + scale exp(b_i) S do_i          dk_j = sum_i Y_ij q_i + exp(b_C - b_j) D v_j
//   dv_j = sum_i X_ij do_i + exp(b_C - b_j) D^T k_j        D_prev = exp(b_C) D + sum_i scale exp(b_i) q_i do_i^T
// A decay g_t scales every path that crosses it, so its gradient is the sum over the pairs on both sides of it,
//   dg_t = sum_{i >= t > j} M_ij,  M_ij = w_ij (q_i . k_j)(do_i . v_j),
// with the state in front of the chunk as one more column, D as one more row.  Only pairs that cross t are added, none is taken off again: behind a
// strong decay exp(g_t) all of them are small, and the others, a factor exp(-g_t) larger, would leave their rounding (as row sums minus column sums in fp32 the
// gradient of a decay of log(1e-6) between chunks of ordinary ones was off by its own size).  For a 16 x 16 tile of M the tokens of its rows take sums of its rows
// from the end, the tokens of its columns sums of its columns from the start, the tokens between them its total; a tile on the diagonal a scan in both
// directions; the pairs with S (q . S do) count as rows, those with D (k . D v) as columns, <D, S> for every token.  One decay for all tokens of a head (token
// stride 0) has the sum over t for its gradient; a chunk's part is left at its first token.
//
// A workgroup walks one segment of one sequence and value head from its end to its start with D in accumulator registers (a wave owns
// 16-column slices of dv).  Segments as in the forward: own contributions, a join in order, the walk.
//
// Measured.  4 x 4096 tokens, 16 heads of 128 x 64 on 2 key heads, bf16: contributions 30 us, join 5.5, walk 182, sum over the heads of a group 47 (5.7 TB/s).  A
// chunk takes a workgroup of 16 waves, one a CU (159 KB of LDS), 24,000 cycles: the matrix units are busy 19% of them and LDS 49% (a third of that bank
// conflicts, most of 8-byte writes), the rest waits between the phases, which need each other's results.  24 x 3136 tokens, 3 heads of 16 x 64 fp32: 15.5 + 5 + 91 us
// (matrix units 39%, LDS 28%).
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

// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_mov<DPP_ROW_ROR(8), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(4), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(2), 0xf, false>(0.0f, v);
    v += dpp_mov<DPP_ROW_ROR(1), 0xf, false>(0.0f, v);
    return v;
}

// ---- the gradients of the decays: a lane is a token of the chunk (lane = 16 gq + l16, tile gq) and adds the pairs that cross it
// sums over the 16 lanes of a DPP row from its end, from its start; lane N of the row in every lane of it
__device__ __forceinline__ float row16_from_end(float v) {
    v += dpp_mov<DPP_ROW_SHL(1), 0xf, true>(0.0f, v);
    v += dpp_mov<DPP_ROW_SHL(2), 0xf, true>(0.0f, v);
    v += dpp_mov<DPP_ROW_SHL(4), 0xf, true>(0.0f, v);
    return v + dpp_mov<DPP_ROW_SHL(8), 0xf, true>(0.0f, v);
}
__device__ __forceinline__ float row16_from_start(float v) {
    v += dpp_mov<DPP_ROW_SHR(1), 0xf, true>(0.0f, v);
    v += dpp_mov<DPP_ROW_SHR(2), 0xf, true>(0.0f, v);
    v += dpp_mov<DPP_ROW_SHR(4), 0xf, true>(0.0f, v);
    return v + dpp_mov<DPP_ROW_SHR(8), 0xf, true>(0.0f, v);
}
__device__ __forceinline__ float row16_shift(float v) { return dpp_mov<DPP_ROW_SHR(1), 0xf, true>(0.0f, v); }      // of the lane before, 0 in the first
template <int N>
__device__ __forceinline__ float row16_lane(float v) { return dpp_mov<0x150 + N, 0xf, false>(0.0f, v); }
__device__ __forceinline__ float rows_sum(float v) {                 // over the four rows of 16 lanes
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// Four values a lane, of indices 4 gq + r, alike in all l16: sums in every row from index l16 on, up to and with it, in front of it
__device__ __forceinline__ float four_from(const f4 &v, int l16, int gq) {
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += 4 * gq + r >= l16 ? v[r] : 0.0f;
    return rows_sum(s);
}
__device__ __forceinline__ float four_up_to(const f4 &v, int l16, int gq) {
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += 4 * gq + r <= l16 ? v[r] : 0.0f;
    return rows_sum(s);
}
__device__ __forceinline__ float four_before(const f4 &v, int l16, int gq) {
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += 4 * gq + r < l16 ? v[r] : 0.0f;
    return rows_sum(s);
}
// of a tile's row sums from the end (rows): the tokens of the tile take theirs, those of earlier tiles the whole
__device__ __forceinline__ float cross_rows(float from_end, int tile, int gq) {
    const float all = row16_lane<0>(from_end);
    return gq < tile ? all : gq == tile ? from_end : 0.0f;
}
// of a tile's column sums from the start: the tokens of the tile take the columns before them, those of later tiles the whole
__device__ __forceinline__ float cross_columns(float from_start, int tile, int gq) {
    const float all = row16_lane<15>(from_start), before = row16_shift(from_start);
    return gq > tile ? all : gq == tile ? before : 0.0f;
}
// of a tile below the diagonal: row sums from the end for its rows' tokens, columns before them for its columns' tokens, the total between
__device__ __forceinline__ float cross_tile(float rows_from_end, float columns_before, int it, int jt, int gq) {
    const float all = row16_lane<0>(rows_from_end);
    return gq == it ? rows_from_end : gq == jt ? columns_before : gq > jt && gq < it ? all : 0.0f;
}

// ---- values that are not finite.  In dq = Y k, dk = Y^T q and dv = X^T dout a NaN or an infinity would meet the zero weights beyond the diagonal and so
// reach rows that do not depend on its own.  In a chunk that holds one they stay out of the products and are added to the rows they belong to alone.
__device__ __forceinline__ float finite_or_0(float x) { return __builtin_isfinite(x) ? x : 0.0f; }
// column c of a tile of `rows` rows: add(row, value) for each value that is not finite
template <typename F>
__device__ __forceinline__ void each_not_finite(const float *column, int pitch, int rows, F add) {
#pragma unroll 1
    for (int t = 0; t < rows; ++t) {
        const float x = column[t * pitch];
        if (!__builtin_isfinite(x)) add(t, x);
    }
}
// the same for four columns of bf16: add(row, r, value)
template <typename F>
__device__ __forceinline__ void each_not_finite4(const unsigned char *columns, int pitch, int rows, F add) {
#pragma unroll 1
    for (int t = 0; t < rows; ++t) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(columns + t * pitch);
        const f2 a = bf16pair_to_f2(w.x), b = bf16pair_to_f2(w.y);
        const float x[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (!__builtin_isfinite(x[r])) add(t, r, x[r]);
    }
}

// seg_states[slot] = D behind the segment; one thread W elements
template <int W>
__global__ __launch_bounds__(NT) void la_join_bwd_kernel(const BwdArgs a, int C) {
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
    if (a.dlast) v = *reinterpret_cast<const V *>(a.dlast + nh * sz + e);
    const long long first = (long long)first_slot(p, n, C) * p.H + nh % p.H, step = p.H * sz;
    float *u = a.seg_states + first * sz + e;
    const double *d = a.seg_decay + first;
    for (int i = ns - 1; i >= 0; i -= 8) {
        V own[8];
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = i - j > 1 ? i - j : 1;             // (the first segment's contribution is not there, and not used)
            own[j] = at(u + k * step);
            f[j] = hw_exp2((float)d[(long long)k * p.H]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i - j >= 0) {
                at(u + (i - j) * step) = v;
                v = v * f[j] + own[j];
            }
        }
    }
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

// fp32: 16 waves a workgroup, so that every result of a chunk -- dq, dk (C x dk) and dv (C x dv) -- is at most one 16 x 16 tile a wave on
// v_mfma_f32_16x16x4_f32; keys up to 16 wide: 8 waves with two tiles of dv, and two workgroups a CU (24 x 3136 tokens, 3 heads of 16 x 64: 96 us, one
// workgroup of 16 waves 120).  A lane holds row / column l16 of an operand and contracted indices 4 gq + r of a 16-block in step r: direct operands are
// 16-byte LDS reads, transposed ones four 4-byte reads, both free of bank conflicts at a pitch of 4 mod 16 floats.  LDS holds the four tiles, X,
// Y and one state at a time: S (for dq), then D (for dk, dv).  The next chunk is in flight in registers.
template <int DK, int DV, int C, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW, 4) void la_bwd_kernel(const BwdArgs a) {
    constexpr int NT = 64 * NW, PK = DK + 4, PV = DV + 4, PP = 20, KT = DK / 16, VT = DV / 16, CT = C / 16;
    constexpr int TW = (KT * VT + NW - 1) / NW;                      // tiles of D a wave owns: wave + NW m
    constexpr int XY = CT * (CT + 1) / 2 * 16 * PP;                  // X, Y: their tiles up to the diagonal
    constexpr int NV = (VT * CT + NW - 1) / NW;                      // tiles of dv a wave owns
    static_assert(KT * CT <= NW && NV <= 2, "tiles of a wave");
    __shared__ __attribute__((aligned(16))) float lds[2 * C * PK + 2 * C * PV + DK * PV + 2 * XY + 10 * 64 + NW * 64 + NW + 4];
    float *Qs = lds, *Ks = Qs + C * PK, *Vs = Ks + C * PK, *Os = Vs + C * PV, *St = Os + C * PV, *Xs = St + DK * PV, *Ys = Xs + XY;
    float *decays = Ys + XY, *parts = decays + 10 * 64, *corners = parts + NW * 64;
    int *poison = reinterpret_cast<int *>(corners + NW);             // the last chunk that held a NaN or an infinity in q, k or dout
    const auto tile_at = [](int it, int jt) { return (it * (it + 1) / 2 + jt) * 16 * PP; };
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane0 = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int walks = p.slots * p.H;
    const int hq = p.H > p.G ? p.H : p.G;                            // heads of dq / dk as written
    if ((int)blockIdx.x >= walks) {                                  // packed rows that belong to no sequence
        const int w = (int)blockIdx.x - walks;
        zero_rows(p, static_cast<float *>(a.dq), (long long)hq * p.dk, w, GAP_WGS);
        zero_rows(p, static_cast<float *>(a.dk_), (long long)hq * p.dk, w, GAP_WGS);
        zero_rows(p, static_cast<float *>(a.dv_), (long long)p.H * p.dv, w, GAP_WGS);
        zero_rows(p, a.dg, p.H, w, GAP_WGS);
        return;
    }
    int id = xcd_remap(blockIdx.x, walks);
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
    const int hk = h / (p.H / p.G);
    const long long ldv = (long long)p.H * p.dv, ldq = (long long)hq * p.dk, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    const long long t0 = s.row * p.tokens + s.start, e0 = (long long)(c1 - 1) * C;              // the tensors' pointers start at the last chunk
    const float *Q = static_cast<const float *>(p.q) + s.row * p.qb + (s.start + e0) * p.ql + hk * p.qh;
    const float *K = static_cast<const float *>(p.k) + s.row * p.kb + (s.start + e0) * p.kl + hk * p.kh;
    const float *V = static_cast<const float *>(p.v) + s.row * p.vb + (s.start + e0) * p.vl + h * p.vh;
    const float *DO = static_cast<const float *>(a.dout) + ((t0 + e0) * p.H + h) * (long long)p.dv;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    float *DQ = static_cast<float *>(a.dq) + ((t0 + e0) * hq + h) * (long long)p.dk;
    float *DKp = static_cast<float *>(a.dk_) + ((t0 + e0) * hq + h) * (long long)p.dk;
    float *DVp = static_cast<float *>(a.dv_) + ((t0 + e0) * p.H + h) * (long long)p.dv;
    float *DG = a.dg + t0 * p.H + h;
    // one tile of dq and dk at most; the last waves take them first, the first waves the scores
    const int wq = NW - 1 - wave, qk = wq % KT, qi = wq / KT, vt = wave % VT;
    const bool has_q = wq < KT * CT, has_v = wave < VT * CT;
    auto state_at = [&](int m, int r, int ln) {                      // element (t, r) of this lane's part of a state: row k, column dv; -1: outside
        const int t = wave + NW * m, k = 16 * (t / VT) + 4 * (ln >> 4) + r, c = 16 * (t % VT) + (ln & 15);
        return t < KT * VT && k < p.dk && c < p.dv ? k * p.dv + c : -1;
    };
    f4 D[TW], sr[TW];
    {
        const float *init = segments_of(p, nch) > 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.dlast ? a.dlast + nh * sz : nullptr;
#pragma unroll
        for (int m = 0; m < TW; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int o = state_at(m, r, lane0);
                D[m][r] = init && o >= 0 ? init[o] : 0.0f;
            }
    }
    TileRegsF<C, DK, PK, NT, VEC> qr, kr;
    TileRegsF<C, DV, PV, NT, VEC> vr, orr;
    qr.init(p.ql, p.dk);
    kr.init(p.kl, p.dk);
    vr.init(p.vl, p.dv);
    orr.init(ldv, p.dv);
    const float *saved = a.chunk_states + ((chunk_base(p, s, n, C) + c1 - 1) * p.H + h) * sz;
    auto rows_of = [&](int c) { const int left = s.len - c * C; return left < C ? left : C; };
    auto fetch = [&](int c) {
        const int nr = rows_of(c), ln = fresh(lane0);
        qr.load(Q, p.ql, nr, p.dk);
        kr.load(K, p.kl, nr, p.dk);
        vr.load(V, p.vl, nr, p.dv);
        orr.load(DO, ldv, nr, p.dv);
#pragma unroll
        for (int m = 0; m < TW; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int o = state_at(m, r, ln);
                const float x = saved[o >= 0 ? o : 0];
                sr[m][r] = o >= 0 ? x : 0.0f;
            }
    };
    float gr = 0.0f;
    auto fetch_g = [&](int c) {
        if (wave == 0 && c >= c0) gr = lane0 < rows_of(c) ? limit_decay(g[((long long)c * C + lane0) * p.gl]) : 0.0f;
    };
    auto scan = [&](int c) {                                         // two chunks of: b (two terms), scale exp(b), exp(b_C - b), exp(b_C)
        if (wave == 0 && c >= c0) {
            float *d = decays + (c & 1) * 5 * 64;
            const double b = chunk_decay_scan(gr), bend = lane63(b);
            const float hi = (float)b;
            d[lane0] = hi;
            d[64 + lane0] = (float)(b - hi);
            d[128 + lane0] = hw_exp2(hi) * p.scale;
            d[192 + lane0] = hw_exp2((float)(bend - b));
            if (lane0 == 63) d[256] = hw_exp2((float)bend);
        }
    };
    auto finish_dg = [&](int c) {                                    // behind a barrier after chunk c: the waves' parts of its decays' gradients
        if (wave == 1) {
            double x = 0.0;
#pragma unroll
            for (int w = 0; w < NW; ++w) x += (double)parts[w * 64 + lane0] + (double)corners[w];
            if (p.gl == 0) {                                         // one decay for all tokens
                if (lane0 >= rows_of(c)) x = 0.0;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
                if (lane0) x = 0.0;
            }
            if (lane0 < rows_of(c)) DG[((long long)c * C + lane0) * p.H] = (float)x;
        }
    };
    auto put_state = [&](const f4 (&x)[TW]) {
        const int ln = fresh(lane0);
#pragma unroll
        for (int m = 0; m < TW; ++m) {
            const int t = wave + NW * m;
            if (t < KT * VT) {
#pragma unroll
                for (int r = 0; r < 4; ++r) St[(16 * (t / VT) + 4 * (ln >> 4) + r) * PV + 16 * (t % VT) + (ln & 15)] = x[m][r];
            }
        }
    };
    auto dot4 = [&](const f4 &x, const f4 &y, f4 acc) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc = mfma4(x[r], y[r], acc);
        return acc;
    };
    fetch_g(c1 - 1);
    scan(c1 - 1);
    fetch_g(c1 - 2);
    if (c0 < c1) fetch(c1 - 1);
    if (tid == 0) *poison = -1;
#pragma unroll 1
    for (int c = c1 - 1; c >= c0; --c) {
        const int nr = rows_of(c);
        const float *bh = decays + (c & 1) * 5 * 64, *bl = bh + 64, *eb = bl + 64, *wt = eb + 64, *tail = wt + 64;
        __syncthreads();
        if (c + 1 < c1) finish_dg(c + 1);
        qr.put(Qs, p.dk);
        kr.put(Ks, p.dk);
        vr.put(Vs, p.dv);
        orr.put(Os, p.dv);
        if (qr.not_finite() || kr.not_finite() || orr.not_finite()) *poison = c;
        put_state(sr);
        float corner = 0.0f;                                         // <D, S>
#pragma unroll
        for (int m = 0; m < TW; ++m) corner += (sr[m].x * D[m].x + sr[m].y * D[m].y) + (sr[m].z * D[m].z + sr[m].w * D[m].w);
        Q -= C * p.ql; K -= C * p.kl; V -= C * p.vl; DO -= C * ldv; saved -= p.H * sz;
        if (c > c0) fetch(c - 1);
        __syncthreads();
        const bool poisoned = __builtin_amdgcn_readfirstlane(*poison) == c;
        const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
        float cross = 0.0f;                                          // what this wave's pairs add to the decay of token `lane`
        // X, Y and the sums of M below the diagonal
#pragma unroll 1
        for (int t = wave; t < CT * (CT + 1) / 2; t += NW) {
            const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
            f4 x = f4{0, 0, 0, 0}, y = f4{0, 0, 0, 0};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
                x = dot4(*reinterpret_cast<const f4 *>(Qs + (16 * it + l16) * PK + 16 * kt + 4 * gq), *reinterpret_cast<const f4 *>(Ks + (16 * jt + l16) * PK + 16 * kt + 4 * gq), x);
#pragma unroll
            for (int v = 0; v < VT; ++v)
                y = dot4(*reinterpret_cast<const f4 *>(Os + (16 * it + l16) * PV + 16 * v + 4 * gq), *reinterpret_cast<const f4 *>(Vs + (16 * jt + l16) * PV + 16 * v + 4 * gq), y);
            const int j = 16 * jt + l16;
            const float hj = bh[j], lj = bl[j];
            const f4 hi = *reinterpret_cast<const f4 *>(bh + 16 * it + 4 * gq), li = *reinterpret_cast<const f4 *>(bl + 16 * it + 4 * gq);
            f4 m;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * gq + r;
                const float w = p.scale * hw_exp2((hi[r] - hj) + (li[r] - lj));
                const float yw = j <= i ? y[r] * w : 0.0f;
                Xs[16 * PP * t + (4 * gq + r) * PP + l16] = j <= i ? x[r] * w : 0.0f;
                Ys[16 * PP * t + (4 * gq + r) * PP + l16] = yw;
                m[r] = j < i ? x[r] * yw : 0.0f;
            }
            if (it == jt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) m[r] = row16_shift(row16_from_start(m[r]));      // of row i, the columns in front of token l16
                const float d = four_from(m, l16, gq);
                cross += gq == it ? d : 0.0f;
            } else {
                const float columns = row16_shift(row16_from_start(rows_sum((m.x + m.y) + (m.z + m.w))));
#pragma unroll
                for (int r = 0; r < 4; ++r) m[r] = row16_sum(m[r]);
                cross += cross_tile(four_from(m, l16, gq), columns, it, jt, gq);
            }
        }
        const int k = 16 * qk + l16;
        f4 dq = f4{0, 0, 0, 0};
        if (has_q) {
#pragma unroll
            for (int v = 0; v < VT; ++v)
                dq = dot4(*reinterpret_cast<const f4 *>(Os + (16 * qi + l16) * PV + 16 * v + 4 * gq), *reinterpret_cast<const f4 *>(St + k * PV + 16 * v + 4 * gq), dq);
            dq *= *reinterpret_cast<const f4 *>(eb + 16 * qi + 4 * gq);
            f4 d;                                                    // pairs with the state in front of the chunk
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = row16_sum(dq[r] * Qs[(16 * qi + 4 * gq + r) * PK + k]);
            cross += cross_rows(four_from(d, l16, gq), qi, gq);
        }
        __syncthreads();                                              // X, Y are there; S is done with
        put_state(D);
        if (has_q) {
            for (int jt = 0; jt <= qi; ++jt) {
                f4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = Ks[(16 * jt + 4 * gq + r) * PK + k];
                if (poisoned) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = finite_or_0(y[r]);
                }
                dq = dot4(*reinterpret_cast<const f4 *>(Ys + tile_at(qi, jt) + l16 * PP + 4 * gq), y, dq);
            }
            if (poisoned)
                each_not_finite(Ks + k, PK, 16 * qi + 16, [&](int j, float x) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (j <= 16 * qi + 4 * gq + r) dq[r] += Ys[tile_at(qi, j >> 4) + (4 * gq + r) * PP + (j & 15)] * x;
                });
            const RowsOut out(DQ, nr, ldq);
#pragma unroll
            for (int r = 0; r < 4; ++r) out.put1(dq[r], 16 * qi + 4 * gq + r, k, ldq, p.dk);
        }
        __syncthreads();                                              // D is there
        const float eend = tail[0];
        if (has_q) {
            f4 dk = f4{0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < VT; ++v)
                dk = dot4(*reinterpret_cast<const f4 *>(Vs + (16 * qi + l16) * PV + 16 * v + 4 * gq), *reinterpret_cast<const f4 *>(St + k * PV + 16 * v + 4 * gq), dk);
            dk *= *reinterpret_cast<const f4 *>(wt + 16 * qi + 4 * gq);
            f4 d;                                                    // pairs with D
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = row16_sum(dk[r] * Ks[(16 * qi + 4 * gq + r) * PK + k]);
            cross += cross_columns(four_up_to(d, l16, gq), qi, gq);
            for (int it = qi; it < CT; ++it) {
                f4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = Ys[tile_at(it, qi) + (4 * gq + r) * PP + l16];
                    y[r] = Qs[(16 * it + 4 * gq + r) * PK + k];
                }
                if (poisoned) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = finite_or_0(y[r]);
                }
                dk = dot4(x, y, dk);
            }
            if (poisoned)
                each_not_finite(Qs + k, PK, C, [&](int i, float x) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i >= 16 * qi + 4 * gq + r) dk[r] += Ys[tile_at(i >> 4, qi) + (i & 15) * PP + 4 * gq + r] * x;
                });
            const RowsOut out(DKp, nr, ldq);
#pragma unroll
            for (int r = 0; r < 4; ++r) out.put1(dk[r], 16 * qi + 4 * gq + r, k, ldq, p.dk);
        }
        parts[wave * 64 + lane] = cross;
        corner = lanes_sum<64>(corner * eend);
        if (lane == 0) corners[wave] = corner;
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            if (!has_v) break;
            const int vj = m ? CT - 1 - wave / VT : wave / VT, col = 16 * vt + l16;      // a long column of products with a short one
            f4 dv = f4{0, 0, 0, 0};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                f4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = St[(16 * kt + 4 * gq + r) * PV + col];
                dv = dot4(*reinterpret_cast<const f4 *>(Ks + (16 * vj + l16) * PK + 16 * kt + 4 * gq), y, dv);
            }
            dv *= *reinterpret_cast<const f4 *>(wt + 16 * vj + 4 * gq);
            for (int it = vj; it < CT; ++it) {
                f4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = Xs[tile_at(it, vj) + (4 * gq + r) * PP + l16];
                    y[r] = Os[(16 * it + 4 * gq + r) * PV + col];
                }
                if (poisoned) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = finite_or_0(y[r]);
                }
                dv = dot4(x, y, dv);
            }
            if (poisoned)
                each_not_finite(Os + col, PV, C, [&](int i, float x) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i >= 16 * vj + 4 * gq + r) dv[r] += Xs[tile_at(i >> 4, vj) + (i & 15) * PP + 4 * gq + r] * x;
                });
            const RowsOut out(DVp, nr, ldv);
#pragma unroll
            for (int r = 0; r < 4; ++r) out.put1(dv[r], 16 * vj + 4 * gq + r, col, ldv, p.dv);
        }
        DQ -= C * ldq; DKp -= C * ldq; DVp -= C * ldv;
        scan(c - 1);
        fetch_g(c - 2);
#pragma unroll
        for (int m = 0; m < TW; ++m) {
            const int t = wave + NW * m;
            if (t >= KT * VT) break;
            D[m] *= eend;
#pragma unroll
            for (int it = 0; it < CT; ++it) {
                f4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = Qs[(16 * it + 4 * gq + r) * PK + 16 * (t / VT) + l16];
                    y[r] = Os[(16 * it + 4 * gq + r) * PV + 16 * (t % VT) + l16];
                }
                D[m] = dot4(x, y * *reinterpret_cast<const f4 *>(eb + 16 * it + 4 * gq), D[m]);
            }
        }
    }
    __syncthreads();
    if (c0 < c1) finish_dg(c0);
    if (a.ds0 && c0 == 0) {
        float *d = a.ds0 + nh * sz;
#pragma unroll
        for (int m = 0; m < TW; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int o = state_at(m, r, lane0);
                if (o >= 0) d[o] = D[m][r];
            }
    }
}

// The same walk for bf16 tensors on the bf16 matrix instruction: chunks of 64, 16 waves a workgroup (dk <= 32 and 64 x 64: 8).  LDS holds the four tiles, X and Y packed
// below the diagonal and the terms of ONE state at a time, transposed (dv x dk): first S (for dq), then D (for dk and dv); with NB = 1 (64 x 64, 128 x 128) one
// term at a time.  X, Y, S and D all enter in three terms: nothing between the inputs and the rounded gradients has less than 24 bits (two terms of X, Y, and of D in
// dv, which leave 2^-17 of a term, took 356 us for 4 x 4096 tokens, 16 heads of 128 x 64, forward and backward, three take 371; of 64 x 64, 208 and 212).
// Direct operands are eight values in a row (one 16-byte LDS read); what they are multiplied with, where it is read transposed, takes its contracted
// rows in the same order (frag_tc).  Products of two transposed operands (over tokens) use frag_t for both.
//
// Up to 64 x 64 two workgroups of eight waves share a CU, so that one works while the other waits at its barriers: X waits in registers until dk is done with Y
// and takes its place, and at 64 x 64 rows are half a pitch step shorter and a state's terms take turns (with two terms of X and Y, 24 x 3136 tokens,
// 3 heads of 16 x 64, forward and backward: 142 us with one workgroup of eight waves a CU, 123 with two; 4 x 4096, 16 heads of 64 x 64: 220 with one of sixteen, 208
// with two of eight; three terms then 212).
template <int DK, int DV, int NW, bool VEC, typename QT>
__global__ __launch_bounds__(64 * NW, DK <= 64 && DV <= 64 ? 4 : NW / 4) void la_bwd_bf16_kernel(const BwdArgs a) {
    constexpr int NT = 64 * NW, C = 64, KT = DK / 16, KS = DK / 32, VT = DV / 16, VS = DV / 32;
    constexpr bool TURNS = DK <= 64 && DV <= 64, TIGHT = DK == 64 && DV == 64;
    constexpr int QP = 2 * DK + (TIGHT ? 16 : 32), VP = 2 * DV + (TIGHT ? 16 : 32), SP = 2 * DK + 16;      // bytes a row
    constexpr int NB = TIGHT || (DK == 128 && DV == 128) ? 1 : 3;                                      // terms of a state in LDS at once
    constexpr int NI = 4 * KT / NW, NJ = 4 * VT / NW, TW = KT * VT / NW;                               // tiles of a wave: rows of dq / dk, rows of dv, D
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * C * QP + 2 * C * VP + (TURNS ? 3 : 6) * PAIRS + NB * DV * SP + (10 * C + NW * C + NW + 4) * 4];
    unsigned char *Qs = lds, *Ks = Qs + C * QP, *Vs = Ks + C * QP, *Os = Vs + C * VP, *Ys = Os + C * VP,
                  *Xs = TURNS ? Ys : Ys + 3 * PAIRS, *St = Xs + 3 * PAIRS;
    float *decays = reinterpret_cast<float *>(St + NB * DV * SP), *parts = decays + 10 * C, *corners = parts + NW * C;
    int *poison = reinterpret_cast<int *>(corners + NW);             // the last chunk that held a NaN or an infinity in q, k or dout
    const Problem &p = a.p;
    const int tid = threadIdx.x, lane0 = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int walks = p.slots * p.H;
    const int hq = p.H > p.G ? p.H : p.G;                            // heads of dq / dk as written
    if ((int)blockIdx.x >= walks) {                                  // packed rows that belong to no sequence
        const int w = (int)blockIdx.x - walks;
        zero_rows(p, static_cast<QT *>(a.dq), (long long)hq * p.dk, w, GAP_WGS);
        zero_rows(p, static_cast<QT *>(a.dk_), (long long)hq * p.dk, w, GAP_WGS);
        zero_rows(p, static_cast<bf16 *>(a.dv_), (long long)p.H * p.dv, w, GAP_WGS);
        zero_rows(p, a.dg, p.H, w, GAP_WGS);
        return;
    }
    int id = xcd_remap(blockIdx.x, walks);
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
    const int hk = h / (p.H / p.G);
    const long long ldv = (long long)p.H * p.dv, ldq = (long long)hq * p.dk, nh = (long long)n * p.H + h, sz = (long long)p.dk * p.dv;
    const long long t0 = s.row * p.tokens + s.start, e0 = (long long)(c1 - 1) * C;              // the tensors' pointers start at the last chunk
    const bf16 *Q = static_cast<const bf16 *>(p.q) + s.row * p.qb + (s.start + e0) * p.ql + hk * p.qh;
    const bf16 *K = static_cast<const bf16 *>(p.k) + s.row * p.kb + (s.start + e0) * p.kl + hk * p.kh;
    const bf16 *V = static_cast<const bf16 *>(p.v) + s.row * p.vb + (s.start + e0) * p.vl + h * p.vh;
    const bf16 *DO = static_cast<const bf16 *>(a.dout) + ((t0 + e0) * p.H + h) * (long long)p.dv;
    const float *g = p.g + s.row * p.gb + s.start * p.gl + h * p.gh;
    QT *DQ = static_cast<QT *>(a.dq) + ((t0 + e0) * hq + h) * (long long)p.dk;
    QT *DKp = static_cast<QT *>(a.dk_) + ((t0 + e0) * hq + h) * (long long)p.dk;
    bf16 *DVp = static_cast<bf16 *>(a.dv_) + ((t0 + e0) * p.H + h) * (long long)p.dv;
    float *DG = a.dg + t0 * p.H + h;
    const int kt = wave % KT, i0 = wave / KT * NI;                   // dq / dk: column tile, first row tile
    const int vt = wave % VT, j0 = wave / VT * NJ, kd = wave / VT * TW;           // dv: column tile, first row tile; D: first row tile
    f4 D[TW];
    TileRegs<C, DK, NT, VEC> qr, kr;
    TileRegs<C, DV, NT, VEC> vr, orr;
    qr.init(Q, p.ql, p.dk);
    kr.init(K, p.kl, p.dk);
    vr.init(V, p.vl, p.dv);
    orr.init(DO, ldv, p.dv);
    f4 sr[TW];                                                       // S in D's arrangement
    const f4 *saved = reinterpret_cast<const f4 *>(a.chunk_states) + ((chunk_base(p, s, n, C) + c1 - 1) * p.H + h) * (DK * DV / 4);
    auto rows_of = [&](int c) { const int left = s.len - c * C; return left < C ? left : C; };
    auto fetch = [&](int c) {
        const int nr = rows_of(c);
        qr.load(Q, p.ql, nr, p.dk);
        kr.load(K, p.kl, nr, p.dk);
        vr.load(V, p.vl, nr, p.dv);
        orr.load(DO, ldv, nr, p.dv);
        const int ln = fresh(lane0);
        const f4 *src = saved + vt * KT * 64 + ln;
#pragma unroll
        for (int t = 0; t < TW; ++t) sr[t] = src[64 * (kd + t)];
    };
    float gr = 0.0f;
    auto fetch_g = [&](int c) {
        if (wave == 0 && c >= c0) gr = lane0 < rows_of(c) ? limit_decay(g[((long long)c * C + lane0) * p.gl]) : 0.0f;
    };
    fetch_g(c1 - 1);
    if (c0 < c1) fetch(c1 - 1);
    {
        const int col = 16 * vt + (lane0 & 15);
        const float *init = segments_of(p, nch) > 1 ? a.seg_states + ((long long)slot * p.H + h) * sz : a.dlast ? a.dlast + nh * sz : nullptr;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = 16 * (kd + t) + 4 * (lane0 >> 4) + r;
                D[t][r] = init && col < p.dv && k < p.dk ? init[k * p.dv + col] : 0.0f;
            }
    }
    auto scan = [&](int c) {                                         // two chunks of: b (two terms), scale exp(b), exp(b_C - b), exp(b_C)
        if (wave == 0 && c >= c0) {
            float *d = decays + (c & 1) * 5 * C;
            const double b = chunk_decay_scan(gr), bend = lane63(b);
            const float hi = (float)b;
            d[lane0] = hi;
            d[C + lane0] = (float)(b - hi);
            d[2 * C + lane0] = hw_exp2(hi) * p.scale;
            d[3 * C + lane0] = hw_exp2((float)(bend - b));
            if (lane0 == 63) d[4 * C] = hw_exp2((float)bend);
        }
    };
    auto finish_dg = [&](int c) {                                    // behind a barrier after chunk c: the waves' parts of its decays' gradients
        if (wave == 1) {
            double x = 0.0;
#pragma unroll
            for (int w = 0; w < NW; ++w) x += (double)parts[w * C + lane0] + (double)corners[w];
            if (p.gl == 0) {                                         // one decay for all tokens
                if (lane0 >= rows_of(c)) x = 0.0;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
                if (lane0) x = 0.0;
            }
            if (lane0 < rows_of(c)) DG[((long long)c * C + lane0) * p.H] = (float)x;
        }
    };
    auto put_terms = [&](const f4 (&x)[TW], int u0) {                // terms u0 ... u0 + NB - 1 of a state -> St, row dv, column k
        const int ln = fresh(lane0), col = 16 * vt + (ln & 15);
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            const int k = 16 * (kd + t) + 4 * (ln >> 4);
            f4 v = x[t];
            unsigned char *d = St + col * SP + 2 * k;
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                if (u >= u0 + NB) break;
                const bf16x4 w = round4(v);
                if (u >= u0) *reinterpret_cast<bf16x4 *>(d + (NB == 3 ? u : 0) * DV * SP) = w;
                v = rest4(v, w);
            }
        }
    };
    if (tid < 128) {                             // the tiles of X and Y behind the diagonal that are read with it (32 columns at a time): zero for good
        const int half = tid >> 6, at = pair_row(half, 32 * half + (tid & 15)) + 2 * (32 * half + 16 + 4 * ((tid >> 4) & 3));
#pragma unroll
        for (int u = 0; u < (TURNS ? 3 : 6); ++u) *reinterpret_cast<u32x2 *>(Ys + u * PAIRS + at) = u32x2{0, 0};
    }
    if (tid == 0) *poison = -1;
    scan(c1 - 1);
    fetch_g(c1 - 2);
#pragma unroll 1
    for (int c = c1 - 1; c >= c0; --c) {
        const int nr = rows_of(c);
        const float *bh = decays + (c & 1) * 5 * C, *bl = bh + C, *eb = bl + C, *wt = eb + C, *tail = wt + C;
        __syncthreads();
        if (c + 1 < c1) finish_dg(c + 1);
        qr.put(Qs, QP, p.dk);
        kr.put(Ks, QP, p.dk);
        vr.put(Vs, VP, p.dv);
        orr.put(Os, VP, p.dv);
        if (qr.not_finite() || kr.not_finite() || orr.not_finite()) *poison = c;
        float corner = 0.0f;                                         // <D, S>
#pragma unroll
        for (int t = 0; t < TW; ++t) corner += (sr[t].x * D[t].x + sr[t].y * D[t].y) + (sr[t].z * D[t].z + sr[t].w * D[t].w);
        put_terms(sr, 0);
        __syncthreads();
        const bool poisoned = __builtin_amdgcn_readfirstlane(*poison) == c;
        const auto pair_of = [](const unsigned char *pairs, int i, int j) { return get_pair(pairs + pair_row(i >> 5, i) + 2 * j); };
        float cross = 0.0f;                                          // what this wave's pairs add to the decay of token `lane`
        // X, Y and the sums of M below the diagonal: ten 16 x 16 tiles dealt to the waves
        constexpr int NTL = (10 + NW - 1) / NW;
        f4 xs[NTL];                                                  // X, where it takes Y's place later
#pragma unroll
        for (int tn = 0; tn < NTL; ++tn) {
            const int t = wave + tn * NW;
            if (t >= 10) break;
            const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
            const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2, i = 16 * it + l16, j = 16 * jt + 4 * gq;
            f4 x = f4{0, 0, 0, 0}, y = f4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) x = mfma8(frag_c(Ks, QP, 16 * jt + l16, ks, gq), frag_c(Qs, QP, i, ks, gq), x);
#pragma unroll
            for (int vs = 0; vs < VS; ++vs) y = mfma8(frag_c(Vs, VP, 16 * jt + l16, vs, gq), frag_c(Os, VP, i, vs, gq), y);
            const float hi = bh[i], li = bl[i];
            const f4 h4 = *reinterpret_cast<const f4 *>(bh + j), l4 = *reinterpret_cast<const f4 *>(bl + j);
            f4 m;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = p.scale * hw_exp2((hi - h4[r]) + (li - l4[r]));
                y[r] = j + r <= i ? y[r] * w : 0.0f;
                m[r] = j + r < i ? x[r] * y[r] : 0.0f;
                x[r] = j + r <= i ? x[r] * w : 0.0f;
            }
            const int at = pair_row(it / 2, i) + 2 * j;
            put_pairs(Ys + at, y);
            if (TURNS) xs[tn] = x;
            else put_pairs(Xs + at, x);
            if (it == jt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) m[r] = row16_from_end(m[r]);        // of column j, the rows from token l16 on
                const float d = four_before(m, l16, gq);
                cross += gq == it ? d : 0.0f;
            } else {
                const float rows = row16_from_end(rows_sum((m.x + m.y) + (m.z + m.w)));
#pragma unroll
                for (int r = 0; r < 4; ++r) m[r] = row16_sum(m[r]);
                cross += cross_tile(rows, four_before(m, l16, gq), it, jt, gq);
            }
        }
        {   // dq
            const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
            f4 acc[NI];
#pragma unroll
            for (int m = 0; m < NI; ++m) acc[m] = f4{0, 0, 0, 0};
#pragma unroll 1
            for (int u0 = 0; u0 < 3; u0 += NB) {
                if (u0 > 0) {
                    __syncthreads();
                    put_terms(sr, u0);
                    __syncthreads();
                }
#pragma unroll
                for (int vs = 0; vs < VS; ++vs) {
                    bf16x8 of[NI];
#pragma unroll
                    for (int m = 0; m < NI; ++m) of[m] = frag_c(Os, VP, 16 * (i0 + m) + l16, vs, gq);
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        const bf16x8 sf = frag_tc(St + u * DV * SP, SP, kt, vs, lane);
#pragma unroll
                        for (int m = 0; m < NI; ++m) acc[m] = mfma8(sf, of[m], acc[m]);
                    }
                }
            }
            const int k = 16 * kt + 4 * gq;
#pragma unroll
            for (int m = 0; m < NI; ++m) {
                const int i = 16 * (i0 + m) + l16;
                acc[m] *= eb[i];
                const u32x2 w = *reinterpret_cast<const u32x2 *>(Qs + i * QP + 2 * k);
                const f2 q0 = bf16pair_to_f2(w.x), q1 = bf16pair_to_f2(w.y);
                const float d = rows_sum((acc[m].x * q0.x + acc[m].y * q0.y) + (acc[m].z * q1.x + acc[m].w * q1.y));
                cross += cross_rows(row16_from_end(d), i0 + m, gq);                  // pairs with the state in front of the chunk
            }
            __syncthreads();                                          // X, Y are there; S is done with
            put_terms(D, 0);
#pragma unroll
            for (int js = 0; js < 2; ++js) {
                bf16x8 kf = frag_tc(Ks, QP, kt, js, lane);
                if (poisoned) finite_only(kf);
#pragma unroll
                for (int m = 0; m < NI; ++m) {
                    if (js > (i0 + m) / 2) continue;
                    const int half = (i0 + m) / 2;
#pragma unroll
                    for (int u = 0; u < 3; ++u)
                        acc[m] = mfma8(kf, frag_c(Ys + u * PAIRS + pair_row(half, 0), pair_pitch(half), 16 * (i0 + m) + l16, js, gq), acc[m]);
                }
            }
            if (poisoned)
                each_not_finite4(Ks + 2 * k, QP, C, [&](int j, int r, float x) {
#pragma unroll
                    for (int m = 0; m < NI; ++m)
                        if (j <= 16 * (i0 + m) + l16) acc[m][r] += pair_of(Ys, 16 * (i0 + m) + l16, j) * x;
                });
            const RowsOut out(DQ, nr, ldq);
#pragma unroll
            for (int m = 0; m < NI; ++m) out.template put4<VEC>(DQ, 16 * (i0 + m) + l16, k, ldq, p.dk, acc[m]);
        }
        __syncthreads();                                              // D's terms are there
        const float eend = tail[0];
        Q -= C * p.ql; K -= C * p.kl; V -= C * p.vl; DO -= C * ldv; saved -= (long long)p.H * (DK * DV / 4);
        if (NB == 3 && c > c0) fetch(c - 1);
        {   // dk and dv
            const int lane = fresh(lane0), l16 = lane & 15, gq = lane >> 4;
            f4 dk[NI], dv[NJ];
#pragma unroll
            for (int m = 0; m < NI; ++m) dk[m] = f4{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < NJ; ++m) dv[m] = f4{0, 0, 0, 0};
            const int vrow = 16 * vt + l16;
#pragma unroll 1
            for (int u0 = 0; u0 < 3; u0 += NB) {
                if (u0 > 0) {
                    __syncthreads();
                    put_terms(D, u0);
                    __syncthreads();
                }
#pragma unroll
                for (int vs = 0; vs < VS; ++vs) {
                    bf16x8 vf[NI];
#pragma unroll
                    for (int m = 0; m < NI; ++m) vf[m] = frag_c(Vs, VP, 16 * (i0 + m) + l16, vs, gq);
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        const bf16x8 df = frag_tc(St + u * DV * SP, SP, kt, vs, lane);
#pragma unroll
                        for (int m = 0; m < NI; ++m) dk[m] = mfma8(df, vf[m], dk[m]);
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    bf16x8 kf[NJ];
#pragma unroll
                    for (int m = 0; m < NJ; ++m) kf[m] = frag_c(Ks, QP, 16 * (j0 + m) + l16, ks, gq);
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        const bf16x8 df = frag_c(St + u * DV * SP, SP, vrow, ks, gq);
#pragma unroll
                        for (int m = 0; m < NJ; ++m) dv[m] = mfma8(df, kf[m], dv[m]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < NI; ++m) {
                const int j = 16 * (i0 + m) + l16;
                dk[m] *= wt[j];
                const u32x2 w = *reinterpret_cast<const u32x2 *>(Ks + j * QP + 2 * (16 * kt + 4 * gq));
                const f2 k0 = bf16pair_to_f2(w.x), k1 = bf16pair_to_f2(w.y);
                const float d = rows_sum((dk[m].x * k0.x + dk[m].y * k0.y) + (dk[m].z * k1.x + dk[m].w * k1.y));
                cross += cross_columns(row16_from_start(d), i0 + m, gq);             // pairs with D
            }
            parts[wave * C + lane] = cross;
            corner = lanes_sum<64>(corner * eend);
            if (lane == 0) corners[wave] = corner;
#pragma unroll
            for (int m = 0; m < NJ; ++m) dv[m] *= wt[16 * (j0 + m) + l16];
            const int k = 16 * kt + 4 * gq, v = 16 * vt + 4 * gq;
            const RowsOut outk(DKp, nr, ldq), outv(DVp, nr, ldv);
#pragma unroll
            for (int is = 0; is < 2; ++is) {
                bf16x8 qf = frag_t(Qs, QP, kt, is, lane);
                if (poisoned) finite_only(qf);
#pragma unroll
                for (int m = 0; m < NI; ++m) {
                    if (is < (i0 + m) / 2) continue;
#pragma unroll
                    for (int u = 0; u < 3; ++u) dk[m] = mfma8(qf, frag_t(Ys + u * PAIRS + pair_row(is, 0), pair_pitch(is), i0 + m, is, lane), dk[m]);
                }
            }
            if (poisoned)
                each_not_finite4(Qs + 2 * k, QP, C, [&](int i, int r, float x) {
#pragma unroll
                    for (int m = 0; m < NI; ++m)
                        if (i >= 16 * (i0 + m) + l16) dk[m][r] += pair_of(Ys, i, 16 * (i0 + m) + l16) * x;
                });
#pragma unroll
            for (int m = 0; m < NI; ++m) outk.template put4<VEC>(DKp, 16 * (i0 + m) + l16, k, ldq, p.dk, dk[m]);
            if (TURNS) {
                __syncthreads();                                      // Y is done with
#pragma unroll
                for (int tn = 0; tn < NTL; ++tn) {
                    const int t = wave + tn * NW, it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
                    if (t < 10) put_pairs(Xs + pair_row(it / 2, 16 * it + l16) + 2 * (16 * jt + 4 * gq), xs[tn]);
                }
                __syncthreads();                                      // X is there
            }
#pragma unroll
            for (int is = 0; is < 2; ++is) {
                bf16x8 of = frag_t(Os, VP, vt, is, lane);
                if (poisoned) finite_only(of);
#pragma unroll
                for (int m = 0; m < NJ; ++m) {
                    if (is < (j0 + m) / 2) continue;
#pragma unroll
                    for (int u = 0; u < 3; ++u) dv[m] = mfma8(of, frag_t(Xs + u * PAIRS + pair_row(is, 0), pair_pitch(is), j0 + m, is, lane), dv[m]);
                }
            }
            if (poisoned)
                each_not_finite4(Os + 2 * v, VP, C, [&](int i, int r, float x) {
#pragma unroll
                    for (int m = 0; m < NJ; ++m)
                        if (i >= 16 * (j0 + m) + l16) dv[m][r] += pair_of(Xs, i, 16 * (j0 + m) + l16) * x;
                });
#pragma unroll
            for (int m = 0; m < NJ; ++m) outv.template put4<VEC>(DVp, 16 * (j0 + m) + l16, v, ldv, p.dv, dv[m]);
        }
        DQ -= C * ldq; DKp -= C * ldq; DVp -= C * ldv;
        {   // D
            const int lane = fresh(lane0), gq = lane >> 4;
            if (NB == 1 && c > c0) fetch(c - 1);
            scan(c - 1);
            fetch_g(c - 2);
            bf16x8 ow[2][3];
#pragma unroll
            for (int is = 0; is < 2; ++is) {
                f4 x, y;
                widen8(frag_t(Os, VP, vt, is, lane), x, y);
                split8<3>(x * *reinterpret_cast<const f4 *>(eb + 32 * is + 4 * gq), y * *reinterpret_cast<const f4 *>(eb + 32 * is + 16 + 4 * gq), ow[is]);
            }
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                D[t] *= eend;
#pragma unroll
                for (int is = 0; is < 2; ++is) {
                    const bf16x8 qf = frag_t(Qs, QP, kd + t, is, lane);
#pragma unroll
                    for (int u = 0; u < 3; ++u) D[t] = mfma8(qf, ow[is][u], D[t]);
                }
            }
        }
    }
    __syncthreads();
    if (c0 < c1) finish_dg(c0);
    if (a.ds0 && c0 == 0) {
        const int col = 16 * vt + (lane0 & 15);
        float *d = a.ds0 + nh * sz;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = 16 * (kd + t) + 4 * (lane0 >> 4) + r;
                if (col < p.dv && k < p.dk) d[k * p.dv + col] = D[t][r];
            }
    }
}

// dq / dk of the value heads that share a key head, summed in order: (rows, G, rep, dk) fp32 -> (rows, G, dk).  W columns a thread
template <int W, typename IO>
__global__ __launch_bounds__(NT) void la_head_sum_kernel(const float *a, const float *b, IO *oa, IO *ob, long long total, int rep, int dk) {
    const long long e = ((long long)blockIdx.x * NT + threadIdx.x) * W;
    if (e >= total) return;
    const long long rg = e / dk;
    const float *src = (blockIdx.y ? b : a) + rg * rep * dk + (e - rg * dk);
    IO *dst = (blockIdx.y ? ob : oa) + e;
    if (W == 4) {
        f4 v = ld4(src);
#pragma unroll 4
        for (int i = 1; i < rep; ++i) v += ld4(src + (long long)i * dk);
        st4(dst, v);
    } else {
        float v = src[0];
        for (int i = 1; i < rep; ++i) v += src[(long long)i * dk];
        st1(dst, v);
    }
}
template <typename IO>
void launch_head_sum(const float *a, const float *b, void *oa, void *ob, long long total, int rep, int dk, hipStream_t s) {
    const int w = dk % 4 == 0 ? 4 : 1;
    const dim3 grid((unsigned)((total / w + NT - 1) / NT), 2);
    if (w == 4) ss2d_launch((la_head_sum_kernel<4, IO>), grid, dim3(NT), 0, s, a, b, static_cast<IO *>(oa), static_cast<IO *>(ob), total, rep, dk);
    else ss2d_launch((la_head_sum_kernel<1, IO>), grid, dim3(NT), 0, s, a, b, static_cast<IO *>(oa), static_cast<IO *>(ob), total, rep, dk);
}

template <int DK, int DV, int C, int NW>
void launch_bwd(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const unsigned walks = (unsigned)((long long)a.p.slots * a.p.H);
    if (a.p.vec) ss2d_launch((la_bwd_kernel<DK, DV, C, NW, true>), dim3(walks + gaps), dim3(64 * NW), 0, s, a);
    else ss2d_launch((la_bwd_kernel<DK, DV, C, NW, false>), dim3(walks + gaps), dim3(64 * NW), 0, s, a);
}
void dispatch_bwd_f32(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const int dk = a.p.dk, dv = a.p.dv;
    if (dv <= 64) {
        if (dk <= 16) launch_bwd<16, 64, 64, 8>(a, gaps, s);
        else if (dk <= 64) launch_bwd<64, 64, 64, 16>(a, gaps, s);
        else launch_bwd<128, 64, 32, 16>(a, gaps, s);
    } else {
        if (dk <= 16) launch_bwd<16, 128, 32, 8>(a, gaps, s);
        else if (dk <= 64) launch_bwd<64, 128, 32, 16>(a, gaps, s);
        else launch_bwd<128, 128, 32, 16>(a, gaps, s);
    }
}

template <int DK, int DV, bool VEC>
void launch_bwd_bf16(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const unsigned walks = (unsigned)((long long)a.p.slots * a.p.H);
    constexpr int NW = DK <= 32 || (DK == 64 && DV == 64) ? 8 : 16;
    if (a.p.H > a.p.G) ss2d_launch((la_bwd_bf16_kernel<DK, DV, NW, VEC, float>), dim3(walks + gaps), dim3(64 * NW), 0, s, a);
    else ss2d_launch((la_bwd_bf16_kernel<DK, DV, NW, VEC, bf16>), dim3(walks + gaps), dim3(64 * NW), 0, s, a);
}
template <bool VEC>
void dispatch_bwd_bf16(const BwdArgs &a, unsigned gaps, hipStream_t s) {
    const Problem &p = a.p;
    const int dk = p.dk;
    if (p.dv <= 64) {
        if (dk <= 32) launch_bwd_bf16<32, 64, VEC>(a, gaps, s);
        else if (dk <= 64) launch_bwd_bf16<64, 64, VEC>(a, gaps, s);
        else launch_bwd_bf16<128, 64, VEC>(a, gaps, s);
    } else {
        if (dk <= 32) launch_bwd_bf16<32, 128, VEC>(a, gaps, s);
        else if (dk <= 64) launch_bwd_bf16<64, 128, VEC>(a, gaps, s);
        else launch_bwd_bf16<128, 128, VEC>(a, gaps, s);
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
    a.p.vec = a.p.vec && (dtype == SS2D_DTYPE_F32 || (uintptr_t)dout % 4 == 0);
    const unsigned gaps = cu_seqlens ? GAP_WGS : 0;
    hipStream_t s = (hipStream_t)stream;
    if (nseg > 1) {
        Problem r = a.p;                          // q in the place of k, dout in that of v
        r.k = q; r.kb = r.qb; r.kl = r.ql; r.kh = r.qh;
        r.v = dout; r.vb = tokens * H * dv; r.vl = (long long)H * dv; r.vh = dv;
        linattn_segment_pass(dtype, r, seg_states, seg_decay, true, s);
        const int C = linattn_chunk(dtype, dk, dv), w = dk * dv % 4 == 0 ? 4 : 1;
        const dim3 grid((unsigned)((dk * dv + NT * w - 1) / (NT * w) * N * H));
        if (w == 4) ss2d_launch(la_join_bwd_kernel<4>, grid, dim3(NT), 0, s, a, C);
        else ss2d_launch(la_join_bwd_kernel<1>, grid, dim3(NT), 0, s, a, C);
    }
    if (dtype == SS2D_DTYPE_F32) dispatch_bwd_f32(a, gaps, s);
    else if (a.p.vec) dispatch_bwd_bf16<true>(a, gaps, s);
    else dispatch_bwd_bf16<false>(a, gaps, s);
    if (H > G) {
        const long long rows = (cu_seqlens ? 1 : N) * tokens, total = rows * G * dk;
        if (dtype == SS2D_DTYPE_BF16) launch_head_sum<bf16>(dq_heads, dk_heads, dq, dk_out, total, H / G, dk, s);
        else launch_head_sum<float>(dq_heads, dk_heads, dq, dk_out, total, H / G, dk, s);
    }
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("linattn_bwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
