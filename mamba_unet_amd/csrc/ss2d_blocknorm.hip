// The norms around a block, with its gate and residual scale, in one pass (gfx950):
//     u = norm(y; w1, b1) * SiLU(z),   x' = x + drop * a * u,   h = norm(x'; w2, b2)
// norm: LayerNorm or RMS norm over the last axis (fp32 statistics); y is the block's output, z its gate, a a per-channel residual scale, drop a
// per-sample factor, x the residual stream and h the next block's input.  Beside ss2d_outnorm_gate (norm and gate in front of a projection) and
// ss2d_layernorm: there the residual stream makes a round trip through memory between the two norms.
//
// Memory-bound.  TPR threads hold one row (NV pieces of VEC elements each), so x, y and z are read once and x', h written once; h's
// statistics are those of the unrounded x'.  The backward recomputes x' from x, y, z (the same bytes as reading a saved x') and walks
// rows with its share of the five column sums in registers; the workgroups' sums go to a workspace and are added in a fixed order.
#include "ss2d_common.h"
#include "../../include/ss2d.h"

namespace {

constexpr int NT = 256;

struct Args {
    const void *x, *y, *z, *dxo, *dh;
    const float *w1, *b1, *w2, *b2, *a, *drop;
    void *xo, *h, *dx, *dy, *dz;
    float *stats;                 // (rows, 4): mean and 1 / deviation of y, then of x'
    float *partials;              // backward: (workgroups, 5, D)
    long long rows, ldx, ldy, ldz;
    unsigned rps;                 // rows a sample
    int D, rms;
    float eps;
};

template <int TPR>
struct Red {                      // sums over the TPR threads of a row, in every one of them
    float *lds;                   // TPR > 64: 2 * 2 * (TPR / 64) floats a row (two buffers: one barrier a sum)
    int flip = 0;
    __device__ __forceinline__ void two(float &a, float &b) {
        if (TPR == 16) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int c[4] = {8, 4, 2, 1};
                if (c[d] == 8) { a += dpp_mov<DPP_ROW_ROR(8), 0xf, false>(0.0f, a); b += dpp_mov<DPP_ROW_ROR(8), 0xf, false>(0.0f, b); }
                if (c[d] == 4) { a += dpp_mov<DPP_ROW_ROR(4), 0xf, false>(0.0f, a); b += dpp_mov<DPP_ROW_ROR(4), 0xf, false>(0.0f, b); }
                if (c[d] == 2) { a += dpp_mov<DPP_ROW_ROR(2), 0xf, false>(0.0f, a); b += dpp_mov<DPP_ROW_ROR(2), 0xf, false>(0.0f, b); }
                if (c[d] == 1) { a += dpp_mov<DPP_ROW_ROR(1), 0xf, false>(0.0f, a); b += dpp_mov<DPP_ROW_ROR(1), 0xf, false>(0.0f, b); }
            }
        } else {
            a = lanes_sum<64>(a);
            b = lanes_sum<64>(b);
            if (TPR > 64) {
                constexpr int W = TPR / 64;
                const int wave = threadIdx.x >> 6, w0 = wave / W * W;
                float *s = lds + flip * 2 * (NT / 64);
                if ((threadIdx.x & 63) == 0) { s[2 * wave] = a; s[2 * wave + 1] = b; }
                __syncthreads();
                a = 0.0f; b = 0.0f;
#pragma unroll
                for (int i = 0; i < W; ++i) { a += s[2 * (w0 + i)]; b += s[2 * (w0 + i) + 1]; }
                flip ^= 1;
            }
        }
    }
    __device__ __forceinline__ float one(float a) { float b = 0.0f; two(a, b); return a; }
};

// NV pieces of VEC elements of a row: element (i, e) is column (i * TPR + t) * VEC + e; past D reads 0
template <int TPR, int NV, int VEC, typename T>
__device__ __forceinline__ void load_row(float (&v)[NV * VEC], const T *row, int t, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        const bool ok = c < D;
        if (VEC == 8) {
            const T *q = row + (ok ? c : 0);
            const f4 a = ld4(q), b = ld4(q + (VEC == 8 ? 4 : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[i * VEC + e] = ok ? a[e] : 0.0f; v[i * VEC + (VEC == 8 ? 4 : 0) + e] = ok ? b[e] : 0.0f; }
        } else {
            const float a = ld1(row + (ok ? c : 0));
            v[i * VEC] = ok ? a : 0.0f;
        }
    }
}
template <int TPR, int NV, int VEC, typename T>
__device__ __forceinline__ void store_row(const float (&v)[NV * VEC], T *row, int t, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c >= D) continue;
        if (VEC == 8) {
            st4(row + c, f4{v[i * VEC], v[i * VEC + (VEC > 1)], v[i * VEC + 2 * (VEC > 2)], v[i * VEC + 3 * (VEC > 3)]});
            st4(row + c + 4, f4{v[i * VEC + 4 * (VEC > 4)], v[i * VEC + 5 * (VEC > 5)], v[i * VEC + 6 * (VEC > 6)], v[i * VEC + 7 * (VEC > 7)]});
        } else {
            st1(row + c, v[i * VEC]);
        }
    }
}
template <int TPR, int NV, int VEC>
__device__ __forceinline__ bool col_ok(int j, int t, int D) { return ((j / VEC) * TPR + t) * VEC < D; }   // element j of a thread
template <int TPR, int NV, int VEC>
__device__ __forceinline__ float param(const float *w, int j, int t, int D, float none) {
    const int c = ((j / VEC) * TPR + t) * VEC + j % VEC;
    return w && c < D ? w[c] : none;
}

// statistics of a row held in v: two passes over registers, so a large mean costs no digits
template <int TPR, int NV, int VEC>
__device__ __forceinline__ void row_stats(const float (&v)[NV * VEC], Red<TPR> &red, int t, int D, float invD, bool rms, float eps, float &mu, float &rs) {
    mu = 0.0f;
    if (!rms) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV * VEC; ++j) s += v[j];
        mu = red.one(s) * invD;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV * VEC; ++j) {
        const float d = v[j] - mu;
        q += col_ok<TPR, NV, VEC>(j, t, D) ? d * d : 0.0f;
    }
    const float var = red.one(q) * invD + eps;
    rs = 1.0f / sqrtf(var);
}

template <int TPR, int NV, int VEC, typename RT, typename IO>
__global__ __launch_bounds__(NT) void block_norm_fwd_kernel(const Args p) {
    constexpr int RPW = NT / TPR, E = NV * VEC;
    __shared__ float lds[4 * (NT / 64)];
    Red<TPR> red{lds};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = p.D;
    const float invD = 1.0f / (float)D;
    // whole workgroups walk together (the sums of a row may use barriers): rows past the end repeat the last one and store nothing
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += (long long)gridDim.x * RPW) {
        const bool live = r0 + sub < p.rows;
        const long long r = live ? r0 + sub : p.rows - 1;
        float x[E], y[E], z[E];
        load_row<TPR, NV, VEC>(y, static_cast<const IO *>(p.y) + r * p.ldy, t, D);
        load_row<TPR, NV, VEC>(x, static_cast<const RT *>(p.x) + r * p.ldx, t, D);
        if (p.z) load_row<TPR, NV, VEC>(z, static_cast<const IO *>(p.z) + r * p.ldz, t, D);
        const float drop = p.drop ? p.drop[(unsigned)(r / p.rps)] : 1.0f;
        float m1, r1, m2, r2;
        row_stats<TPR, NV, VEC>(y, red, t, D, invD, p.rms, p.eps, m1, r1);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float u = (y[j] - m1) * r1 * param<TPR, NV, VEC>(p.w1, j, t, D, 0.0f) + param<TPR, NV, VEC>(p.b1, j, t, D, 0.0f);
            if (p.z) u *= z[j] * sigmoidf_fast(z[j]);
            x[j] += drop * param<TPR, NV, VEC>(p.a, j, t, D, 1.0f) * u;
            if (!col_ok<TPR, NV, VEC>(j, t, D)) x[j] = 0.0f;
        }
        row_stats<TPR, NV, VEC>(x, red, t, D, invD, p.rms, p.eps, m2, r2);
#pragma unroll
        for (int j = 0; j < E; ++j)
            y[j] = (x[j] - m2) * r2 * param<TPR, NV, VEC>(p.w2, j, t, D, 0.0f) + param<TPR, NV, VEC>(p.b2, j, t, D, 0.0f);
        if (live) {
            store_row<TPR, NV, VEC>(x, static_cast<RT *>(p.xo) + r * D, t, D);
            store_row<TPR, NV, VEC>(y, static_cast<IO *>(p.h) + r * D, t, D);
            if (p.stats && t == 0) *reinterpret_cast<f4 *>(p.stats + 4 * r) = f4{m1, r1, m2, r2};
        }
    }
}

template <int TPR, int NV, int VEC, typename RT, typename IO>
__global__ __launch_bounds__(NT) void block_norm_bwd_kernel(const Args p) {
    constexpr int RPW = NT / TPR, E = NV * VEC;
    __shared__ float lds[4 * (NT / 64)];
    __shared__ float cols[RPW > 1 ? RPW * TPR * E : 1];
    Red<TPR> red{lds};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = p.D;
    const float invD = 1.0f / (float)D;
    float aw1[E], ab1[E], aa[E], aw2[E], ab2[E];
#pragma unroll
    for (int j = 0; j < E; ++j) aw1[j] = ab1[j] = aa[j] = aw2[j] = ab2[j] = 0.0f;
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += (long long)gridDim.x * RPW) {
        const bool live = r0 + sub < p.rows;
        const long long r = live ? r0 + sub : p.rows - 1;
        float x[E], y[E], z[E], g[E], dh[E];
        load_row<TPR, NV, VEC>(y, static_cast<const IO *>(p.y) + r * p.ldy, t, D);
        load_row<TPR, NV, VEC>(x, static_cast<const RT *>(p.x) + r * p.ldx, t, D);
        if (p.z) load_row<TPR, NV, VEC>(z, static_cast<const IO *>(p.z) + r * p.ldz, t, D);
        if (p.dh) load_row<TPR, NV, VEC>(dh, static_cast<const IO *>(p.dh) + r * D, t, D);
        if (p.dxo) load_row<TPR, NV, VEC>(g, static_cast<const RT *>(p.dxo) + r * D, t, D);
        const f4 st = *reinterpret_cast<const f4 *>(p.stats + 4 * r);
        const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w, drop = p.drop ? p.drop[(unsigned)(r / p.rps)] : 1.0f;
        // y becomes its normalised value, x the normalised x', u = post-norm times gate
        float u[E], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (!p.dh) dh[j] = 0.0f;
            if (!p.dxo) g[j] = 0.0f;
            y[j] = (y[j] - m1) * r1;
            const float v = y[j] * param<TPR, NV, VEC>(p.w1, j, t, D, 0.0f) + param<TPR, NV, VEC>(p.b1, j, t, D, 0.0f);
            u[j] = p.z ? v * (z[j] * sigmoidf_fast(z[j])) : v;
            x[j] = (x[j] + drop * param<TPR, NV, VEC>(p.a, j, t, D, 1.0f) * u[j] - m2) * r2;
            const float d = dh[j] * param<TPR, NV, VEC>(p.w2, j, t, D, 0.0f);       // 0 past D
            s1 += d;
            s2 += d * x[j];
            if (live) { aw2[j] += dh[j] * x[j]; ab2[j] += dh[j]; }
        }
        red.two(s1, s2);
        s1 = p.rms ? 0.0f : s1 * invD;
        s2 *= invD;
        float q1 = 0.0f, q2 = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            g[j] += r2 * (dh[j] * param<TPR, NV, VEC>(p.w2, j, t, D, 0.0f) - s1 - x[j] * s2);      // dx
            const float gd = g[j] * drop, du = gd * param<TPR, NV, VEC>(p.a, j, t, D, 1.0f);
            if (live) aa[j] += gd * u[j];
            float dv = du;
            if (p.z) {
                const float v = y[j] * param<TPR, NV, VEC>(p.w1, j, t, D, 0.0f) + param<TPR, NV, VEC>(p.b1, j, t, D, 0.0f);
                const float sg = sigmoidf_fast(z[j]);
                dv = du * (z[j] * sg);
                z[j] = du * v * (sg * (1.0f + z[j] * (1.0f - sg)));                               // dz
            }
            if (live) { aw1[j] += dv * y[j]; ab1[j] += dv; }
            u[j] = col_ok<TPR, NV, VEC>(j, t, D) ? dv * param<TPR, NV, VEC>(p.w1, j, t, D, 0.0f) : 0.0f;
            q1 += u[j];
            q2 += u[j] * y[j];
        }
        red.two(q1, q2);
        q1 = p.rms ? 0.0f : q1 * invD;
        q2 *= invD;
#pragma unroll
        for (int j = 0; j < E; ++j) u[j] = r1 * (u[j] - q1 - y[j] * q2);                           // dy
        if (live) {
            store_row<TPR, NV, VEC>(g, static_cast<RT *>(p.dx) + r * D, t, D);
            store_row<TPR, NV, VEC>(u, static_cast<IO *>(p.dy) + r * D, t, D);
            if (p.z) store_row<TPR, NV, VEC>(z, static_cast<IO *>(p.dz) + r * D, t, D);
        }
    }
    // this workgroup's column sums
    float *dst = p.partials + (long long)blockIdx.x * 5 * D;
    auto put = [&](const float (&v)[E], int which) {
        if (RPW > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < E; ++j) cols[(sub * TPR + t) * E + j] = v[j];
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float s = 0.0f;
                    for (int k = 0; k < RPW; ++k) s += cols[(k * TPR + t) * E + j];
                    const int c = ((j / VEC) * TPR + t) * VEC + j % VEC;
                    if (c < D) dst[which * D + c] = s;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int c = ((j / VEC) * TPR + t) * VEC + j % VEC;
                if (c < D) dst[which * D + c] = v[j];
            }
        }
    };
    put(aw1, 0); put(ab1, 1); put(aa, 2); put(aw2, 3); put(ab2, 4);
}

// out (5, D) = sum of the workgroups' partial rows, in order; 64 columns x 4 row lanes a workgroup
__global__ __launch_bounds__(NT) void block_norm_cols_kernel(const float *partials, float *out, int n, int wgs) {
    __shared__ float red[NT];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < n)
        for (int w = part; w < wgs; w += 4) s += partials[(long long)w * n + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (part == 0 && c < n) out[c] = (red[threadIdx.x] + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
}

int bwd_wgs(long long rows, int D) {
    const int tpr = D <= 128 ? 16 : D <= 1024 ? 64 : 256;
    const long long n = (rows + NT / tpr - 1) / (NT / tpr);
    return (int)(n < 512 ? n : 512);
}

template <int TPR, int NV, int VEC, typename RT, typename IO>
void launch_one(bool bwd, const Args &p, hipStream_t s) {
    constexpr int RPW = NT / TPR;
    if (!bwd) {
        long long n = (p.rows + RPW - 1) / RPW;
        if (n > 4096) n = 4096;
        ss2d_launch((block_norm_fwd_kernel<TPR, NV, VEC, RT, IO>), dim3((unsigned)n), dim3(NT), 0, s, p);
    } else {
        ss2d_launch((block_norm_bwd_kernel<TPR, NV, VEC, RT, IO>), dim3((unsigned)bwd_wgs(p.rows, p.D)), dim3(NT), 0, s, p);
    }
}
template <typename RT, typename IO>
void launch(bool bwd, bool vec, const Args &p, hipStream_t s) {
    if (p.D <= 128) vec ? launch_one<16, 1, 8, RT, IO>(bwd, p, s) : launch_one<16, 8, 1, RT, IO>(bwd, p, s);
    else if (p.D <= 512) vec ? launch_one<64, 1, 8, RT, IO>(bwd, p, s) : launch_one<64, 8, 1, RT, IO>(bwd, p, s);
    else if (p.D <= 1024) vec ? launch_one<64, 2, 8, RT, IO>(bwd, p, s) : launch_one<64, 16, 1, RT, IO>(bwd, p, s);
    else if (p.D <= 2048) vec ? launch_one<256, 1, 8, RT, IO>(bwd, p, s) : launch_one<256, 8, 1, RT, IO>(bwd, p, s);
    else if (p.D <= 4096) vec ? launch_one<256, 2, 8, RT, IO>(bwd, p, s) : launch_one<256, 16, 1, RT, IO>(bwd, p, s);
    else vec ? launch_one<256, 4, 8, RT, IO>(bwd, p, s) : launch_one<256, 32, 1, RT, IO>(bwd, p, s);
}
void dispatch(bool bwd, int rt, int io, bool vec, const Args &p, hipStream_t s) {
    if (rt == SS2D_DTYPE_F32) io == SS2D_DTYPE_F32 ? launch<float, float>(bwd, vec, p, s) : launch<float, bf16>(bwd, vec, p, s);
    else io == SS2D_DTYPE_F32 ? launch<bf16, float>(bwd, vec, p, s) : launch<bf16, bf16>(bwd, vec, p, s);
}

int check(const Args &p, int rt, int io, const char *name) {
    if ((rt != SS2D_DTYPE_F32 && rt != SS2D_DTYPE_BF16) || (io != SS2D_DTYPE_F32 && io != SS2D_DTYPE_BF16)) { ss2d_set_error("%s: unknown dtype", name); return -1; }
    if (p.rows <= 0 || p.D <= 0 || p.rows > 0xffffffffLL) { ss2d_set_error("%s: size out of range", name); return -3; }
    if (p.D > 8192) { ss2d_set_error("%s: D %d must be <= 8192", name, p.D); return -4; }
    if (p.ldx < p.D || p.ldy < p.D || (p.z && p.ldz < p.D)) { ss2d_set_error("%s: rows overlap", name); return -4; }
    return 0;
}
bool vec_ok(const Args &p) {
    const uintptr_t all = (uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.z | (uintptr_t)p.dxo | (uintptr_t)p.dh | (uintptr_t)p.xo | (uintptr_t)p.h | (uintptr_t)p.dx
        | (uintptr_t)p.dy | (uintptr_t)p.dz;
    return p.D % 8 == 0 && p.ldx % 8 == 0 && p.ldy % 8 == 0 && (!p.z || p.ldz % 8 == 0) && all % 16 == 0;
}

}  // namespace

extern "C" int ss2d_block_norm_fwd(int res_dtype, int dtype, const void *x, const void *y, const void *z, const float *w1, const float *b1, const float *w2,
                                   const float *b2, const float *res_scale, const float *drop, long long rows_per_sample, void *x_out, void *h,
                                   float *stats, long long rows, int D, long long ldx, long long ldy, long long ldz, float eps, int rms, void *stream) {
    Args p{};
    p.x = x; p.y = y; p.z = z; p.w1 = w1; p.b1 = b1; p.w2 = w2; p.b2 = b2; p.a = res_scale; p.drop = drop; p.xo = x_out; p.h = h; p.stats = stats;
    p.rows = rows; p.D = D; p.ldx = ldx; p.ldy = ldy; p.ldz = ldz; p.eps = eps; p.rms = rms;
    if (!x || !y || !w1 || !w2 || !x_out || !h) { ss2d_set_error("block_norm_fwd: null pointer"); return -2; }
    int rc = check(p, res_dtype, dtype, "block_norm_fwd");
    if (rc) return rc;
    if (drop && (rows_per_sample <= 0 || rows_per_sample > rows)) { ss2d_set_error("block_norm_fwd: rows_per_sample %lld", rows_per_sample); return -3; }
    p.rps = drop ? (unsigned)rows_per_sample : 1u;
    dispatch(false, res_dtype, dtype, vec_ok(p), p, (hipStream_t)stream);
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("block_norm_fwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}

extern "C" size_t ss2d_block_norm_bwd_workspace_floats(long long rows, int D) { return rows <= 0 || D <= 0 ? 0 : (size_t)bwd_wgs(rows, D) * 5 * (size_t)D; }

extern "C" int ss2d_block_norm_bwd(int res_dtype, int dtype, const void *dx_out, const void *dh, const void *x, const void *y, const void *z, const float *w1,
                                   const float *b1, const float *w2, const float *res_scale, const float *drop, long long rows_per_sample,
                                   const float *stats, void *dx, void *dy, void *dz, float *dparams, float *workspace, long long rows, int D,
                                   long long ldx, long long ldy, long long ldz, int rms, void *stream) {
    Args p{};
    p.x = x; p.y = y; p.z = z; p.dxo = dx_out; p.dh = dh; p.w1 = w1; p.b1 = b1; p.w2 = w2; p.a = res_scale; p.drop = drop; p.dx = dx; p.dy = dy; p.dz = dz;
    p.stats = const_cast<float *>(stats); p.partials = workspace; p.rows = rows; p.D = D; p.ldx = ldx; p.ldy = ldy; p.ldz = ldz; p.rms = rms;
    if (!x || !y || !w1 || !w2 || !stats || !dx || !dy || (z && !dz) || !dparams || !workspace) { ss2d_set_error("block_norm_bwd: null pointer"); return -2; }
    int rc = check(p, res_dtype, dtype, "block_norm_bwd");
    if (rc) return rc;
    if (drop && (rows_per_sample <= 0 || rows_per_sample > rows)) { ss2d_set_error("block_norm_bwd: rows_per_sample %lld", rows_per_sample); return -3; }
    p.rps = drop ? (unsigned)rows_per_sample : 1u;
    dispatch(true, res_dtype, dtype, vec_ok(p), p, (hipStream_t)stream);
    ss2d_launch(block_norm_cols_kernel, dim3((unsigned)((5 * D + 63) / 64)), dim3(NT), 0, (hipStream_t)stream, workspace, dparams, 5 * D, bwd_wgs(rows, D));
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("block_norm_bwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
