// The norms around a block, with its gate and residual scale, in one pass (gfx950):
//     u = norm(y; w1, b1) * SiLU(z),   x' = x + drop * a * u,   h = norm(x'; w2, b2)
// norm: LayerNorm or RMS norm over the last axis (fp32 statistics); y is the block's output, z its gate, a a per-channel residual scale, drop a
// per-sample factor, x the residual stream and h the next block's input.  Beside ss2d_outnorm_gate (norm and gate in front of a projection) and
// ss2d_layernorm: there the residual stream makes a round trip through memory between the two norms.
//
// Memory-bound.  TPR threads hold one row, eight elements each (16 bytes of bf16; rows that are not made of 16-byte pieces: single
// elements TPR apart), so x, y and z are read once and x', h written once; h's statistics are those of the unrounded x'.  A thread's parameters
// stay in registers over all its rows, and the next row is in flight while one is worked on.  The backward recomputes x' from x, y, z (the
// same bytes as reading a saved x') and holds its share of the five column sums in registers; the workgroups' sums go to a workspace and
// are added in a fixed order.
#include "ss2d_common.h"
#include "../../include/ss2d.h"

namespace {

constexpr int E = 8;              // elements of a row a thread holds

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

template <int TPR> constexpr int threads_of() { return TPR > 256 ? TPR : 256; }

template <int TPR>
struct Red {                      // sums over the TPR threads of a row, in every one of them
    static constexpr int WAVES = threads_of<TPR>() / 64;
    float *lds;                   // TPR > 64: two buffers of 2 floats a wave (so a sum needs one barrier)
    int flip = 0;
    __device__ __forceinline__ static float row16(float v) {
        v += dpp_mov<DPP_ROW_ROR(8), 0xf, false>(0.0f, v);
        v += dpp_mov<DPP_ROW_ROR(4), 0xf, false>(0.0f, v);
        v += dpp_mov<DPP_ROW_ROR(2), 0xf, false>(0.0f, v);
        return v + dpp_mov<DPP_ROW_ROR(1), 0xf, false>(0.0f, v);
    }
    __device__ __forceinline__ void two(float &a, float &b) {
        if (TPR == 16) {
            a = row16(a);
            b = row16(b);
            return;
        }
        a = lanes_sum<64>(a);
        b = lanes_sum<64>(b);
        if (TPR > 64) {
            constexpr int W = TPR / 64;
            const int wave = threadIdx.x >> 6, w0 = wave / W * W;
            float *s = lds + flip * 2 * WAVES;
            if ((threadIdx.x & 63) == 0) *reinterpret_cast<f2 *>(s + 2 * wave) = f2{a, b};
            __syncthreads();
            f2 v = *reinterpret_cast<const f2 *>(s + 2 * w0);
#pragma unroll
            for (int i = 1; i < W; ++i) v += *reinterpret_cast<const f2 *>(s + 2 * (w0 + i));
            a = v.x;
            b = v.y;
            flip ^= 1;
        }
    }
    __device__ __forceinline__ float one(float a) { float b = 0.0f; two(a, b); return a; }
};

// column of element j of thread t; VEC: eight side by side
template <int TPR, bool VEC>
__device__ __forceinline__ int column(int j, int t) { return VEC ? E * t + j : j * TPR + t; }

// a thread's share of a row as it lies in memory; columns past D are read at a clamped place and come out as 0
template <int TPR, bool VEC, typename T>
struct Piece {
    static constexpr int N = VEC ? (sizeof(T) == 2 ? 1 : 2) : 1;
    u32x4 v[N];
    T s[VEC ? 1 : E];
    __device__ __forceinline__ void load(const T *row, int t, int D) {
        if (VEC) {
            const u32x4 *q = reinterpret_cast<const u32x4 *>(row + (E * t < D ? E * t : 0));
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = q[i];
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int c = column<TPR, VEC>(j, t);
                s[VEC ? 0 : j] = row[c < D ? c : D - 1];
            }
        }
    }
    __device__ __forceinline__ void get(float (&o)[E], int t, int D) const {
        if (VEC) {
            const bool ok = E * t < D;
            if (sizeof(T) == 2) {
                const unsigned w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned x = ok ? w[i] : 0u;
                    o[2 * i] = __builtin_bit_cast(float, x << 16);
                    o[2 * i + 1] = __builtin_bit_cast(float, x & 0xffff0000u);
                }
            } else {
                const u32x4 a = v[0], b = v[N - 1];
                const unsigned w[E] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int j = 0; j < E; ++j) o[j] = ok ? __builtin_bit_cast(float, w[j]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] = column<TPR, VEC>(j, t) < D ? ld1(&s[VEC ? 0 : j]) : 0.0f;
        }
    }
};
template <int TPR, bool VEC, typename T>
__device__ __forceinline__ void store_row(const float (&v)[E], T *row, int t, int D) {
    if (VEC) {
        if (E * t < D) {
            st4(row + E * t, f4{v[0], v[1], v[2], v[3]});
            st4(row + E * t + 4, f4{v[4], v[5], v[6], v[7]});
        }
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int c = column<TPR, VEC>(j, t);
            if (c < D) st1(row + c, v[j]);
        }
    }
}
template <int TPR, bool VEC>
__device__ __forceinline__ void params(float (&o)[E], const float *w, int t, int D, float none) {
    if (VEC && w) {
        const bool ok = E * t < D;
        const float *q = w + (ok ? E * t : 0);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float v = q[j];
            o[j] = ok ? v : 0.0f;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int c = column<TPR, VEC>(j, t);
        o[j] = c < D ? (w ? w[c] : none) : 0.0f;
    }
}

// statistics of a row held in v: two passes over registers, so a large mean costs no digits
template <int TPR, bool VEC>
__device__ __forceinline__ void row_stats(const float (&v)[E], Red<TPR> &red, int t, int D, float invD, bool rms, float eps, float &mu, float &rs) {
    mu = 0.0f;
    if (!rms) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) s += v[j];
        mu = red.one(s) * invD;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = column<TPR, VEC>(j, t) < D ? v[j] - mu : 0.0f;
        q += d * d;
    }
    rs = 1.0f / sqrtf(red.one(q) * invD + eps);
}

template <int TPR, bool VEC, typename RT, typename IO>
__global__ __launch_bounds__(threads_of<TPR>()) void block_norm_fwd_kernel(const Args p) {
    constexpr int NT = threads_of<TPR>(), RPW = NT / TPR;
    __shared__ __attribute__((aligned(16))) float lds[4 * (NT / 64)];
    Red<TPR> red{lds};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = p.D;
    const float invD = 1.0f / (float)D;
    float w1[E], b1[E], a[E], w2[E], b2[E];
    params<TPR, VEC>(w1, p.w1, t, D, 1.0f);
    params<TPR, VEC>(b1, p.b1, t, D, 0.0f);
    params<TPR, VEC>(a, p.a, t, D, 1.0f);
    params<TPR, VEC>(w2, p.w2, t, D, 1.0f);
    params<TPR, VEC>(b2, p.b2, t, D, 0.0f);
    Piece<TPR, VEC, RT> px;
    Piece<TPR, VEC, IO> py, pz;
    // whole workgroups walk together (the sums of a row may use barriers): rows past the end repeat the last one and store nothing
    auto fetch = [&](long long r0) {
        const long long r = r0 + sub < p.rows ? r0 + sub : p.rows - 1;
        py.load(static_cast<const IO *>(p.y) + r * p.ldy, t, D);
        px.load(static_cast<const RT *>(p.x) + r * p.ldx, t, D);
        if (p.z) pz.load(static_cast<const IO *>(p.z) + r * p.ldz, t, D);
    };
    const long long step = (long long)gridDim.x * RPW;
    fetch((long long)blockIdx.x * RPW);
#pragma unroll 1
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += step) {
        const long long r = r0 + sub;
        float x[E], y[E], z[E];
        py.get(y, t, D);
        px.get(x, t, D);
        if (p.z) pz.get(z, t, D);
        fetch(r0 + step);
        const float drop = p.drop ? p.drop[(unsigned)(r < p.rows ? r : 0) / p.rps] : 1.0f;
        float m1, r1, m2, r2;
        row_stats<TPR, VEC>(y, red, t, D, invD, p.rms, p.eps, m1, r1);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float u = (y[j] - m1) * r1 * w1[j] + b1[j];
            if (p.z) u *= z[j] * sigmoidf_fast(z[j]);
            x[j] += drop * a[j] * u;                               // 0 past D
        }
        row_stats<TPR, VEC>(x, red, t, D, invD, p.rms, p.eps, m2, r2);
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = (x[j] - m2) * r2 * w2[j] + b2[j];
        if (r < p.rows) {
            store_row<TPR, VEC>(x, static_cast<RT *>(p.xo) + r * D, t, D);
            store_row<TPR, VEC>(y, static_cast<IO *>(p.h) + r * D, t, D);
            if (p.stats && t == 0) *reinterpret_cast<f4 *>(p.stats + 4 * r) = f4{m1, r1, m2, r2};
        }
    }
}

template <int TPR, bool VEC, typename RT, typename IO>
__global__ __launch_bounds__(threads_of<TPR>()) void block_norm_bwd_kernel(const Args p) {
    constexpr int NT = threads_of<TPR>(), RPW = NT / TPR;
    __shared__ __attribute__((aligned(16))) float lds[4 * (NT / 64)];
    __shared__ float cols[RPW > 1 ? NT * E : 1];
    Red<TPR> red{lds};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = p.D;
    const float invD = 1.0f / (float)D;
    // 1024 threads leave 128 registers each: parameters are read again for every row (from the cache), and rows are not fetched ahead
    constexpr bool LEAN = TPR == 1024;
    float w1[E], b1[E], a[E], w2[E];
    auto read_params = [&](int tt) {
        params<TPR, VEC>(w1, p.w1, tt, D, 1.0f);
        params<TPR, VEC>(b1, p.b1, tt, D, 0.0f);
        params<TPR, VEC>(a, p.a, tt, D, 1.0f);
        params<TPR, VEC>(w2, p.w2, tt, D, 1.0f);
    };
    if (!LEAN) read_params(t);
    float aw1[E], ab1[E], aa[E], aw2[E], ab2[E];
#pragma unroll
    for (int j = 0; j < E; ++j) aw1[j] = ab1[j] = aa[j] = aw2[j] = ab2[j] = 0.0f;
    Piece<TPR, VEC, RT> px, pg;
    Piece<TPR, VEC, IO> py, pz, ph;
    f4 st;
    auto fetch = [&](long long r0) {
        const long long r = r0 + sub < p.rows ? r0 + sub : p.rows - 1;
        st = *reinterpret_cast<const f4 *>(p.stats + 4 * r);
        py.load(static_cast<const IO *>(p.y) + r * p.ldy, t, D);
        px.load(static_cast<const RT *>(p.x) + r * p.ldx, t, D);
        if (p.z) pz.load(static_cast<const IO *>(p.z) + r * p.ldz, t, D);
        if (p.dh) ph.load(static_cast<const IO *>(p.dh) + r * D, t, D);
        if (p.dxo) pg.load(static_cast<const RT *>(p.dxo) + r * D, t, D);
    };
    const long long step = (long long)gridDim.x * RPW;
    if (!LEAN) fetch((long long)blockIdx.x * RPW);
#pragma unroll 1
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += step) {
        if (LEAN) {
            int tt = t;
            asm volatile("" : "+v"(tt));
            fetch(r0);
            read_params(tt);
        }
        const long long r = r0 + sub;
        const bool live = r < p.rows;
        float x[E], y[E], z[E], g[E], dh[E];
        py.get(y, t, D);
        px.get(x, t, D);
        if (p.z) pz.get(z, t, D);
        if (p.dh) ph.get(dh, t, D);
        if (p.dxo) pg.get(g, t, D);
        const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w, drop = p.drop ? p.drop[(unsigned)(live ? r : 0) / p.rps] : 1.0f;
        if (!LEAN) fetch(r0 + step);
        // y becomes its normalised value, x the normalised x', u = post-norm times gate; a row past the end adds nothing
        float u[E], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            dh[j] = p.dh && live ? dh[j] : 0.0f;
            g[j] = p.dxo && live ? g[j] : 0.0f;
            y[j] = (y[j] - m1) * r1;
            const float v = y[j] * w1[j] + b1[j];
            u[j] = p.z ? v * (z[j] * sigmoidf_fast(z[j])) : v;
            x[j] = (x[j] + drop * a[j] * u[j] - m2) * r2;
            const float d = dh[j] * w2[j];                             // 0 past D
            s1 += d;
            s2 += d * x[j];
            aw2[j] += dh[j] * x[j];
            ab2[j] += dh[j];
        }
        red.two(s1, s2);
        s1 = p.rms ? 0.0f : s1 * invD;
        s2 *= invD;
        float q1 = 0.0f, q2 = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            g[j] += r2 * (dh[j] * w2[j] - s1 - x[j] * s2);            // dx
            const float gd = g[j] * drop, du = gd * a[j];              // a is 0 past D
            aa[j] += gd * u[j];
            float dv = du;
            if (p.z) {
                const float v = y[j] * w1[j] + b1[j], sg = sigmoidf_fast(z[j]);
                dv = du * (z[j] * sg);
                z[j] = du * v * (sg * (1.0f + z[j] * (1.0f - sg)));   // dz
            }
            aw1[j] += dv * y[j];
            ab1[j] += dv;
            u[j] = dv * w1[j];
            q1 += u[j];
            q2 += u[j] * y[j];
        }
        red.two(q1, q2);
        q1 = p.rms ? 0.0f : q1 * invD;
        q2 *= invD;
#pragma unroll
        for (int j = 0; j < E; ++j) u[j] = r1 * (u[j] - q1 - y[j] * q2);  // dy
        if (live) {
            store_row<TPR, VEC>(g, static_cast<RT *>(p.dx) + r * D, t, D);
            store_row<TPR, VEC>(u, static_cast<IO *>(p.dy) + r * D, t, D);
            if (p.z) store_row<TPR, VEC>(z, static_cast<IO *>(p.dz) + r * D, t, D);
        }
    }
    // this workgroup's column sums
    float *dst = p.partials + (long long)blockIdx.x * 5 * D;
    auto put = [&](const float (&v)[E], int which) {
        if (RPW > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < E; ++j) cols[(sub * E + j) * TPR + t] = v[j];
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float s = 0.0f;
#pragma unroll
                    for (int k = 0; k < RPW; ++k) s += cols[(k * E + j) * TPR + t];
                    const int c = column<TPR, VEC>(j, t);
                    if (c < D) dst[which * D + c] = s;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int c = column<TPR, VEC>(j, t);
                if (c < D) dst[which * D + c] = v[j];
            }
        }
    };
    put(aw1, 0); put(ab1, 1); put(aa, 2); put(aw2, 3); put(ab2, 4);
}

// out (5, D) = sum of the workgroups' partial rows in a fixed order: 16 columns x 16 row lanes a workgroup, eight loads in flight
__global__ __launch_bounds__(256) void block_norm_cols_kernel(const float *partials, float *out, int n, int wgs) {
    __shared__ float red[256];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    float s = 0.0f;
    if (c < n) {
        int w = part;
        for (; w + 112 < wgs; w += 128) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = partials[(long long)(w + 16 * u) * n + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; w < wgs; w += 16) s += partials[(long long)w * n + c];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (part == 0 && c < n) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[16 * k + threadIdx.x];
        out[c] = s;
    }
}

int tpr_of(int D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }
int bwd_wgs(long long rows, int D) {      // as many as are resident at once: every workgroup leaves a partial row
    const int tpr = tpr_of(D), rpw = tpr > 256 ? 1 : 256 / tpr, most = tpr > 256 ? 256 : 512;
    const long long n = (rows + rpw - 1) / rpw;
    return (int)(n < most ? n : most);
}

template <int TPR, bool VEC, typename RT, typename IO>
void launch_one(bool bwd, const Args &p, hipStream_t s) {
    constexpr int NT = threads_of<TPR>(), RPW = NT / TPR;
    if (!bwd) {
        long long n = (p.rows + RPW - 1) / RPW;
        const long long most = NT > 256 ? 512 : 1024;
        if (n > most) n = most;
        ss2d_launch((block_norm_fwd_kernel<TPR, VEC, RT, IO>), dim3((unsigned)n), dim3(NT), 0, s, p);
    } else {
        ss2d_launch((block_norm_bwd_kernel<TPR, VEC, RT, IO>), dim3((unsigned)bwd_wgs(p.rows, p.D)), dim3(NT), 0, s, p);
    }
}
template <bool VEC, typename RT, typename IO>
void launch(bool bwd, const Args &p, hipStream_t s) {
    switch (tpr_of(p.D)) {
        case 16: launch_one<16, VEC, RT, IO>(bwd, p, s); break;
        case 64: launch_one<64, VEC, RT, IO>(bwd, p, s); break;
        case 128: launch_one<128, VEC, RT, IO>(bwd, p, s); break;
        case 256: launch_one<256, VEC, RT, IO>(bwd, p, s); break;
        case 512: launch_one<512, VEC, RT, IO>(bwd, p, s); break;
        default: launch_one<1024, VEC, RT, IO>(bwd, p, s); break;
    }
}
template <typename RT, typename IO>
void launch(bool bwd, bool vec, const Args &p, hipStream_t s) { vec ? launch<true, RT, IO>(bwd, p, s) : launch<false, RT, IO>(bwd, p, s); }
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
    ss2d_launch(block_norm_cols_kernel, dim3((unsigned)((5 * D + 15) / 16)), dim3(256), 0, (hipStream_t)stream, workspace, dparams, 5 * D, bwd_wgs(rows, D));
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("block_norm_bwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
