// The norms around a block, with its gate and residual scale, in one pass (gfx950):
//     u = norm(y; w1, b1) * SiLU(z),   x' = x + drop * a * u,   h = norm(x'; w2, b2)
// norm: LayerNorm or RMS norm over the last axis (fp32 statistics); y is the block's output, z its gate, a a per-channel residual scale, drop a
// per-sample factor, x the residual stream and h the next block's input.  Beside ss2d_outnorm_gate (norm and gate in front of a projection) and
// ss2d_layernorm: there the residual stream makes a round trip through memory between the two norms.
//
// Memory-bound.  TPR threads hold one row, eight elements each (16 bytes of bf16), so x, y and z are read once and x', h written once; h's statistics are those of the unrounded x'.  A thread's parameters
// stay in registers over all its rows, and the next row is in flight while one is worked on.  The backward recomputes x' from x, y, z (the
// same bytes as reading a saved x') and holds its share of the five column sums in registers; the workgroups' sums go to a workspace and
// are added in a fixed order.
// Measured: 65536 rows of 768 bf16 with fp32 residual, forward and backward, 3.8 TB/s; 16384 rows of 4096 bf16 128 us forward (5.2 TB/s) and
// 246 + 8 us backward (5.0 TB/s); a 1 GB copy reaches 5.0 TB/s.
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
            constexpr int W = TPR > 64 ? TPR / 64 : 1;
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

// A thread's eight columns, base + j, of which those with j >= skip are its own.  Rows made of whole groups of eight (VEC): all or none.  Else the last
// group is moved back to end with the row, so that every group is read and written as 16-byte pieces at whatever alignment they fall on (fp32
// rows of 1001: 4.9 TB/s, as fast as rows of 1000; held element by element, bf16 rows of 4100 took 3.3 times as long); base is negative in rows
// of less than eight.
struct Place {
    int base, skip;
};
template <bool VEC>
__device__ __forceinline__ Place place_of(int t, int D) {
    const int c = E * t;
    if (VEC) return c < D ? Place{c, 0} : Place{0, E};
    if (c >= D) return Place{D < E ? D - E : 0, E};
    return c + E <= D ? Place{c, 0} : Place{D - E, c + E - D};
}

// a thread's share of a row as it lies in memory; columns that are not its own come out as 0
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef f4 __attribute__((aligned(4))) f4_any;
template <int TPR, bool VEC, typename T>
struct Piece {
    static constexpr int N = sizeof(T) == 2 ? 1 : 2;
    u32x4 v[N];
    __device__ __forceinline__ void load(const T *row, Place at, int D) {
        if (VEC || TPR > 16 || D >= E) {                               // more than 16 threads a row: D > 128
            const u32x4_any *q = reinterpret_cast<const u32x4_any *>(row + at.base);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = q[i];
        } else {
            T s[E];
#pragma unroll
            for (int j = 0; j < E; ++j) s[j] = row[at.base + j > 0 ? at.base + j : 0];
            __builtin_memcpy(v, s, sizeof(s));
        }
    }
    __device__ __forceinline__ void get(float (&o)[E], Place at) const {
        if (sizeof(T) == 2) {
            const unsigned w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[2 * i] = __builtin_bit_cast(float, w[i] << 16);
                o[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
            }
        } else {
            const u32x4 a = v[0], b = v[N - 1];
            const unsigned w[E] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] = __builtin_bit_cast(float, w[j]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = (VEC ? 0 : j) >= at.skip ? o[j] : 0.0f;
    }
};
__device__ __forceinline__ void store8(const float (&v)[E], float *q) {
    *reinterpret_cast<f4_any *>(q) = f4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f4_any *>(q + 4) = f4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(const float (&v)[E], bf16 *q) {
    bf16 s[E];
    u32x4 w;
#pragma unroll
    for (int j = 0; j < E; ++j) s[j] = (bf16)v[j];
    __builtin_memcpy(&w, s, 16);
    *reinterpret_cast<u32x4_any *>(q) = w;
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_row(const float (&v)[E], T *row, Place at) {
    if (at.skip == 0) {
        store8(v, row + at.base);
    } else if (!VEC) {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j >= at.skip) st1(row + at.base + j, v[j]);
    }
}
// statistics of a row held in v: two passes over registers, so a large mean costs no digits
template <bool VEC, int TPR>
__device__ __forceinline__ void row_stats(const float (&v)[E], Red<TPR> &red, Place at, float invD, bool rms, float eps, float &mu, float &rs) {
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
        const float d = (VEC ? 0 : j) >= at.skip ? v[j] - mu : 0.0f;
        q += d * d;
    }
    rs = 1.0f / sqrtf(red.one(q) * invD + eps);
}

// Four columns of a parameter: own columns 4 i .. 4 i + 3 of the thread, 0 in others
template <int TPR, bool VEC>
__device__ __forceinline__ f4 param4(const float *w, int i, Place at, int D, float none) {
    f4 q{none, none, none, none};
    if (w && (VEC || TPR > 16 || D >= E)) {
        q = *reinterpret_cast<const f4_any *>(w + (unsigned)at.base + 4 * i);
    } else if (w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = w[(VEC ? 0 : 4 * i + e) >= at.skip ? at.base + 4 * i + e : 0];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = (VEC ? 0 : 4 * i + e) >= at.skip ? q[e] : 0.0f;
    return q;
}
// K rows of per-column values of a thread, in fours: in registers, or (HELD) in LDS, each thread its own 16-byte slots, a wave's side by side.
// 1024 threads have 128 registers each, which hold a row but not the parameters of the forward or the column sums of the backward besides.
template <int NT, int K, bool HELD>
struct Columns {
    static constexpr int SLOTS = HELD ? 2 * K * NT : 1;
    f4 r[HELD ? 1 : 2 * K];
    f4 *mine;
    __device__ __forceinline__ explicit Columns(f4 *lds) : mine(lds + (HELD ? threadIdx.x : 0)) {}
    __device__ __forceinline__ f4 get(int k, int i) const { return HELD ? mine[(2 * k + i) * NT] : r[HELD ? 0 : 2 * k + i]; }
    __device__ __forceinline__ void set(int k, int i, f4 v) {
        if (HELD) mine[(2 * k + i) * NT] = v;
        else r[HELD ? 0 : 2 * k + i] = v;
    }
    __device__ __forceinline__ void add(int k, int i, f4 v) { set(k, i, get(k, i) + v); }
};

template <int TPR, bool VEC, typename RT, typename IO>
__global__ __launch_bounds__(threads_of<TPR>()) void block_norm_fwd_kernel(const Args p) {
    constexpr int NT = threads_of<TPR>(), RPW = NT / TPR;
    __shared__ __attribute__((aligned(16))) float lds[4 * (NT / 64)];
    Red<TPR> red{lds};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = p.D;
    const float invD = 1.0f / (float)D;
    const Place at = place_of<VEC>(t, D);
    __shared__ f4 held[Columns<NT, 4, TPR == 1024>::SLOTS];
    Columns<NT, 4, TPR == 1024> par(held);                         // w1, b1, a, w2
    f4 b2[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        par.set(0, i, param4<TPR, VEC>(p.w1, i, at, D, 1.0f));
        par.set(1, i, param4<TPR, VEC>(p.b1, i, at, D, 0.0f));
        par.set(2, i, param4<TPR, VEC>(p.a, i, at, D, 1.0f));
        par.set(3, i, param4<TPR, VEC>(p.w2, i, at, D, 1.0f));
        b2[i] = param4<TPR, VEC>(p.b2, i, at, D, 0.0f);
    }
    Piece<TPR, VEC, RT> px;
    Piece<TPR, VEC, IO> py, pz;
    // whole workgroups walk together (the sums of a row may use barriers): rows past the end repeat the last one and store nothing
    auto fetch = [&](long long r0) {
        const long long r = r0 + sub < p.rows ? r0 + sub : p.rows - 1;
        py.load(static_cast<const IO *>(p.y) + r * p.ldy, at, D);
        px.load(static_cast<const RT *>(p.x) + r * p.ldx, at, D);
        if (p.z) pz.load(static_cast<const IO *>(p.z) + r * p.ldz, at, D);
    };
    const long long step = (long long)gridDim.x * RPW;
    fetch((long long)blockIdx.x * RPW);
#pragma unroll 1
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += step) {
        const long long r = r0 + sub;
        float x[E], y[E], z[E];
        py.get(y, at);
        px.get(x, at);
        if (p.z) pz.get(z, at);
        fetch(r0 + step);
        const float drop = p.drop ? p.drop[(unsigned)(r < p.rows ? r : 0) / p.rps] : 1.0f;
        float m1, r1, m2, r2;
        row_stats<VEC>(y, red, at, invD, p.rms, p.eps, m1, r1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f4 w1 = par.get(0, i), b1 = par.get(1, i), a = par.get(2, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = 4 * i + e;
                float u = (y[j] - m1) * r1 * w1[e] + b1[e];
                if (p.z) u *= z[j] * sigmoidf_fast(z[j]);
                x[j] += drop * a[e] * u;                           // 0 in columns that are not its own
            }
        }
        row_stats<VEC>(x, red, at, invD, p.rms, p.eps, m2, r2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f4 w2 = par.get(3, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[4 * i + e] = (x[4 * i + e] - m2) * r2 * w2[e] + b2[i][e];
        }
        if (r < p.rows) {
            store_row<VEC>(x, static_cast<RT *>(p.xo) + r * D, at);
            store_row<VEC>(y, static_cast<IO *>(p.h) + r * D, at);
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
    const Place at = place_of<VEC>(t, D);
    // 1024 threads: four of the five column sums lie in LDS, and the parameters are read again where they are used
    constexpr bool LEAN = TPR == 1024;
    __shared__ f4 held[Columns<NT, 4, LEAN>::SLOTS];
    Columns<NT, 4, LEAN> sum(held);                                // of w1, b1, w2, b2
    f4 w1s[2], b1s[2], as[2], w2s[2], suma[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        suma[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; ++k) sum.set(k, i, suma[i]);
        if (!LEAN) {
            w1s[i] = param4<TPR, VEC>(p.w1, i, at, D, 1.0f);
            b1s[i] = param4<TPR, VEC>(p.b1, i, at, D, 0.0f);
            as[i] = param4<TPR, VEC>(p.a, i, at, D, 1.0f);
            w2s[i] = param4<TPR, VEC>(p.w2, i, at, D, 1.0f);
        }
    }
    Piece<TPR, VEC, RT> px, pg;
    Piece<TPR, VEC, IO> py, pz, ph;
    f4 st;
    auto fetch = [&](long long r0) {
        const long long r = r0 + sub < p.rows ? r0 + sub : p.rows - 1;
        st = *reinterpret_cast<const f4 *>(p.stats + 4 * r);
        py.load(static_cast<const IO *>(p.y) + r * p.ldy, at, D);
        px.load(static_cast<const RT *>(p.x) + r * p.ldx, at, D);
        if (p.z) pz.load(static_cast<const IO *>(p.z) + r * p.ldz, at, D);
        if (p.dh) ph.load(static_cast<const IO *>(p.dh) + r * D, at, D);
        if (p.dxo) pg.load(static_cast<const RT *>(p.dxo) + r * D, at, D);
    };
    const long long step = (long long)gridDim.x * RPW;
    fetch((long long)blockIdx.x * RPW);
#pragma unroll 1
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < p.rows; r0 += step) {
        const long long r = r0 + sub;
        const bool live = r < p.rows;
        float x[E], y[E], z[E], g[E], dh[E];
        py.get(y, at);
        px.get(x, at);
        if (p.z) pz.get(z, at);
        if (p.dh) ph.get(dh, at);
        if (p.dxo) pg.get(g, at);
        const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w, drop = p.drop ? p.drop[(unsigned)(live ? r : 0) / p.rps] : 1.0f;
        if (!LEAN) fetch(r0 + step);
        // y becomes its normalised value, x the normalised x'; a row past the end adds nothing
        float u[E], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f4 w1 = LEAN ? param4<TPR, VEC>(p.w1, i, at, D, 1.0f) : w1s[i], b1 = LEAN ? param4<TPR, VEC>(p.b1, i, at, D, 0.0f) : b1s[i];
            const f4 a = LEAN ? param4<TPR, VEC>(p.a, i, at, D, 1.0f) : as[i], w2 = LEAN ? param4<TPR, VEC>(p.w2, i, at, D, 1.0f) : w2s[i];
            f4 m, n;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = 4 * i + e;
                dh[j] = p.dh && live ? dh[j] : 0.0f;
                g[j] = p.dxo && live ? g[j] : 0.0f;
                y[j] = (y[j] - m1) * r1;
                const float v = y[j] * w1[e] + b1[e], uj = p.z ? v * (z[j] * sigmoidf_fast(z[j])) : v;
                x[j] = (x[j] + drop * a[e] * uj - m2) * r2;
                const float d = dh[j] * w2[e];                          // 0 in columns that are not its own
                s1 += d;
                s2 += d * x[j];
                m[e] = dh[j] * x[j];
                n[e] = dh[j];
            }
            sum.add(2, i, m);
            sum.add(3, i, n);
        }
        red.two(s1, s2);
        if (LEAN) {                                                    // taken as new, so that nothing made from them above is kept for below
#pragma unroll
            for (int j = 0; j < E; ++j) asm volatile("" : "+v"(y[j]), "+v"(z[j]));
        }
        s1 = p.rms ? 0.0f : s1 * invD;
        s2 *= invD;
        float q1 = 0.0f, q2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f4 w1 = LEAN ? param4<TPR, VEC>(p.w1, i, at, D, 1.0f) : w1s[i], b1 = LEAN ? param4<TPR, VEC>(p.b1, i, at, D, 0.0f) : b1s[i];
            const f4 a = LEAN ? param4<TPR, VEC>(p.a, i, at, D, 1.0f) : as[i], w2 = LEAN ? param4<TPR, VEC>(p.w2, i, at, D, 1.0f) : w2s[i];
            f4 m, n;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = 4 * i + e;
                g[j] += r2 * (dh[j] * w2[e] - s1 - x[j] * s2);        // dx
                const float gd = g[j] * drop, du = gd * a[e];           // a is 0 in columns that are not its own
                const float v = y[j] * w1[e] + b1[e];
                float dv = du, gate = 1.0f;
                if (p.z) {
                    const float sg = sigmoidf_fast(z[j]);
                    gate = z[j] * sg;
                    dv = du * gate;
                    z[j] = du * v * (sg * (1.0f + z[j] * (1.0f - sg)));   // dz
                }
                suma[i][e] += gd * (v * gate);
                m[e] = dv * y[j];
                n[e] = dv;
                u[j] = dv * w1[e];
                q1 += u[j];
                q2 += u[j] * y[j];
            }
            sum.add(0, i, m);
            sum.add(1, i, n);
        }
        if (LEAN) fetch(r0 + step);
        red.two(q1, q2);
        q1 = p.rms ? 0.0f : q1 * invD;
        q2 *= invD;
#pragma unroll
        for (int j = 0; j < E; ++j) u[j] = r1 * (u[j] - q1 - y[j] * q2);  // dy
        if (live) {
            store_row<VEC>(g, static_cast<RT *>(p.dx) + r * D, at);
            store_row<VEC>(u, static_cast<IO *>(p.dy) + r * D, at);
            if (p.z) store_row<VEC>(z, static_cast<IO *>(p.dz) + r * D, at);
        }
    }
    // this workgroup's column sums
    float *dst = p.partials + (long long)blockIdx.x * 5 * D;
    auto put = [&](int which, f4 lo, f4 hi) {
        float v[E];
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
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
                    if ((VEC ? 0 : j) >= at.skip) dst[which * D + at.base + j] = s;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if ((VEC ? 0 : j) >= at.skip) dst[which * D + at.base + j] = v[j];
        }
    };
    put(0, sum.get(0, 0), sum.get(0, 1));
    put(1, sum.get(1, 0), sum.get(1, 1));
    put(2, suma[0], suma[1]);
    put(3, sum.get(2, 0), sum.get(2, 1));
    put(4, sum.get(3, 0), sum.get(3, 1));
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
    dispatch(false, res_dtype, dtype, D % E == 0, p, (hipStream_t)stream);
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
    dispatch(true, res_dtype, dtype, D % E == 0, p, (hipStream_t)stream);
    ss2d_launch(block_norm_cols_kernel, dim3((unsigned)((5 * D + 15) / 16)), dim3(256), 0, (hipStream_t)stream, workspace, dparams, 5 * D, bwd_wgs(rows, D));
    rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("block_norm_bwd: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
