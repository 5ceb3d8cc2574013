// One new token of linear attention for each of B requests (formulas: ss2d_linattn.h), for gfx950: the recurrent form
//     S <- exp(g) S + k v^T,   o = scale * S^T q
// on the states of a pool, in place.  Bound by the state: dk * dv fp32 values are read and written once for every request and head, all
// else is small.  A workgroup takes one (request, head) and a slice of dv: its threads hold the slice in registers (four columns x every
// RG-th row each), so every state element is loaded once, updated, stored and multiplied into the output, and the partial sums over dk
// meet in LDS.  Measured: 250 requests, 32 heads of 128 x 64, 93 us (527 MB, 5.7 TB/s, some of it from the last-level cache; 111 with a cold one); one request,
// 16 heads of 64 x 64, 4.7 us, a launch; 128 requests, 16 heads of 64 x 65 (a second workgroup for the last column) 27 us, of 64 x 64 16.
//
// With slot indices two requests may name one slot.  Then the first of them applies all of that slot's tokens in request order,
// and the others leave: the result does not depend on the order of execution.  Every workgroup looks through all B indices for that, which costs
// nothing up to a thousand requests and more than the states beyond ten thousand (4 heads of 64 x 64, us without / with indices: 1024 requests 25 / 29, 4096 97 / 139,
// 16384 392 / 911).
#include "ss2d_common.h"
#include "../../include/ss2d.h"

namespace {

constexpr int NT = 256, NC = 16;

struct StepArgs {
    float *state;
    const void *q, *k, *v;
    const float *g;
    void *o;
    const void *idx;              // request -> slot: int32 or int64; null: slot = request
    long long slot_stride, pool;
    long long qb, qh, kb, kh, vb, vh, gb, gh;
    int B, H, G, dk, dv, idx64;
    float scale;
};

__device__ __forceinline__ long long slot_of(const StepArgs &a, int b) {
    if (!a.idx) return b;
    return a.idx64 ? static_cast<const long long *>(a.idx)[b] : (long long)static_cast<const int *>(a.idx)[b];
}

// Four neighbouring columns of a row that lies on any 32-bit word; the last group of a row may hold less than four (n: what is left of the row)
typedef f4 __attribute__((aligned(4))) f4_any;
__device__ __forceinline__ f4 load_columns(const float *s, int n) {
    if (n >= 4) return *reinterpret_cast<const f4_any *>(s);
    return f4{n > 0 ? s[0] : 0.0f, n > 1 ? s[1] : 0.0f, n > 2 ? s[2] : 0.0f, 0.0f};
}
__device__ __forceinline__ void store_columns(float *s, int n, f4 v) {
    if (n >= 4) { *reinterpret_cast<f4_any *>(s) = v; return; }
    if (n > 0) s[0] = v.x;
    if (n > 1) s[1] = v.y;
    if (n > 2) s[2] = v.z;
}

// NC groups of four columns a workgroup; RG = 256 / NC rows are in flight per trip, NR trips cover dk
template <int NR, typename IO>
__global__ __launch_bounds__(NT) void la_step_kernel(const StepArgs a) {
    constexpr int RG = NT / NC;
    __shared__ float red[RG][NC * 4 + 1];
    const int tid = threadIdx.x, cg = tid % NC, rg = tid / NC;
    const int tiles = (a.dv + NC * 4 - 1) / (NC * 4);
    int id = blockIdx.x;
    const int tile = id % tiles; id /= tiles;
    const int h = id % a.H, b0 = id / a.H;
    const int c0 = (tile * NC + cg) * 4, left = a.dv - c0;  // columns of the row from c0 on
    IO *O = static_cast<IO *>(a.o);
    const long long slot = slot_of(a, b0);
    if (slot < 0 || slot >= a.pool) {                      // no state: the output is zero
        if (rg == 0)
            for (int e = 0; e < 4 && e < left; ++e) st1(O + ((long long)b0 * a.H + h) * a.dv + c0 + e, 0.0f);
        return;
    }
    float *S = a.state + slot * a.slot_stride + (long long)h * a.dk * a.dv + c0;
    f4 s[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int k = rg + RG * r;
        s[r] = load_columns(S + (long long)k * a.dv, k < a.dk ? left : 0);
    }
    int last = b0;                                         // the last request of this slot
    if (a.idx) {
        int before = 0, after = -1;
        for (int b = tid; b < a.B; b += NT)
            if (b != b0 && slot_of(a, b) == slot) { if (b < b0) before = 1; else after = b; }
        if (__syncthreads_or(before)) return;
        if (__syncthreads_or(after >= 0)) last = a.B - 1;
    }
    const int hk = h / (a.H / a.G);
    for (int b = b0; b <= last; ++b) {
        if (b != b0 && slot_of(a, b) != slot) continue;
        const IO *q = static_cast<const IO *>(a.q) + b * a.qb + hk * a.qh;
        const IO *kk = static_cast<const IO *>(a.k) + b * a.kb + hk * a.kh;
        const IO *v = static_cast<const IO *>(a.v) + b * a.vb + h * a.vh + c0;
        const float decay = expf(a.g[b * a.gb + h * a.gh]);
        f4 vv, o = f4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) vv[e] = e < left ? ld1(v + e) : 0.0f;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int k = rg + RG * r;
            if (k < a.dk) {
                const float kv = ld1(kk + k), qv = ld1(q + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[r][e] = fmaf(s[r][e], decay, kv * vv[e]);
                    o[e] = fmaf(s[r][e], qv, o[e]);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) red[rg][cg * 4 + e] = o[e];
        __syncthreads();
        if (tid < NC * 4) {
            const int c = tile * NC * 4 + tid;
            float t = 0.0f;
#pragma unroll
            for (int r = 0; r < RG; ++r) t += red[r][tid];
            if (c < a.dv) st1(O + ((long long)b * a.H + h) * a.dv + c, t * a.scale);
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int k = rg + RG * r;
        store_columns(S + (long long)k * a.dv, k < a.dk ? left : 0, s[r]);
    }
}

template <typename IO>
void launch(const StepArgs &a, hipStream_t s) {
    constexpr int RG = NT / NC;
    const int tiles = (a.dv + NC * 4 - 1) / (NC * 4), nr = (a.dk + RG - 1) / RG;
    const dim3 grid((unsigned)((long long)a.B * a.H * tiles));
    if (nr <= 1) ss2d_launch((la_step_kernel<1, IO>), grid, dim3(NT), 0, s, a);
    else if (nr <= 2) ss2d_launch((la_step_kernel<2, IO>), grid, dim3(NT), 0, s, a);
    else if (nr <= 4) ss2d_launch((la_step_kernel<4, IO>), grid, dim3(NT), 0, s, a);
    else ss2d_launch((la_step_kernel<8, IO>), grid, dim3(NT), 0, s, a);
}

}  // namespace

extern "C" int ss2d_linattn_step(int dtype, float *state, const void *q, const void *k, const void *v, const float *g, const long long *strides,
                                 const void *slots, int slots64, void *out, long long pool, long long slot_stride, int B, int H, int G, int dk,
                                 int dv, float scale, void *stream) {
    if (dtype != SS2D_DTYPE_F32 && dtype != SS2D_DTYPE_BF16) { ss2d_set_error("linattn_step: unknown dtype %d", dtype); return -1; }
    if (!state || !q || !k || !v || !g || !strides || !out) { ss2d_set_error("linattn_step: null pointer"); return -2; }
    if (B <= 0 || H <= 0 || G <= 0 || pool <= 0) { ss2d_set_error("linattn_step: non-positive size"); return -3; }
    if (H % G) { ss2d_set_error("linattn_step: %d heads are not a multiple of %d key heads", H, G); return -4; }
    if (dk < 1 || dk > 128 || dv < 1 || dv > 128) { ss2d_set_error("linattn_step: dk %d and dv %d must be 1 ... 128", dk, dv); return -5; }
    if (slot_stride < (long long)H * dk * dv) { ss2d_set_error("linattn_step: slots overlap (stride %lld)", slot_stride); return -4; }
    if ((long long)B * H * 8 > 0x7fffffffLL) { ss2d_set_error("linattn_step: too many requests and heads"); return -6; }
    if (!slots && pool < B) { ss2d_set_error("linattn_step: %d requests, %lld states", B, pool); return -3; }
    StepArgs a{state, q, k, v, g, out, slots, slot_stride, pool, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7],
               B, H, G, dk, dv, slots64, scale};
    if (dtype == SS2D_DTYPE_BF16) launch<bf16>(a, (hipStream_t)stream); else launch<float>(a, (hipStream_t)stream);
    const int rc = ss2d_take_launch_rc();
    if (rc) ss2d_set_error("linattn_step: launch failed: %s", hipGetErrorString((hipError_t)rc));
    return rc;
}
