// One new token of linear attention for each of B requests (formulas: ss2d_linattn.h), for gfx950: the recurrent form
//     S <- exp(g) S + k v^T,   o = scale * S^T q
// on the states of a pool, in place.  Bound by the state: dk * dv fp32 values are read and written once for every request and head, all
// else is small.  A workgroup takes one (request, head) and a slice of dv: its threads hold the slice in registers (VW columns x every
// RG-th row each), so every state element is loaded once, updated, stored and multiplied into the output, and the partial sums over dk
// meet in LDS.
//
// With slot indices two requests may name one slot.  Then the first of them applies all of that slot's tokens in request order,
// and the others leave: the result does not depend on the order of execution.
#include "ss2d_common.h"
#include "../../include/ss2d.h"

namespace {

constexpr int NT = 256;

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

// NC: column groups of VW columns a workgroup (a power of two); RG = 256 / NC rows are in flight per trip; NR trips cover dk
template <int VW, int NC, int NR, typename IO>
__global__ __launch_bounds__(NT) void la_step_kernel(const StepArgs a) {
    constexpr int RG = NT / NC;
    __shared__ float red[RG][NC * VW + 1];
    const int tid = threadIdx.x, cg = tid % NC, rg = tid / NC;
    const int tiles = (a.dv + NC * VW - 1) / (NC * VW);
    int id = blockIdx.x;
    const int tile = id % tiles; id /= tiles;
    const int h = id % a.H, b0 = id / a.H;
    const int c0 = (tile * NC + cg) * VW;
    const bool cok = c0 < a.dv;                            // VW > 1 only with dv a multiple of VW
    IO *O = static_cast<IO *>(a.o);
    const long long slot = slot_of(a, b0);
    if (slot < 0 || slot >= a.pool) {                      // no state: the output is zero
        if (rg == 0 && cok)
            for (int e = 0; e < VW; ++e) st1(O + ((long long)b0 * a.H + h) * a.dv + c0 + e, 0.0f);
        return;
    }
    float *S = a.state + slot * a.slot_stride + (long long)h * a.dk * a.dv + c0;
    float s[NR][VW];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int k = rg + RG * r;
        const bool ok = cok && k < a.dk;
        if (VW == 4) {
            const f4 t = *reinterpret_cast<const f4 *>(ok ? S + (long long)k * a.dv : a.state);
            s[r][0] = t.x; s[r][VW > 1 ? 1 : 0] = VW > 1 ? t.y : t.x; s[r][VW > 2 ? 2 : 0] = VW > 2 ? t.z : t.x; s[r][VW > 3 ? 3 : 0] = VW > 3 ? t.w : t.x;
        } else {
            s[r][0] = ok ? S[(long long)k * a.dv] : 0.0f;
        }
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
        float vv[VW], o[VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) { vv[e] = cok ? ld1(v + e) : 0.0f; o[e] = 0.0f; }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int k = rg + RG * r;
            if (k < a.dk) {
                const float kv = ld1(kk + k), qv = ld1(q + k);
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    s[r][e] = fmaf(s[r][e], decay, kv * vv[e]);
                    o[e] = fmaf(s[r][e], qv, o[e]);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < VW; ++e) red[rg][cg * VW + e] = o[e];
        __syncthreads();
        if (tid < NC * VW) {
            const int c = tile * NC * VW + tid;
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
        if (cok && k < a.dk) {
            if (VW == 4) *reinterpret_cast<f4 *>(S + (long long)k * a.dv) = f4{s[r][0], s[r][VW > 1 ? 1 : 0], s[r][VW > 2 ? 2 : 0], s[r][VW > 3 ? 3 : 0]};
            else S[(long long)k * a.dv] = s[r][0];
        }
    }
}

template <int VW, int NC, typename IO>
void launch_nc(const StepArgs &a, hipStream_t s) {
    constexpr int RG = NT / NC;
    const int tiles = (a.dv + NC * VW - 1) / (NC * VW), nr = (a.dk + RG - 1) / RG;
    const dim3 grid((unsigned)((long long)a.B * a.H * tiles));
    if (nr <= 1) ss2d_launch((la_step_kernel<VW, NC, 1, IO>), grid, dim3(NT), 0, s, a);
    else if (nr <= 2) ss2d_launch((la_step_kernel<VW, NC, 2, IO>), grid, dim3(NT), 0, s, a);
    else if (nr <= 4) ss2d_launch((la_step_kernel<VW, NC, 4, IO>), grid, dim3(NT), 0, s, a);
    else if (nr <= 8) ss2d_launch((la_step_kernel<VW, NC, 8, IO>), grid, dim3(NT), 0, s, a);
    else ss2d_launch((la_step_kernel<VW, NC, 128 / RG < 1 ? 1 : 128 / RG, IO>), grid, dim3(NT), 0, s, a);
}

template <typename IO>
void launch(const StepArgs &a, hipStream_t s) {
    if (a.dv % 4 == 0 && ((uintptr_t)a.state % 16) == 0 && a.slot_stride % 4 == 0) launch_nc<4, 16, IO>(a, s);
    else launch_nc<1, 64, IO>(a, s);
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
