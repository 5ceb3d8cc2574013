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
    int nseg, segc;               // segments a sequence may have (1: not split), chunks a segment
    int slots;                    // segments of all sequences: the walks of a head
    int vec;                      // rows are made of 16-byte pieces that begin on 32-bit words
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
// Segments.  A batch has nseg of each sequence, the last one takes whatever is left.  Packed sequences have as many as they need: floor(start / span) + n is
// a sequence's first slot, which leaves room for every earlier sequence's last, partly filled segment, and a walk finds its sequence by bisection.
__device__ __forceinline__ int first_slot(const Problem &p, int n, int C) {
    if (!p.cu || p.nseg == 1) return n * p.nseg;
    const long long a = p.cu[n];
    return (int)((unsigned)(a < 0 ? 0 : a > p.tokens ? p.tokens : a) / (unsigned)(p.segc * C)) + n;
}
__device__ __forceinline__ void walk_of(const Problem &p, int slot, int C, int &n, int &seg) {       // seg < 0: a slot of no sequence
    if (!p.cu || p.nseg == 1) {
        n = slot / p.nseg;
        seg = slot % p.nseg;
        return;
    }
    int lo = 0, hi = p.N - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_slot(p, mid, C) <= slot) lo = mid;
        else hi = mid - 1;
    }
    n = lo;
    seg = slot - first_slot(p, lo, C);
}
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
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double b) {          // b + (b of the lane that CTRL names; 0 where there is none or the row is not in ROWS)
    const long long u = __builtin_bit_cast(long long, b);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return b + __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}
__device__ __forceinline__ double chunk_decay_scan(float g) {
    double b = (double)g * 1.4426950408889634074;
    b = dpp_add<DPP_ROW_SHR(1), 0xf>(b);
    b = dpp_add<DPP_ROW_SHR(2), 0xf>(b);
    b = dpp_add<DPP_ROW_SHR(4), 0xf>(b);
    b = dpp_add<DPP_ROW_SHR(8), 0xf>(b);
    b = dpp_add<0x142, 0xa>(b);                                // lane 15 of rows 0 and 2 into rows 1 and 3
    return dpp_add<0x143, 0xc>(b);                             // lane 31 into rows 2 and 3
}
__device__ __forceinline__ double lane63(double b) {
    const long long u = __builtin_bit_cast(long long, b);
    const unsigned lo = __builtin_amdgcn_readlane((int)u, 63), hi = __builtin_amdgcn_readlane((int)(u >> 32), 63);
    return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}

// a value that the compiler takes as new: addresses made from it are computed where they are used instead of living across a loop
__device__ __forceinline__ int fresh(int v) { asm volatile("" : "+v"(v)); return v; }

// ---- bf16 operands on v_mfma_f32_16x16x32_bf16.  A lane (l16 = lane & 15, gq = lane >> 4) holds row / column l16 of an operand and eight of the 32
// contracted indices.  Here they are 4 gq + {0..3} and 16 + 4 gq + {0..3} for every operand: the two halves are then exactly the rows that
// the lane holds of two neighbouring 16 x 16 results, so a state in accumulators is an operand without moving data.
// fp32 factors (states, weighted values, weights) enter as sums of three bf16 values, which leave nothing of their 24 bits.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f4 mfma8(bf16x8 a, bf16x8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ bf16x8 join8(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ bf16x4 round4(f4 v) { return __builtin_convertvector(v, bf16x4); }
// v minus its rounded value; the halves are taken from the packed words (converted back one by one, the compiler rounds them a second time)
__device__ __forceinline__ f4 rest4(f4 v, bf16x4 h) {
    const u32x2 w = __builtin_bit_cast(u32x2, h);
    const unsigned a = w.x, b = w.y;
    return f4{v.x - __builtin_bit_cast(float, a << 16), v.y - __builtin_bit_cast(float, a & 0xffff0000u), v.z - __builtin_bit_cast(float, b << 16),
              v.w - __builtin_bit_cast(float, b & 0xffff0000u)};
}
__device__ __forceinline__ void widen8(bf16x8 v, f4 &a, f4 &b) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    const unsigned w0 = w.x, w1 = w.y, w2 = w.z, w3 = w.w;
    a = f4{__builtin_bit_cast(float, w0 << 16), __builtin_bit_cast(float, w0 & 0xffff0000u), __builtin_bit_cast(float, w1 << 16), __builtin_bit_cast(float, w1 & 0xffff0000u)};
    b = f4{__builtin_bit_cast(float, w2 << 16), __builtin_bit_cast(float, w2 & 0xffff0000u), __builtin_bit_cast(float, w3 << 16), __builtin_bit_cast(float, w3 & 0xffff0000u)};
}
// NaN and infinities -> 0; whether there were any
__device__ __forceinline__ bool finite_only(bf16x8 &v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned m = ((w[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;       // the halves that are not finite
        any |= m;
        w[i] &= ~(m | (m - (m >> 15)));
    }
    v = __builtin_bit_cast(bf16x8, w);
    return any;
}
// eight fp32 values -> NT bf16 operands that add up to them
template <int N>
__device__ __forceinline__ void split8(f4 a, f4 b, bf16x8 (&o)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bf16x4 x = round4(a), y = round4(b);
        o[i] = join8(x, y);
        if (i + 1 < N) { a = rest4(a, x); b = rest4(b, y); }
    }
}
// An operand from LDS, contracted index contiguous: row `row`, indices 32 s + ...  Two 8-byte reads that are kept apart: merged into one
// instruction they cost 8 to 32 cycles by pitch, apart 4 to 8 (2 x 16 rows x 8 bytes).
__device__ __forceinline__ bf16x8 frag(const unsigned char *tile, int pitch, int row, int s, int gq) {
    const int at = row * pitch + (32 * s + 4 * gq) * 2;
    return join8(*reinterpret_cast<const bf16x4 *>(tile + at), *reinterpret_cast<const bf16x4 *>(tile + fresh(at + 32)));
}
// the same from a tile whose 32-column blocks are stored in operand order (index 16 u + 4 a + r at 8 a + 4 u + r): one 16-byte read
__device__ __forceinline__ bf16x8 frag_p(const unsigned char *tile, int pitch, int row, int s, int gq) {
    return *reinterpret_cast<const bf16x8 *>(tile + row * pitch + (32 * s + 8 * gq) * 2);
}
__device__ __forceinline__ int operand_pos(int c) { return (c & ~31) + 8 * ((c >> 2) & 3) + 4 * ((c >> 4) & 1); }      // of a group of four, c % 4 == 0
// an operand from LDS, contracted index along the rows (rows 32 s + ...), columns 16 c .. 16 c + 15: ds_read_b64_tr_b16 hands every lane of 16 its
// column of four rows; lane 4 a + b of the 16 addresses row a, columns 4 b .. 4 b + 3
__device__ __forceinline__ bf16x8 frag_t(const unsigned char *tile, int pitch, int c, int s, int lane) {
    typedef s16x4 __attribute__((address_space(3))) *lp;
    const unsigned char *q = tile + (32 * s + 4 * (lane >> 4) + ((lane >> 2) & 3)) * pitch + (16 * c + 4 * (lane & 3)) * 2;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 16 * pitch));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// the same with the contracted indices 8 gq + {0..7} of every 32, beside direct operands read as eight values in a row (frag_c)
__device__ __forceinline__ bf16x8 frag_tc(const unsigned char *tile, int pitch, int c, int s, int lane) {
    typedef s16x4 __attribute__((address_space(3))) *lp;
    const unsigned char *q = tile + (32 * s + 8 * (lane >> 4) + ((lane >> 2) & 3)) * pitch + (16 * c + 4 * (lane & 3)) * 2;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 4 * pitch));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ bf16x8 frag_c(const unsigned char *tile, int pitch, int row, int s, int gq) {
    return *reinterpret_cast<const bf16x8 *>(tile + row * pitch + (32 * s + 8 * gq) * 2);
}

// The weights of a chunk's pairs (64 x 64, below the diagonal) in LDS, three planes of PAIRS bytes, a bf16 term each: rows 0 ... 31 hold 32 columns, rows 32 ... 63
// hold 64.  pair_row(half, i): row i from a plane's start (row 0 where its pitch would put it).
constexpr int PAIR_PITCH0 = 64 + 16, PAIR_PITCH1 = 128 + 16, PAIRS = 32 * (PAIR_PITCH0 + PAIR_PITCH1);
__device__ __forceinline__ constexpr int pair_pitch(int half) { return half ? PAIR_PITCH1 : PAIR_PITCH0; }
__device__ __forceinline__ constexpr int pair_row(int half, int i) { return (half ? 32 * (PAIR_PITCH0 - PAIR_PITCH1) : 0) + i * pair_pitch(half); }
__device__ __forceinline__ void put_pairs(unsigned char *at, f4 v) {
#pragma unroll
    for (int u = 0; u < 3; ++u) {
        const bf16x4 w = round4(v);
        *reinterpret_cast<bf16x4 *>(at + u * PAIRS) = w;
        v = rest4(v, w);
    }
}
__device__ __forceinline__ float get_pair(const unsigned char *at) {
    return ((float)*reinterpret_cast<const bf16 *>(at + 2 * PAIRS) + (float)*reinterpret_cast<const bf16 *>(at + PAIRS)) + (float)*reinterpret_cast<const bf16 *>(at);
}

// A C x DP tile of bf16 on its way from memory to LDS, in 16-byte pieces of a row that wait in registers, so a chunk is in flight while the previous
// one is worked on; rows past n and columns past D are zero.  VEC: rows are made of such pieces.  Else a piece may begin in the middle of a 32-bit
// word: five words are read and shifted, and the last piece of a row is masked (4 x 4096 tokens, 16 heads of 100 x 96, forward and backward:
// 595 us; element by element 1004).  Every row, head and batch starts on an even or odd element for good: C rows are an even number.
template <int C, int DP, int NT, bool VEC>
struct TileRegs {
    static constexpr int PR = DP / 8, N = C * PR / NT > 0 ? C * PR / NT : 1, STEP = NT / PR;     // pieces a row, pieces a thread, rows from one to the next
    static_assert(C % 2 == 0 && STEP % 2 == 0, "a thread's pieces begin alike");
    u32x4 v[N];
    unsigned last[VEC ? 1 : N];
    int voff, shift;                                               // bytes from the chunk's first row; pieces past D lie outside every descriptor
    __device__ __forceinline__ void init(const bf16 *src, long long ld, int D) {
        const int r = threadIdx.x / PR, c = 8 * (threadIdx.x % PR), off = (r * (int)ld + c) * 2 + (VEC ? 0 : (int)((uintptr_t)src & 2));
        voff = c < D && r < C ? off & ~3 : SS2D_BUF_OOR;
        shift = (off & 2) * 8;
    }
    // a descriptor of n rows: later rows read as zero.  D <= ld < 2^22 elements (host)
    __device__ __forceinline__ void load(const bf16 *src, long long ld, int n, int D) {
        if (VEC) {
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(src, (unsigned)(n * (int)ld * 2));
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, voff, j * STEP * (int)ld * 2, 0);
        } else {
            const int lead = (int)((uintptr_t)src & 2);            // whole words, the first and last of which may be half outside
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const char *>(src) - lead, n > 0 ? (unsigned)(lead + ((n - 1) * (int)ld + D) * 2 + 3) & ~3u : 0u);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int at = (int)threadIdx.x / PR + j * STEP < n ? voff : SS2D_BUF_OOR;
                v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, at, j * STEP * (int)ld * 2, 0);
                last[VEC ? 0 : j] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, j * STEP * (int)ld * 2 + 16, 0);
            }
        }
    }
    // whether a NaN or an infinity is among the values: an exponent of ones carries into the sign's place
    __device__ __forceinline__ bool not_finite() const {
        unsigned any = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= (v[j][i] & 0x7f807f80u) + 0x00800080u;
#pragma unroll
        for (int j = 0; j < (VEC ? 0 : N); ++j) any |= (last[j] & 0x7f807f80u) + 0x00800080u;     // (words past a row's end: a false alarm only costs time)
        return any & 0x80008000u;
    }
    // ORDERED: 32-column blocks in operand order (frag_p)
    template <bool ORDERED = false>
    __device__ __forceinline__ void put(unsigned char *tile, int pitch, int D) const {
        const int c = 8 * (threadIdx.x % PR);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = threadIdx.x / PR + j * STEP;
            if (C * PR % NT == 0 || r < C) {
                u32x4 w = v[j];
                if (!VEC) {
                    const unsigned q[5] = {w.x, w.y, w.z, w.w, last[VEC ? 0 : j]};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned both = __builtin_amdgcn_alignbit(q[i + 1], q[i], (unsigned)shift);
                        w[i] = c + 2 * i + 1 < D ? both : c + 2 * i < D ? both & 0xffffu : 0u;
                    }
                }
                unsigned char *d = tile + r * pitch;
                if (ORDERED) {
                    *reinterpret_cast<u32x2 *>(d + 2 * operand_pos(c)) = u32x2{w.x, w.y};
                    *reinterpret_cast<u32x2 *>(d + 2 * operand_pos(c + 4)) = u32x2{w.z, w.w};
                } else {
                    *reinterpret_cast<u32x4 *>(d + 2 * c) = w;
                }
            }
        }
    }
};

// the same for fp32 tiles (C x DP, PITCH floats a row), groups of four columns: a group may begin on any word, so only a row's last group differs
template <int C, int DP, int PITCH, int NT, bool VEC>
struct TileRegsF {
    static constexpr int PR = DP / 4, N = (C * PR + NT - 1) / NT, STEP = NT / PR;
    f4 v[N];
    int voff;
    __device__ __forceinline__ void init(long long ld, int D) {
        const int r = threadIdx.x / PR, c = 4 * (threadIdx.x % PR);
        voff = c < D && r < C ? (r * (int)ld + c) * 4 : SS2D_BUF_OOR;
    }
    __device__ __forceinline__ void load(const float *src, long long ld, int n, int D) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(src, VEC ? (unsigned)(n * (int)ld * 4) : n > 0 ? (unsigned)(((n - 1) * (int)ld + D) * 4) : 0u);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = VEC || (int)threadIdx.x / PR + j * STEP < n ? voff : SS2D_BUF_OOR;
            v[j] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, j * STEP * (int)ld * 4, 0));
        }
    }
    __device__ __forceinline__ bool not_finite() const {
        unsigned any = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[j][i];
                any |= (__builtin_bit_cast(unsigned, x) & 0x7f800000u) + 0x00800000u;
            }
        return any & 0x80000000u;
    }
    __device__ __forceinline__ void put(float *tile, int D) const {
        const int c = 4 * (threadIdx.x % PR);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = threadIdx.x / PR + j * STEP;
            if (C * PR % NT == 0 || r < C) {
                f4 w = v[j];
                if (!VEC) {
#pragma unroll
                    for (int i = 1; i < 4; ++i) w[i] = c + i < D ? w[i] : 0.0f;
                }
                *reinterpret_cast<f4 *>(tile + r * PITCH + c) = w;
            }
        }
    }
};

// Results of a chunk leave through a descriptor of its rows: rows past the last token and columns past D fall outside and are dropped, without a branch
// that would split the products around it into pieces waiting for LDS one by one.
struct RowsOut {
    __amdgpu_buffer_rsrc_t rs;
    template <typename T>
    __device__ __forceinline__ RowsOut(T *base, int n, long long ld) : rs(make_rsrc(base, (unsigned)(n * (int)ld * (int)sizeof(T)))) {}
    // four columns c .. c + 3 of row r; VEC, or D a multiple of 4: all four or none inside
    template <bool VEC>
    __device__ __forceinline__ void put4(bf16 *, int r, int c, long long ld, int D, f4 v) const {
        const u32x2 w = __builtin_bit_cast(u32x2, round4(v));
        const int off = (r * (int)ld + c) * 2;
        if (VEC || D % 4 == 0) {
            __builtin_amdgcn_raw_buffer_store_b64(w, rs, c < D ? off : SS2D_BUF_OOR, 0, 0);
        } else {
            const unsigned a = w.x, b = w.y;
            const unsigned short h[4] = {(unsigned short)a, (unsigned short)(a >> 16), (unsigned short)b, (unsigned short)(b >> 16)};
#pragma unroll
            for (int e = 0; e < 4; ++e) __builtin_amdgcn_raw_buffer_store_b16(h[e], rs, c + e < D ? off + 2 * e : SS2D_BUF_OOR, 0, 0);
        }
    }
    template <bool VEC>
    __device__ __forceinline__ void put4(float *, int r, int c, long long ld, int D, f4 v) const {
        const int off = (r * (int)ld + c) * 4;
        if (VEC || D % 4 == 0) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, c < D ? off : SS2D_BUF_OOR, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = v[e];
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), rs, c + e < D ? off + 4 * e : SS2D_BUF_OOR, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void put1(float v, int r, int c, long long ld, int D) const {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rs, c < D ? (r * (int)ld + c) * 4 : SS2D_BUF_OOR, 0, 0);
    }
};

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// tokens of a chunk: the backward holds q, k, v, dout, a dk x dv state and two C x C matrices in 160 KB of LDS
inline int linattn_chunk(int dtype, int dk, int dv) { return dtype || (dk <= 64 && dv <= 64) ? 64 : 32; }

// Segments.  One workgroup walks a segment; with fewer workgroups than the card holds at once it idles, and a segment costs a second pass over k and v (q
// and dout in the backward) and a state's round trip.  So all tokens of all sequences and heads are dealt to a number of workgroups, at
// least two chunks each, in equal parts of the longest sequence: in the forward to as many as are resident (three a CU up to 64 x 64 in bf16, else two); in the
// backward to one a CU with keys beyond 64 wide in bf16, else to two.  Two are resident with keys up to 16 wide in fp32 and up to 64 x 64 in bf16; the others in
// fp32, and 64 x 128 in bf16, hold one a CU and take two rounds of pieces half as long: a few per cent more for few long sequences, less where the pieces of a batch
// would not divide by the CUs (us, forward and backward, 256 / 512 workgroups: 2 x 16384 tokens, 4 heads of 64 x 64 fp32 227 / 237, 24 x 784 tokens, 6 heads 265 /
// 233; 64 x 128 bf16 163 / 175 and 183 / 165; 4 x 4096, 16 heads of 128 x 128 fp32 1257 / 1291).  Measured, us, for half the workgroups / these / twice / no split: 24 x 3136 tokens, 3 heads of 16 x 64 fp32, forward and
// backward 271 / 180 / 190 / 574; 4 x 4096 tokens, 16 heads of 128 x 64 bf16, both ways 551 / 364 / 381 / 973; 65536 tokens, 8 heads of 128 x 128 bf16, forward
// 283 / 250 / 263 / 5402.  Short ones, 4 heads of 64 x 64 bf16: a chunk takes 3 us and the two further launches as much as two chunks: 256 tokens (4 chunks) 16 us in
// one walk, 19 split; 384 tokens (6) 22 and 19.
// Returns the segments of the longest sequence in the upper and the chunks a segment in the lower 32 bits; 1 segment: no sequence is split.
inline long long linattn_segments(int dtype, long long all_tokens, long long max_len, int H, int dk, int dv, int backward) {
    const int C = linattn_chunk(dtype, dk, dv);
    const long long nch = (max_len + C - 1) / C, all = (all_tokens + C - 1) / C * H * (backward || dtype ? 1 : (dv + 63) / 64);
    const long long wgs = backward ? (dtype && dk > 64 ? 256 : 512) : dtype && dk <= 64 && dv <= 64 ? 768 : 512;
    long long segc = (all + wgs - 1) / wgs;
    if (segc < 2) segc = 2;
    if (segc >= nch || nch < 6) return (1LL << 32) | (nch > 0 ? nch : 1);
    const long long nseg = (nch + segc - 1) / segc;
    return nseg << 32 | (nch + nseg - 1) / nseg;
}

// floats of one chunk's saved state.  bf16 kernels: accumulator order, padded to whole tiles (16-byte pieces of a wave side by side)
inline long long linattn_state_floats(int dtype, int dk, int dv) {
    return dtype ? (long long)(dk <= 32 ? 32 : dk <= 64 ? 64 : 128) * (dv <= 64 ? 64 : 128) : (long long)dk * dv;
}

// segments of all sequences, in front of which a state is kept
inline long long linattn_slots(int packed, long long N, long long tokens, long long nseg, long long segc, int C) {
    return nseg == 1 ? N : packed ? tokens / (segc * C) + N : N * nseg;
}

inline int linattn_problem(Problem &p, int dtype, const void *q, const void *k, const void *v, const float *g, const long long *st, const int *cu,
                           int N, long long tokens, int H, int G, int dk, int dv, float scale, int nseg, int segc, const char *name) {
    if (dtype != 0 && dtype != 1) { ss2d_set_error("%s: unknown dtype %d", name, dtype); return -1; }
    if (!q || !k || !v || !g || !st) { ss2d_set_error("%s: null pointer", name); return -2; }
    if (N <= 0 || tokens <= 0 || tokens > 0x7fffff00LL || H <= 0 || G <= 0 || nseg <= 0 || segc <= 0) { ss2d_set_error("%s: size out of range", name); return -3; }
    if (H % G) { ss2d_set_error("%s: %d heads are not a multiple of %d key heads", name, H, G); return -4; }
    if (dk < 1 || dk > 128 || dv < 1 || dv > 128) { ss2d_set_error("%s: dk %d and dv %d must be 1 ... 128", name, dk, dv); return -5; }
    if ((long long)H * dk >= (1 << 22) || (long long)H * dv >= (1 << 22)) { ss2d_set_error("%s: %d heads are too many", name, H); return -6; }
    const int C = linattn_chunk(dtype, dk, dv);
    if (segc > 0x7fffffff / C) segc = 0x7fffffff / C;
    const long long slots = linattn_slots(cu ? 1 : 0, N, tokens, nseg, segc, C);
    if (slots * H * 2 > 0x7ffffff0LL || (long long)N * H > 65535LL * 32) { ss2d_set_error("%s: too many sequences and heads", name); return -6; }
    if (cu && nseg > 1) nseg = 0x7fffffff;
    p.slots = (int)slots;
    p.q = q; p.k = k; p.v = v; p.g = g; p.cu = cu; p.tokens = tokens; p.N = N; p.H = H; p.G = G; p.dk = dk; p.dv = dv; p.scale = scale; p.nseg = nseg; p.segc = segc;
    p.qb = st[0]; p.ql = st[1]; p.qh = st[2]; p.kb = st[3]; p.kl = st[4]; p.kh = st[5];
    p.vb = st[6]; p.vl = st[7]; p.vh = st[8]; p.gb = st[9]; p.gl = st[10]; p.gh = st[11];
    // rows come through descriptors of a chunk: they must not overlap, nor lie 2^22 elements apart
    if (st[1] < dk || st[4] < dk || st[7] < dv || st[1] >= (1 << 22) || st[4] >= (1 << 22) || st[7] >= (1 << 22)) {
        ss2d_set_error("%s: token strides %lld, %lld, %lld", name, st[1], st[4], st[7]);
        return -4;
    }
    const int m = dtype ? 8 : 4;                                // elements of a 16-byte piece
    bool vec = dk % m == 0 && dv % m == 0;
    if (dtype) {                                                // fp32 pieces may begin on any word, bf16 ones only on a word's start
        vec = vec && ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 4 == 0;
        for (int i = 0; i < 9; ++i) vec = vec && st[i] % 2 == 0;
    }
    p.vec = vec;
    return 0;
}

// W neighbouring elements of a state, on any 32-bit word
template <int W> struct Elements { typedef float type; };
template <> struct Elements<4> { typedef f4 __attribute__((aligned(4))) type; };

}  // namespace linattn

// the pass over segments that leaves their own contributions (forward: k v^T; reverse: q dout^T, with q in the place of k and dout in that of v),
// defined beside the forward
void linattn_segment_pass(int dtype, const linattn::Problem &p, float *seg_states, double *seg_decay, bool reverse, hipStream_t s);
