// Attention of whole prompts packed one after another, and its gradient (gfx950).
//
// Sequence b holds tokens cu[b] .. cu[b+1] of q (N, Hq, D), k and v (N, Hkv, D)
// in 16 bits; within it, with kv head h / G of query head h,
//   o_t = sum_s p_ts v_s,   p_ts = exp(scale q_t . k_s - lse_t),
//   lse_t = log sum_s exp(scale q_t . k_s),      s <= t when causal.
// The dense counterpart in the reference takes padded fp32 batches and has no
// kernel (attention/reference.py:72-177).
#include <math.h>

#include <type_traits>

#include "omni_common.h"

namespace omni {

typedef float pf16_t __attribute__((ext_vector_type(16)));
typedef short ps4_t __attribute__((ext_vector_type(4)));
typedef short ps8_t __attribute__((ext_vector_type(8)));
typedef __bf16 pb8_t __attribute__((ext_vector_type(8)));
typedef _Float16 ph8_t __attribute__((ext_vector_type(8)));
#define PT_LDS __attribute__((address_space(3)))

constexpr int kPtWaves = 4;
constexpr int kPtRows = 32 * kPtWaves;   // query rows of a block
constexpr int kPtKeys = 64;              // keys of a tile
constexpr int kPtBufWord3 = 0x00020000;
// Exponents of two: a row's running maximum follows its tiles only when one is
// above it by kPtSlack (rescaling costs D / 2 products a lane), and f16
// probabilities are kept times 2^kPtF16Up, so that they reach 2^15 at most and
// the smallest subnormal is 2^-31 of the maximum (bf16 has fp32's range).
constexpr float kPtSlack = 8.0f;
constexpr float kPtF16Up = 7.0f;

struct PromptHeads {
    const char *p;
    int64_t st, sh;                      // byte strides of a token and a head
};

struct PromptArgs {
    PromptHeads q, k, v, o, olo;         // olo: what rounding took from o, for the gradient
    PromptHeads g, dq, dk, dv;           // backward: the output's gradient, and those of q, k and v
    float *lse;                          // (Hq, N), or NULL
    float *lse2, *delta;                 // backward, (Hq, N): lse log2 e (f16: less kPtF16P), and -sum_d g o
    float *parts;                        // backward, (heads of the group in parts, dk and dv, N, Hkv, D)
    float *peaks;                        // backward in f16: kPtPeaks largest squared norms of g's rows, then of v's
    const int32_t *cu;
    int64_t N;
    int B, Hq, Hkv, G;
    int causal, negate, fill;            // fill: rows of no sequence get zeros
    int peak_rows, n_parts;
    float c, cs, scale;                  // |scale| log2(e), scale log2(e)
    float hide;                          // a hidden score: cs times it is -inf
};

// ── types ───────────────────────────────────────────────────────────────

template <int DT>
__device__ __forceinline__ pf16_t pt_mfma(ps8_t a, ps8_t b, pf16_t c) {
    if constexpr (DT == OMNI_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pb8_t, a), __builtin_bit_cast(pb8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pt_pack(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 t = {a, b};
    if constexpr (DT == OMNI_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, b2));
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, h2));
    }
}

// Sum of the two values of a word and c.
template <int DT>
__device__ __forceinline__ float pt_add2(uint32_t v, float c) {
    if constexpr (DT == OMNI_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, v), __builtin_bit_cast(b2, 0x3f803f80u), c, false);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v), __builtin_bit_cast(h2, 0x3c003c00u), c, false);
    }
}

// x . y of eight values each, and c.
template <int DT>
__device__ __forceinline__ float pt_dot8(ps8_t x, ps8_t y, float c) {
    const uint4 a = __builtin_bit_cast(uint4, x), b = __builtin_bit_cast(uint4, y);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w}, w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == OMNI_BF16) {
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, u[i]), __builtin_bit_cast(b2, w[i]), c, false);
        } else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            c = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, u[i]), __builtin_bit_cast(h2, w[i]), c, false);
        }
    }
    return c;
}

__device__ __forceinline__ ps8_t pt_frag(const uint32_t *p) {
    return __builtin_bit_cast(ps8_t, make_uint4(p[0], p[1], p[2], p[3]));
}

template <int DT>
__device__ __forceinline__ float pt_value(uint32_t h) {     // low 16 bits
    return DT == OMNI_BF16 ? bf16_to_f32((uint16_t)h) : f16_to_f32((uint16_t)h);
}

__device__ __forceinline__ float pt_max_halves(float m) {
    const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1]));
}
__device__ __forceinline__ float pt_sum_halves(float m) {
    const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __uint_as_float(u[0]) + __uint_as_float(u[1]);
}

// Barrier that also waits for the wave's own copies into LDS: they have no
// register result for the compiler to wait for, and the barrier's own fence
// does not follow them around a loop.
__device__ __forceinline__ void pt_sync() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
}

// ── tiles in LDS ────────────────────────────────────────────────────────
//
// A tile's rows of D 16-bit values lie one after another, the 16-byte chunks
// of row r in the order chunk ^ pt_swz(r): both the row reads (16 lanes, a
// chunk of 16 rows each) and the transposed reads (16 lanes, 32 bytes of four
// rows, two such groups side by side) then meet every bank once.

template <int D>
__device__ __forceinline__ int pt_swz(int r) {
    if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (D == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
}

// The copy of a tile, N instructions a wave, each a KB of LDS in lane order (so
// the swizzle is in the address read): instruction u takes rows
// RPI * kPtWaves * u on, 16, 32 or 64 rows apart, which swizzle alike.
template <int D, int ROWS>
struct PtCopy {
    static constexpr int CH = D / 8, RPI = 64 / CH, STEP = RPI * kPtWaves, N = ROWS / STEP;
    static_assert(N >= 1 && ROWS % STEP == 0, "whole instructions");
    int row, chunk;                      // lane's row and byte in the row, of instruction 0

    // by wave w (uniform) of four
    __device__ __forceinline__ void init(int w) {
        const int lane = threadIdx.x & 63;
        row = w * RPI + lane / CH;
        chunk = ((lane % CH) ^ pt_swz<D>(row)) * 16;
    }
    // Rows r0 .. r0 + ROWS - 1 of a head at `base` (its row 0) to `lds`; rows from `len` on repeat the last.
    __device__ __forceinline__ void issue(const char *base, int64_t st, int r0, int len, char *lds, int w) const {
        const uint32_t stride = (uint32_t)st;
        const int left = min(len - r0, ROWS);
        const __amdgpu_buffer_rsrc_t R = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(base + (int64_t)r0 * st), (short)0, (int)((uint32_t)(left - 1) * stride + 2 * D), kPtBufWord3);
        char *dst = lds + w * 1024;
        int r = row;
        asm volatile("" : "+v"(r));      // no register for each instruction's offset through the loop
        if (left == ROWS) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(R, (PT_LDS void *)(dst + u * 1024 * kPtWaves), 16,
                                                         (uint32_t)r * stride + chunk, STEP * u * stride, 0, 0);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(R, (PT_LDS void *)(dst + u * 1024 * kPtWaves), 16,
                                                         (uint32_t)min(r + STEP * u, left - 1) * stride + chunk, 0, 0, 0);
        }
    }
};

// A lane's byte offsets in a tile: of its row's chunk in the row reads, and of
// its part of four rows in the transposed ones.  Every other read of the lane
// is these with bits flipped and a constant added (the swizzle of rows 16 on is
// the same; dims and the upper eight rows flip chunk bits).  fresh() hides that
// they do not change: the compiler would keep each sum of a buffer's address
// and an offset in a register of its own through the loop, 50 of them, instead
// of adding it in the read.
template <int D>
struct PtLane {
    uint32_t r, c;
    // of the tile's rows from row0 (a multiple of 32) on
    __device__ __forceinline__ void init(int row0 = 0) {
        const int lane = threadIdx.x & 63, half = lane >> 5, n = lane & 31, i = lane & 15;
        r = (row0 + n) * (2 * D) + ((half ^ pt_swz<D>(n)) * 16);
        const int row = 4 * half + i / 4, byte = (16 * ((lane >> 4) & 1) + 4 * (i & 3)) * 2;
        c = (row0 + row) * (2 * D) + (((byte >> 4) ^ pt_swz<D>(row)) * 16) + (byte & 15);
    }
    __device__ __forceinline__ PtLane fresh() const {
        PtLane x = *this;
        asm volatile("" : "+v"(x.r), "+v"(x.c));
        return x;
    }
    // A operand of rows r0 .. r0 + 31 (a multiple of 32), dims 16 kk .. 16 kk + 15
    __device__ __forceinline__ ps8_t rows(const char *tile, int r0, int kk) const {
        return *reinterpret_cast<const ps8_t *>(tile + ((r ^ (uint32_t)(32 * kk)) + (uint32_t)(r0 * 2 * D)));
    }
    // A operand of the transposed tile: dims 32 dt .. 32 dt + 31 by rows r0 .. r0 +
    // 15, the rows in the order of an MFMA result's registers: slot (half, j) is
    // row 8 (j / 4) + 4 half + j % 4
    __device__ __forceinline__ ps8_t cols(const char *tile, int r0, int dt) const {
        ps4_t v[2];
#pragma unroll
        for (int g = 0; g < 2; ++g)
            v[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (PT_LDS ps4_t *)(tile + ((c ^ (uint32_t)(64 * dt + 32 * g)) + (uint32_t)((r0 + 8 * g) * 2 * D))));
        return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// Row operand of 32 rows straight from memory: lane's row at `p`, dims 8 half on.
template <int D>
__device__ __forceinline__ void pt_load_rows(const char *p, ps8_t (&f)[D / 16], uint32_t flip = 0) {
    p += 16 * ((threadIdx.x >> 5) & 1);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        uint4 u = *reinterpret_cast<const uint4 *>(p + 32 * kk);
        u.x ^= flip; u.y ^= flip; u.z ^= flip; u.w ^= flip;
        f[kk] = __builtin_bit_cast(ps8_t, u);
    }
}

// x times f, of the lane's row, to `p`: register i of block d is dim
// 32 d + 8 (i / 4) + 4 half + i % 4; after the swap each half holds eight dims.
// LO: what the rounding leaves, rounded, to `q`.
template <int DT, int D, bool LO = false>
__device__ __forceinline__ void pt_store(char *p, const pf16_t (&x)[D / 32], float f, bool mine, char *q = nullptr) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            uint32_t u[2][2], w[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float y[4] = {x[d][4 * g + 2 * e] * f, x[d][4 * g + 2 * e + 1] * f, x[d][4 * g + 4 + 2 * e] * f,
                                    x[d][4 * g + 4 + 2 * e + 1] * f};
                const uint32_t lo = pt_pack<DT>(y[0], y[1]), hi = pt_pack<DT>(y[2], y[3]);
                const auto t = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
                u[0][e] = t[0];
                u[1][e] = t[1];
                if constexpr (LO) {
                    const auto r = __builtin_amdgcn_permlane32_swap(
                        pt_pack<DT>(y[0] - pt_value<DT>(lo), y[1] - pt_value<DT>(lo >> 16)),
                        pt_pack<DT>(y[2] - pt_value<DT>(hi), y[3] - pt_value<DT>(hi >> 16)), false, false);
                    w[0][e] = r[0];
                    w[1][e] = r[1];
                }
            }
            const int at = (32 * d + 8 * (g + half)) * 2;
            if (mine) *reinterpret_cast<uint4 *>(p + at) = make_uint4(u[0][0], u[0][1], u[1][0], u[1][1]);
            if constexpr (LO) {
                if (mine) *reinterpret_cast<uint4 *>(q + at) = make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
            }
        }
}

// Zeros to rows row0 .. row0 + R - 1 of a slot's: token r / G, head h0 + r % G.
template <int D, int R>
__device__ __forceinline__ void pt_zero_rows(const PromptHeads &o, int start, int row0, int len, int h0, int G) {
    constexpr int CH = D / 8;
    for (int e = threadIdx.x; e < R * CH; e += blockDim.x) {
        const int r = row0 + e / CH, t = r / G;
        if (t < len)
            *reinterpret_cast<uint4 *>(const_cast<char *>(o.p) + (int64_t)(start + t) * o.st + (h0 + r - t * G) * o.sh + e % CH * 16) =
                make_uint4(0, 0, 0, 0);
    }
}

// Hidden keys and rows count for nothing, whatever they hold, but a matrix unit
// multiplies their weight of 0 with it.  Tiles that hide some are therefore
// looked through (a tenth of such a tile's time), and a wave that met an
// infinity or a NaN there computes its result again, term by term and from
// memory.  (Tokens behind the sequence have its last token in their place.)
template <int DT>
__device__ __forceinline__ bool pt_all_finite(const char *tile, int bytes) {
    // an exponent of ones carries into the sign's place
    constexpr uint32_t ONES = DT == OMNI_BF16 ? 0x7f807f80u : 0x7c007c00u, LAST = DT == OMNI_BF16 ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
    for (int at = (threadIdx.x & 63) * 16; at < bytes; at += 1024) {
        const uint4 u = *reinterpret_cast<const uint4 *>(tile + at);
        any |= ((u.x & ONES) + LAST) | ((u.y & ONES) + LAST) | ((u.z & ONES) + LAST) | ((u.w & ONES) + LAST);
    }
    return __builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0) == 0;
}

// acc += sum over rows r0 .. r0 + 31 of x (its row 0 at `base`) of w times the
// row, where the lane's column sees it, rows first .. end - 1.  w is laid out as
// an MFMA result.
template <int DT, int D>
__device__ __forceinline__ void pt_add_terms(float (&acc)[D / 32][16], const pf16_t &weights, const char *base, int64_t st, int r0, int first, int end) {
    const int half = (threadIdx.x >> 5) & 1;
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = weights[i];
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
        // the weights of the lower half's row and of the upper's; the next ones move up
        const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(w[0]), __float_as_uint(w[0]), false, false);
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
            const float f = __uint_as_float(h ? u[1] : u[0]);
            const int r = r0 + 8 * (i / 4) + 4 * h + i % 4;
            if (r < first || r >= end) continue;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(base + (int64_t)r * st + (32 * d + 8 * g + 4 * half) * 2);
                    const float x[4] = {pt_value<DT>(v.x), pt_value<DT>(v.x >> 16), pt_value<DT>(v.y), pt_value<DT>(v.y >> 16)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][4 * g + e] = fmaf(f, x[e], acc[d][4 * g + e]);
                }
        }
#pragma unroll
        for (int k = 0; k < 15; ++k) w[k] = w[k + 1];
    }
}

template <int NT>
__device__ __forceinline__ void pt_clear(float (&x)[NT][16]) {
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[d][i] = 0.0f;
}
template <int NT>
__device__ __forceinline__ void pt_assign(pf16_t (&y)[NT], const float (&x)[NT][16]) {
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[d][i] = x[d][i];
}

// x . y of 32 rows of each: A operand rows r0 .. of x from memory (rows from len
// on repeat the last), B operand y(kk).
template <int DT, int D, class Y>
__device__ __forceinline__ pf16_t pt_product(const char *base, int64_t st, int r0, int len, float init, Y y) {
    const char *p = base + (int64_t)min(r0 + (int)(threadIdx.x & 31), len - 1) * st + 16 * ((threadIdx.x >> 5) & 1);
    pf16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = init;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) s = pt_mfma<DT>(*reinterpret_cast<const ps8_t *>(p + 32 * kk), y(kk), s);
    return s;
}

// ── which rows a block takes ────────────────────────────────────────────
//
// A sequence's rows are its tokens, or its tokens' query heads of one kv head,
// head by head (row r: token r / G, head r % G of the group), so that a short
// sequence's heads fill a tile together and share its keys.  Tiles of R rows
// are dealt to slots: sequence b has the slots from G cu[b] / R + b on, one more
// than its tiles at most, so no list is made and the grid, G N / R + B + 1
// slots, needs only the total.  The slots behind the last sequence's are those
// of the tokens of none.  Of a sequence's tiles those with the most work under a
// causal mask come first: the last query rows, the first keys.

struct PtSlot {
    int start, len, tile;                // tokens; tile < 0: nothing to do
    bool none;                           // tokens of no sequence
};

template <int R>
__device__ __forceinline__ PtSlot pt_slot(const int32_t *cu, int B, int64_t N, int G, int64_t slot, bool last_first) {
    const int lane = threadIdx.x & 63;
    auto base = [&](int b) { return (int64_t)((uint64_t)(uint32_t)cu[b] * (uint32_t)G / R) + b; };
    // the last b in [0, B] with base(b) <= slot, 64 ways a step
    int lo = 0, n = B + 1;
    while (n > 1) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const bool below = lane * step < n && base(b) <= slot;
        const int at = 63 - __builtin_clzll(__ballot(below) | 1ull);
        lo += at * step;
        n = min(step, n - at * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    PtSlot s;
    const int64_t a = cu[lo], e = lo < B ? (int64_t)cu[lo + 1] : N;
    s.none = lo == B;
    // whatever cu holds, tokens stay within 0 .. N
    s.start = (int)(a < 0 ? 0 : a > N ? N : a);
    const int64_t end = e > N ? N : e;
    s.len = end > s.start ? (int)(end - s.start) : 0;
    const int64_t tiles = ((int64_t)s.len * G + R - 1) / R, at = slot - base(lo);
    s.tile = at < 0 || at >= tiles ? -1 : (int)(last_first ? tiles - 1 - at : at);
    return s;
}

// The wave's 32 query rows from row w0 of the sequence's (kv head hk).
struct PtQueries {
    int t, h;                            // the lane's token and head (its row, or the last)
    int first, last;                     // the wave's tokens
    bool mine, live;                     // the lane's row is one; the wave's first is
    __device__ __forceinline__ void init(const PromptArgs &a, const PtSlot &S, int hk, int w0) {
        const int rows = S.len * a.G, row = w0 + (threadIdx.x & 31), r = min(row, rows - 1);
        mine = row < rows;
        live = w0 < rows;
        t = r / a.G;
        h = hk * a.G + r - t * a.G;
        first = w0 / a.G;
        last = min((w0 + 31) / a.G, S.len - 1);
    }
};

// Sums of one wave to another by way of 128 D bytes of LDS, a KB for four registers of its lanes.
template <int NT>
__device__ __forceinline__ void pt_give(char *lds, const pf16_t (&x)[NT]) {
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4 *>(lds + (4 * d + i / 4) * 1024 + (threadIdx.x & 63) * 16) =
                make_float4(x[d][i], x[d][i + 1], x[d][i + 2], x[d][i + 3]);
}
template <int NT>
__device__ __forceinline__ void pt_take(const char *lds, pf16_t (&x)[NT], float f = 1.0f) {
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 y = *reinterpret_cast<const float4 *>(lds + (4 * d + i / 4) * 1024 + (threadIdx.x & 63) * 16);
            x[d][i] = fmaf(y.x, f, x[d][i]); x[d][i + 1] = fmaf(y.y, f, x[d][i + 1]);
            x[d][i + 2] = fmaf(y.z, f, x[d][i + 2]); x[d][i + 3] = fmaf(y.w, f, x[d][i + 3]);
        }
}

// ── forward ─────────────────────────────────────────────────────────────
//
// A wave holds 32 query rows as the B operand of S^T = K Q^T, so lane n and
// n + 32 share query row n: row statistics are register reductions with one
// exchange, and the probabilities, rounded to the input's 16 bits, are the B
// operand of O^T += V^T P^T where they are, with V^T read transposed from LDS.
// P's rounding, half a step of the inputs' type for each term, is what feeding
// the matrix units 16 bits costs; all else is fp32.  The output is divided by
// the sum of the rounded terms, so that weights sum to one and a row with one
// large term has no error from it; lse is of the unrounded ones.
//
// For a gradient (LO) the output's own rounding is kept as well, and the first
// tile of keys, which is all that the first rows of a causal sequence and all
// rows of a short one see, adds the probabilities' rounding errors as a second
// product: delta_t = sum_d g_td o_td is taken from dp_ts, and where few keys hold
// the weight the difference is a small one of large terms.  With o in 16 bits
// alone dq and dk were off by 1.5 to 2.8 times what rounding them costs
// (sequences of 8 to 1024, scores of deviation 1 to 3), so by 1.4 to 1.5.
//
// Bound by matrix and vector instructions that hardly overlap: 32 heads over 8 of
// 128 in bf16, one causal sequence of 32768 tokens 7.7 to 8.2 ms on different
// cards, 1.07 to 1.14 PFLOP/s, where a large library product reaches 1.5; 8192
// tokens without a mask 970 to 990 us, 1.12 PFLOP/s, with the matrix units busy
// in half of the cycles, vector instructions issuing in the other half (49.6 and
// 48.5 %), no LDS bank conflict and a clock of 2.0 GHz.  Power is the lesser
// part: the same call on zeros, which draw less, takes 857 us, still 1.28
// PFLOP/s.  Two ways to more overlap did not pay: eight waves of which four
// always multiply while four take exponentials, kept in turn by barriers, 1030
// us; scores one tile ahead of the products with V, 990.  64 rows a wave, which
// would halve the LDS reads, does not fit the registers of two waves a SIMD.

template <int DT, int D>
struct PtRow {
    static constexpr int NT = D / 32;
    ps8_t q[D / 16];
    pf16_t o[NT];
    float m;                             // running maximum of scale s log2 e
    float l, l16;                        // the lane's share of the sum of the probabilities, and of the rounded ones
    int t;                               // the row's token (of the sequence)
    bool met;                            // an infinity or NaN among hidden values
};

// at: the tile's bytes in K and V (in the lane's offsets already).  LO: of the first tile, the probabilities' rounding errors, rounded in turn, are
// added as well.
template <int DT, int D, bool LO>
__device__ __forceinline__ void pt_forward_tile(const PromptArgs &a, const PtLane<D> &lane_at, PtRow<DT, D> &R, const char *K,
                                                const char *V, int at, int j0, int len, bool masked, bool first) {
    constexpr int NT = PtRow<DT, D>::NT;
    const PtLane<D> A = lane_at.fresh();
    const int half = (threadIdx.x >> 5) & 1;
    // issue order only: of a SIMD's two waves the one feeding the matrix units goes
    // first (8192 tokens without a mask 1025 -> 978 us; no gain in the gradient's kernels)
    __builtin_amdgcn_s_setprio(1);
    pf16_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        s[b] = pf16_t{};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) s[b] = pt_mfma<DT>(A.rows(K, 32 * b, kk), R.q[kk], s[b]);
    }
    __builtin_amdgcn_s_setprio(0);
    R.met = R.met || (masked && !pt_all_finite<DT>(V + at, kPtKeys * 2 * D));
    if (masked) {
        // the keys of register i of block b: j0 + 32 b + 8 (i / 4) + 4 half + i % 4
        const int seen = (a.causal ? min(R.t, len - 1) : len - 1) - j0 - 4 * half;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (32 * b + 8 * (i / 4) + i % 4 > seen) s[b][i] = -INFINITY;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[b][i]);
    mt = pt_max_halves(mt) * a.c;
    if (__builtin_amdgcn_ballot_w64(mt > R.m + kPtSlack)) {
        const float mn = fmaxf(R.m, mt);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(R.m - mn);
        R.l *= f;
        R.l16 *= f;
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) R.o[d][i] *= f;
        R.m = mn;
    }
    const float off = (R.m == -INFINITY ? 0.0f : R.m) - (DT == OMNI_F16 ? kPtF16Up : 0.0f);
    uint32_t p[2][8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], a.c, -off));
        }
        float sum16 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[b][i] = pt_pack<DT>(x[2 * i], x[2 * i + 1]);
            sum16 = pt_add2<DT>(p[b][i], sum16);
        }
        if (LO && first) {
            uint32_t lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                lo[i] = pt_pack<DT>(x[2 * i] - pt_value<DT>(p[b][i]), x[2 * i + 1] - pt_value<DT>(p[b][i] >> 16));
                sum16 = pt_add2<DT>(lo[i], sum16);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int d = 0; d < NT; ++d) R.o[d] = pt_mfma<DT>(A.cols(V, 32 * b + 16 * k, d), pt_frag(lo + 4 * k), R.o[d]);
        }
        R.l16 += sum16;
        if (a.lse) {
#pragma unroll
            for (int w = 8; w > 0; w /= 2)
#pragma unroll
                for (int i = 0; i < w; ++i) x[i] += x[i + w];
            R.l += x[0];
        }
    }
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const ps8_t pb = pt_frag(p[b] + 4 * k);
#pragma unroll
            for (int d = 0; d < NT; ++d) {
                R.o[d] = pt_mfma<DT>(A.cols(V, 32 * b + 16 * k, d), pb, R.o[d]);
            }
        }
    __builtin_amdgcn_s_setprio(0);
}

// KS = 2: four more waves hold the same rows and take every second tile of keys;
// the halves are joined through LDS at the end.
template <int DT, int D, bool LO, int KS>
__global__ __launch_bounds__(64 * kPtWaves * KS, 2) void prompt_forward_kernel(PromptArgs a) {
    constexpr int TILE = kPtKeys * 2 * D, STEP = KS * kPtKeys;
    __shared__ __attribute__((aligned(16))) char k0[KS * TILE], k1[KS * TILE];
    __shared__ __attribute__((aligned(16))) char v0[KS * TILE], v1[KS * TILE];
    constexpr int NT = D / 32;
    // kv heads vary fastest, so that with eight of them (or a multiple) a kv
    // head's blocks share an XCD and its L2
    const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int hk = (int)(bid % a.Hkv);
    const PtSlot S = pt_slot<kPtRows>(a.cu, a.B, a.N, a.G, bid / a.Hkv, true);
    if (S.tile < 0) return;
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wave = all & (kPtWaves - 1), upper = KS == 2 ? all / kPtWaves : 0;
    const int row0 = S.tile * kPtRows;
    if (S.none) {
        if (!a.fill) return;
        pt_zero_rows<D, kPtRows>(a.o, S.start, row0, S.len, hk * a.G, a.G);
        for (int e = threadIdx.x; a.lse && e < kPtRows; e += blockDim.x) {
            const int r = row0 + e, t = r / a.G;
            if (t < S.len) a.lse[(int64_t)(hk * a.G + r - t * a.G) * a.N + S.start + t] = -INFINITY;
        }
        return;
    }
    const char *kb = a.k.p + (int64_t)S.start * a.k.st + hk * a.k.sh, *vb = a.v.p + (int64_t)S.start * a.v.st + hk * a.v.sh;
    const int kend = a.causal ? min((row0 + kPtRows - 1) / a.G + 1, S.len) : S.len;   // keys that the block sees
    PtCopy<D, kPtKeys> cp;
    cp.init(wave);
    // this half's tile of the pair from key j on
    auto copy = [&](int j, char *K, char *V) {
        j += kPtKeys * upper;
        if (j >= kend) return;
        cp.issue(kb, a.k.st, j, S.len, K + TILE * upper, wave);
        cp.issue(vb, a.v.st, j, S.len, V + TILE * upper, wave);
    };
    copy(0, k0, v0);

    PtLane<D> A;
    A.init(kPtKeys * upper);
    PtQueries W;
    W.init(a, S, hk, row0 + 32 * wave);
    PtRow<DT, D> R;
    R.t = W.t;
    pt_load_rows<D>(a.q.p + (int64_t)(S.start + W.t) * a.q.st + W.h * a.q.sh, R.q, a.negate ? 0x80008000u : 0u);
    R.m = -INFINITY;
    R.l = R.l16 = 0.0f;
    R.met = false;
#pragma unroll
    for (int d = 0; d < NT; ++d) R.o[d] = pf16_t{};

    const int wlast = a.causal ? W.last : S.len - 1;                                  // the last that the wave sees
    auto step = [&](const char *K, const char *V, int j0) {
        j0 += kPtKeys * upper;
        if (!W.live || j0 > wlast) return;
        const bool masked = j0 + kPtKeys > S.len || (a.causal && j0 + kPtKeys - 1 > W.first);
        pt_forward_tile<DT, D, LO>(a, A, R, K, V, TILE * upper, j0, S.len, masked, j0 == 0);
    };
    for (int j0 = 0; j0 < kend; j0 += 2 * STEP) {
        pt_sync();                       // this tile is there, the other buffers are read
        copy(j0 + STEP, k1, v1);
        step(k0, v0, j0);
        if (j0 + STEP >= kend) break;
        pt_sync();
        copy(j0 + 2 * STEP, k0, v0);
        step(k1, v1, j0 + STEP);
    }
    if constexpr (KS == 2) {
        char *lds = (wave & 2 ? k1 : k0) + (wave & 1) * TILE;
        float4 *stat = reinterpret_cast<float4 *>(v0) + wave * 64 + (threadIdx.x & 63);
        __syncthreads();
        if (upper) {
            pt_give(lds, R.o);
            *stat = make_float4(R.m, R.l, R.l16, R.met ? 1.0f : 0.0f);
        }
        __syncthreads();
        if (upper) return;
        const float4 u = *stat;
        const float mn = fmaxf(R.m, u.x);
        const float f = R.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R.m - mn), fu = u.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(u.x - mn);
        R.l = R.l * f + u.y * fu;
        R.l16 = R.l16 * f + u.z * fu;
        R.m = mn;
        R.met = R.met || u.w != 0.0f;
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) R.o[d][i] *= f;
        pt_take(lds, R.o, fu);
    }
    if (!W.live) return;
    if (R.met) {
        // term by term, the maximum being known (of the rounded probabilities' sums alone)
        const float off = (R.m == -INFINITY ? 0.0f : R.m) - (DT == OMNI_F16 ? kPtF16Up : 0.0f);
        const int end = a.causal ? R.t + 1 : S.len;
        R.l = 0.0f;
        float o[NT][16];
        pt_clear(o);
#pragma unroll 1
        for (int j0 = 0; j0 <= wlast; j0 += 32) {
            pf16_t p = pt_product<DT, D>(kb, a.k.st, j0, S.len, 0.0f, [&](int kk) { return R.q[kk]; });
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], a.c, -off));
                if (j0 + 8 * (i / 4) + 4 * (int)((threadIdx.x >> 5) & 1) + i % 4 >= end) p[i] = 0.0f;
                R.l += p[i];
            }
            pt_add_terms<DT, D>(o, p, vb, a.v.st, j0, 0, end);
        }
        R.l16 = R.l;
        pt_assign(R.o, o);
    }

    const int64_t at = S.start + W.t;
    const float inv = 1.0f / pt_sum_halves(R.l16), l = pt_sum_halves(R.l);
    char *op = const_cast<char *>(a.o.p) + at * a.o.st + W.h * a.o.sh;
    if constexpr (LO) pt_store<DT, D, true>(op, R.o, inv, W.mine, const_cast<char *>(a.olo.p) + at * a.olo.st + W.h * a.olo.sh);
    else pt_store<DT, D>(op, R.o, inv, W.mine);
    if (a.lse && W.mine && (threadIdx.x & 32) == 0)
        a.lse[(int64_t)W.h * a.N + at] = (R.m - (DT == OMNI_F16 ? kPtF16Up : 0.0f) + __log2f(l)) * 0.69314718f;
}

// ── backward ────────────────────────────────────────────────────────────
//
// delta_t = sum_d g_td o_td;  p_ts = exp(scale q_t . k_s - lse_t);
//   dv_s = sum_t p_ts g_t,            ds_ts = p_ts (g_t . v_s - delta_t),
//   dq_t = scale sum_s ds_ts k_s,     dk_s = scale sum_t ds_ts q_t,
// dk and dv summed over the group's query heads.  Two launches without atomics,
// so that results repeat bit for bit: delta and dq by blocks of query rows; dk
// and dv by blocks of keys (delta in a launch of its own, which reads what dq's
// reads again, took 46 us of a gradient of 8192 tokens).  Scores and g . v are formed twice for it,
// seven products instead of five.
//
// 8192 tokens of 32 heads over 8 of 128 without a mask, bf16: dq 1.40 to 1.50 ms,
// 1.10 to 1.18 PFLOP/s of its three products, dk and dv 1.90 to 2.07 ms, 1.06 to
// 1.16 of theirs; matrix units busy in 57 and 54 % of the cycles, clocks of 1.85
// to 2.0 GHz, the forward that keeps what a gradient needs 1.05 to 1.12 ms.  All
// three gradients are formed, also where only one is asked for.
//
// p and ds go to the matrix units in the inputs' 16 bits.  In f16, p is scaled
// by 2^14 (p <= 1) and ds by the power of two that brings its bound, twice the
// largest |g_t| |v_s|, to 2^15; the sums are scaled back in fp32.

constexpr int kPtPeaks = 512;
constexpr float kPtF16P = 14.0f;

// f16: largest squared norms of the rows of g and of v, a pair for each block.
template <int D>
__global__ __launch_bounds__(256) void prompt_peaks_kernel(PromptArgs a) {
    constexpr int LPH = D / 8, HPW = 64 / LPH;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, sub = lane % LPH, grp = lane / LPH;
    auto norm = [&](const PromptHeads &x, int64_t t, int h) {
        const ps8_t v = *reinterpret_cast<const ps8_t *>(x.p + t * x.st + h * x.sh + sub * 16);
        float s = pt_dot8<OMNI_F16>(v, v, 0.0f);
#pragma unroll
        for (int m = LPH / 2; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
        return s < INFINITY ? s : 0.0f;              // what is not finite has no say: its results are not either
    };
    float pg = 0.0f, pv = 0.0f;
    const int64_t rows = min((int64_t)max(a.cu[a.B], 0), a.N);   // what lies behind the last sequence counts for nothing
    for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < rows; t += (int64_t)gridDim.x * 4) {
        for (int h = 0; h < a.Hq; h += HPW) pg = fmaxf(pg, norm(a.g, t, min(h + grp, a.Hq - 1)));
        for (int h = 0; h < a.Hkv; h += HPW) pv = fmaxf(pv, norm(a.v, t, min(h + grp, a.Hkv - 1)));
    }
    __shared__ float peak[2][4];
#pragma unroll
    for (int m = 32; m >= LPH; m /= 2) {
        pg = fmaxf(pg, __shfl_xor(pg, m, 64));
        pv = fmaxf(pv, __shfl_xor(pv, m, 64));
    }
    if (lane == 0) {
        peak[0][wave] = pg;
        peak[1][wave] = pv;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float *p = peak[threadIdx.x];
        a.peaks[threadIdx.x * kPtPeaks + blockIdx.x] = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
    }
}

// The power of two for ds in f16 (1 in bf16), the same in every block.
template <int DT>
__device__ __forceinline__ float pt_ds_scale(const PromptArgs &a) {
    if constexpr (DT == OMNI_BF16) return 1.0f;
    float m[2] = {0.0f, 0.0f};
    for (int i = threadIdx.x & 63; i < a.peak_rows; i += 64)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[e] = fmaxf(m[e], a.peaks[e * kPtPeaks + i]);
#pragma unroll
    for (int w = 32; w > 0; w /= 2)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[e] = fmaxf(m[e], __shfl_xor(m[e], w, 64));
    const float bound = 2.0f * sqrtf(m[0]) * sqrtf(m[1]);
    if (!(bound > 0.0f)) return 1.0f;
    const int e = 14 - ilogbf(bound);                        // bound 2^e in [2^14, 2^15)
    return ldexpf(1.0f, min(max(e, -100), 100));
}

template <int DT, int D>
struct PtGradRow {
    static constexpr int NT = D / 32;
    ps8_t q[D / 16], g[D / 16];
    pf16_t dq[NT];
    float lse2, delta;
    int t;
    bool met;                            // an infinity or NaN among hidden keys
};

// One tile of 64 keys for the wave's 32 query rows; transposed like the forward.
template <int DT, int D>
__device__ __forceinline__ void pt_dq_tile(const PromptArgs &a, const PtLane<D> &lane_at, PtGradRow<DT, D> &R, const char *K, const char *V, int j0, int len,
                                           bool masked, float up) {
    const PtLane<D> A = lane_at.fresh();
    const int half = (threadIdx.x >> 5) & 1;
    R.met = R.met || (masked && !pt_all_finite<DT>(K, kPtKeys * 2 * D));
    const int seen = (a.causal ? min(R.t, len - 1) : len - 1) - j0 - 4 * half;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        pf16_t s = {}, dp;
        float first = R.delta;
        asm volatile("" : "+v"(first));  // sixteen copies made here, not kept through the loop
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = first;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) s = pt_mfma<DT>(A.rows(K, 32 * b, kk), R.q[kk], s);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) dp = pt_mfma<DT>(A.rows(V, 32 * b, kk), R.g[kk], dp);
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (32 * b + 8 * (i / 4) + i % 4 > seen) {
                    s[i] = a.hide;
                    dp[i] = 0.0f;
                }
        }
        uint32_t x[8];
        float ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i], a.cs, -R.lse2));
            ds[i] = p * (DT == OMNI_F16 ? dp[i] * up : dp[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = pt_pack<DT>(ds[2 * i], ds[2 * i + 1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const ps8_t xb = __builtin_bit_cast(ps8_t, make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]));
#pragma unroll
            for (int d = 0; d < D / 32; ++d) R.dq[d] = pt_mfma<DT>(A.cols(K, 32 * b + 16 * k, d), xb, R.dq[d]);
        }
    }
}

template <int DT, int D>
__global__ __launch_bounds__(64 * kPtWaves, 2) void prompt_dq_kernel(PromptArgs a) {
    __shared__ __attribute__((aligned(16))) char k0[kPtKeys * 2 * D], k1[kPtKeys * 2 * D];
    __shared__ __attribute__((aligned(16))) char v0[kPtKeys * 2 * D], v1[kPtKeys * 2 * D];
    const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int hk = (int)(bid % a.Hkv);
    const PtSlot S = pt_slot<kPtRows>(a.cu, a.B, a.N, a.G, bid / a.Hkv, true);
    if (S.tile < 0) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int row0 = S.tile * kPtRows;
    if (S.none) {
        pt_zero_rows<D, kPtRows>(a.dq, S.start, row0, S.len, hk * a.G, a.G);
        return;
    }
    const char *kb = a.k.p + (int64_t)S.start * a.k.st + hk * a.k.sh, *vb = a.v.p + (int64_t)S.start * a.v.st + hk * a.v.sh;
    PtCopy<D, kPtKeys> ck, cv;
    ck.init(wave);
    cv.init(wave);
    ck.issue(kb, a.k.st, 0, S.len, k0, wave);
    cv.issue(vb, a.v.st, 0, S.len, v0, wave);

    PtLane<D> A;
    A.init();
    PtQueries W;
    W.init(a, S, hk, row0 + 32 * wave);
    PtGradRow<DT, D> R;
    R.t = W.t;
    const int64_t at = S.start + W.t;
    pt_load_rows<D>(a.q.p + at * a.q.st + W.h * a.q.sh, R.q);
    pt_load_rows<D>(a.g.p + at * a.g.st + W.h * a.g.sh, R.g);
    {
        // delta of the rows, for the launch after this one as well
        ps8_t o[D / 16], rest[D / 16];
        pt_load_rows<D>(a.o.p + at * a.o.st + W.h * a.o.sh, o);
        pt_load_rows<D>(a.olo.p + at * a.olo.st + W.h * a.olo.sh, rest);
        float d[2] = {0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            d[0] = pt_dot8<DT>(R.g[kk], o[kk], d[0]);
            d[1] = pt_dot8<DT>(R.g[kk], rest[kk], d[1]);
        }
        R.delta = -pt_sum_halves(d[0] + d[1]);
        R.lse2 = a.lse[(int64_t)W.h * a.N + at] * 1.44269504f;
        if (W.mine && (threadIdx.x & 32) == 0) {
            a.delta[(int64_t)W.h * a.N + at] = R.delta;
            a.lse2[(int64_t)W.h * a.N + at] = R.lse2 - (DT == OMNI_F16 ? kPtF16P : 0.0f);
        }
    }
    const float up = pt_ds_scale<DT>(a);
#pragma unroll
    for (int d = 0; d < D / 32; ++d) R.dq[d] = pf16_t{};
    R.met = false;

    const int kend = a.causal ? min((row0 + kPtRows - 1) / a.G + 1, S.len) : S.len;
    const int wlast = a.causal ? W.last : S.len - 1;
    auto step = [&](const char *K, const char *V, int j0) {
        if (!W.live || j0 > wlast) return;
        pt_dq_tile<DT, D>(a, A, R, K, V, j0, S.len, j0 + kPtKeys > S.len || (a.causal && j0 + kPtKeys - 1 > W.first), up);
    };
    for (int j0 = 0; j0 < kend; j0 += 2 * kPtKeys) {
        pt_sync();
        if (j0 + kPtKeys < kend) {
            ck.issue(kb, a.k.st, j0 + kPtKeys, S.len, k1, wave);
            cv.issue(vb, a.v.st, j0 + kPtKeys, S.len, v1, wave);
        }
        step(k0, v0, j0);
        if (j0 + kPtKeys >= kend) break;
        pt_sync();
        if (j0 + 2 * kPtKeys < kend) {
            ck.issue(kb, a.k.st, j0 + 2 * kPtKeys, S.len, k0, wave);
            cv.issue(vb, a.v.st, j0 + 2 * kPtKeys, S.len, v0, wave);
        }
        step(k1, v1, j0 + kPtKeys);
    }
    if (!W.live) return;
    if (R.met) {
        float dq[D / 32][16];
        pt_clear(dq);
#pragma unroll 1
        for (int j0 = 0; j0 <= wlast; j0 += 32) {
            const pf16_t s = pt_product<DT, D>(kb, a.k.st, j0, S.len, 0.0f, [&](int kk) { return R.q[kk]; });
            pf16_t ds = pt_product<DT, D>(vb, a.v.st, j0, S.len, R.delta, [&](int kk) { return R.g[kk]; });
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] *= __builtin_amdgcn_exp2f(fmaf(s[i], a.cs, -R.lse2)) * up;
            pt_add_terms<DT, D>(dq, ds, kb, a.k.st, j0, 0, a.causal ? R.t + 1 : S.len);
        }
        pt_assign(R.dq, dq);
    }
    pt_store<DT, D>(const_cast<char *>(a.dq.p) + at * a.dq.st + W.h * a.dq.sh, R.dq, a.scale / up, W.mine);
}

// dk and dv: a wave holds 32 keys as B operands of S = Q K^T and G V^T, so
// that p and ds (rows on registers, keys on lanes) are the B operands of
// dv^T += G^T P and dk^T += Q^T dS; tiles of 64 rows of q and g go through LDS,
// one query head of the group after another.  Four waves share 128 keys and the
// first 32 rows of every tile, four more the same keys and the other rows; the
// halves are added through LDS at the end.  A wave's own run, every row that
// sees its keys, times the group, is the longest there is: at 4096 of 8192
// packed tokens and G = 4 it is longer than a CU's share of all, and with one
// wave for all rows (two blocks a CU) the launch took 690 us instead of 525 us.
//
// At D = 128 the sums of dk and dv take 128 registers a lane.  Two waves a SIMD
// (256 registers) then leave room for v's operands but not k's, which are read
// from LDS again for every tile.
constexpr int kPtKvWaves = 8;
constexpr int kPtKvKeys = 128;
constexpr int kPtQRows = 64;

template <int DT, int D>
struct PtGradKey {
    static constexpr int NT = D / 32;
    static constexpr bool KLDS = D == 128;
    ps8_t k[KLDS ? 1 : D / 16], v[D / 16];
    pf16_t dk[NT], dv[NT];
    int s;
    bool met;                            // an infinity or NaN among hidden rows, their statistics included
};

// Whether the row statistic's 32 values at `p` are finite.  A row may have none
// (a NaN, or an infinite score) where q and g are ordinary, and the exponential
// of a hidden score less a NaN is no 0.
__device__ __forceinline__ bool pt_stat_finite(const float *p) {
    return __builtin_amdgcn_ballot_w64((__float_as_uint(p[threadIdx.x & 31]) & 0x7f800000u) == 0x7f800000u) == 0;
}

// 32 rows from row j0 on, in the tiles from row r0 on.
template <int DT, int D>
__device__ __forceinline__ void pt_dkv_tile(const PromptArgs &a, const PtLane<D> &lane_at, PtGradKey<DT, D> &R, const char *K,
                                            const PtLane<D> &key_at, const char *Q, const char *G, const float *lse2,
                                            const float *delta, int j0, int r0, int len, bool masked, float up) {
    constexpr bool KLDS = PtGradKey<DT, D>::KLDS;
    const PtLane<D> A = lane_at.fresh(), AK = KLDS ? key_at.fresh() : A;
    R.met = R.met || (masked && !(pt_all_finite<DT>(Q + r0 * 2 * D, 64 * D) && pt_all_finite<DT>(G + r0 * 2 * D, 64 * D) &&
                                  pt_stat_finite(lse2)));
    const int half = (threadIdx.x >> 5) & 1;
    pf16_t s = {}, dp;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 d4 = *reinterpret_cast<const float4 *>(delta + 2 * i + 4 * half);
        dp[i] = d4.x; dp[i + 1] = d4.y; dp[i + 2] = d4.z; dp[i + 3] = d4.w;
    }
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        s = pt_mfma<DT>(A.rows(Q, 0, kk), KLDS ? AK.rows(K, 0, kk) : R.k[KLDS ? 0 : kk], s);
        dp = pt_mfma<DT>(A.rows(G, 0, kk), R.v[kk], dp);
    }
    if (masked) {
        // register i is row j0 + 8 (i / 4) + 4 half + i % 4
        const int first = (a.causal ? R.s : 0) - j0 - 4 * half, end = len - j0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 8 * (i / 4) + i % 4;
            if (row < first || row >= end) {
                s[i] = a.hide;
                dp[i] = 0.0f;
            }
        }
    }
    uint32_t x[8], y[8];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 l4 = *reinterpret_cast<const float4 *>(lse2 + 2 * i + 4 * half);
        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
        float p[4], ds[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(s[i + e], a.cs, -l[e]));
            ds[e] = p[e] * (DT == OMNI_F16 ? dp[i + e] * up : dp[i + e]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            x[i / 2 + e] = pt_pack<DT>(p[2 * e], p[2 * e + 1]);
            y[i / 2 + e] = pt_pack<DT>(ds[2 * e], ds[2 * e + 1]);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const ps8_t xb = pt_frag(x + 4 * k), yb = pt_frag(y + 4 * k);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            R.dv[d] = pt_mfma<DT>(A.cols(G, 16 * k, d), xb, R.dv[d]);
            R.dk[d] = pt_mfma<DT>(A.cols(Q, 16 * k, d), yb, R.dk[d]);
        }
    }
}

// kPtQRows floats of a row statistic, from row j0 of the sequence on (rows from len on repeat the last).
__device__ __forceinline__ void pt_copy_stat(const float *base, int j0, int len, float *lds) {
    const int left = min(len - j0, kPtQRows);
    const __amdgpu_buffer_rsrc_t R = __builtin_amdgcn_make_buffer_rsrc((void *)(base + j0), (short)0, left * 4, kPtBufWord3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(R, (PT_LDS void *)lds, 4, (uint32_t)min((int)(threadIdx.x & 63), left - 1) * 4u, 0, 0, 0);
}

template <int DT, int D>
__global__ __launch_bounds__(64 * kPtKvWaves, 2) void prompt_dkv_kernel(PromptArgs a) {
    constexpr bool KLDS = PtGradKey<DT, D>::KLDS;
    __shared__ __attribute__((aligned(16))) char q0[kPtQRows * 2 * D], q1[kPtQRows * 2 * D];
    __shared__ __attribute__((aligned(16))) char g0[kPtQRows * 2 * D], g1[kPtQRows * 2 * D];
    __shared__ __attribute__((aligned(16))) char kt[KLDS ? kPtKvKeys * 2 * D : 16];
    __shared__ __attribute__((aligned(16))) float l0[kPtQRows], l1[kPtQRows], d0[kPtQRows], d1[kPtQRows];
    const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int hk = (int)(bid % a.Hkv);
    // the first keys are seen by the most rows
    const int64_t rest = bid / a.Hkv;
    const int part = (int)(rest % a.n_parts), GP = a.G / a.n_parts, h0 = hk * a.G + part * GP;   // the query heads of this block
    const PtSlot S = pt_slot<kPtKvKeys>(a.cu, a.B, a.N, 1, rest / a.n_parts, false);
    if (S.tile < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kw = wave & 3, upper = wave >> 2;
    const int key0 = S.tile * kPtKvKeys;
    if (S.none) {
        if (part) return;
        pt_zero_rows<D, kPtKvKeys>(a.dk, S.start, key0, S.len, hk, 1);
        pt_zero_rows<D, kPtKvKeys>(a.dv, S.start, key0, S.len, hk, 1);
        return;
    }
    const int first = a.causal ? key0 / kPtQRows : 0, tiles = (S.len + kPtQRows - 1) / kPtQRows - first;
    const int n = tiles * GP;
    PtCopy<D, kPtQRows> cp;
    cp.init(kw);
    const PromptHeads &src = upper ? a.g : a.q;          // the lower waves copy q, the upper g
    const char *sb = src.p + (int64_t)S.start * src.st + (int64_t)h0 * src.sh;
    const float *stat = (upper ? a.delta : a.lse2) + (int64_t)h0 * a.N + S.start;
    int gi = 0, ji = first;              // head and tile that the next copy takes
    auto copy = [&](char *Q, char *G, float *L, float *Dl) {
        cp.issue(sb + gi * src.sh, src.st, ji * kPtQRows, S.len, upper ? G : Q, kw);
        if (kw == 0) pt_copy_stat(stat + gi * a.N, ji * kPtQRows, S.len, upper ? Dl : L);
        if (++ji == first + tiles) {
            ji = first;
            ++gi;
        }
    };
    if constexpr (KLDS) {
        static_assert(kPtKvKeys == 2 * kPtQRows, "a half of the keys by either half of the waves");
        const int k0 = key0 + kPtQRows * upper;
        if (k0 < S.len)
            cp.issue(a.k.p + (int64_t)S.start * a.k.st + hk * a.k.sh, a.k.st, k0, S.len, kt + kPtQRows * 2 * D * upper, kw);
    }
    copy(q0, g0, l0, d0);

    PtLane<D> A, AK;
    A.init(32 * upper);
    AK.init(32 * kw);
    PtGradKey<DT, D> R;
    const int w0 = key0 + 32 * kw;
    R.s = w0 + (lane & 31);
    const int64_t at = S.start + min(R.s, S.len - 1);
    if constexpr (!KLDS) pt_load_rows<D>(a.k.p + at * a.k.st + hk * a.k.sh, R.k);
    pt_load_rows<D>(a.v.p + at * a.v.st + hk * a.v.sh, R.v);
    const float scale = pt_ds_scale<DT>(a), up = DT == OMNI_F16 ? scale * 6.103515625e-5f : 1.0f;   // p is times 2^14
#pragma unroll
    for (int d = 0; d < D / 32; ++d) R.dk[d] = R.dv[d] = pf16_t{};
    R.met = false;
    const bool live = w0 < S.len;
    int jc = first;                      // tile in hand
    auto step = [&](const char *Q, const char *G, const float *L, const float *Dl) {
        const int j0 = jc * kPtQRows + 32 * upper;
        jc = jc + 1 == first + tiles ? first : jc + 1;
        if (!live || j0 >= S.len || (a.causal && j0 + 31 < w0)) return;
        pt_dkv_tile<DT, D>(a, A, R, kt, AK, Q, G, L + 32 * upper, Dl + 32 * upper, j0, 32 * upper, S.len,
                           j0 + 32 > S.len || (a.causal && j0 < w0 + 31), up);
    };
    for (int i = 0; i < n; i += 2) {
        pt_sync();
        if (i + 1 < n) copy(q1, g1, l1, d1);
        step(q0, g0, l0, d0);
        if (i + 1 >= n) break;
        pt_sync();
        if (i + 2 < n) copy(q0, g0, l0, d0);
        step(q1, g1, l1, d1);
    }
    if (R.met) {
        // dk, then dv, each alone: both at once take registers that the loop above could not have
        auto again = [&](pf16_t (&sum)[D / 32], auto keys) {
            constexpr bool DK = decltype(keys)::value;
            float acc[D / 32][16];
            pt_clear(acc);
#pragma unroll 1
            for (int g = 0; g < GP; ++g) {
                const int64_t h = h0 + g;
                const char *qb = a.q.p + (int64_t)S.start * a.q.st + h * a.q.sh, *gb = a.g.p + (int64_t)S.start * a.g.st + h * a.g.sh;
#pragma unroll 1
                for (int j0 = (a.causal ? w0 / 64 * 64 : 0) + 32 * upper; j0 < S.len; j0 += 64) {   // the rows that this half takes in every tile
                    if (a.causal && j0 + 31 < w0) continue;
                    const int64_t row = h * a.N + S.start + min(j0 + (lane & 31), S.len - 1);
                    const float l = a.lse2[row], d = a.delta[row];
                    pf16_t w = pt_product<DT, D>(qb, a.q.st, j0, S.len, 0.0f, [&](int kk) { return KLDS ? AK.rows(kt, 0, kk) : R.k[KLDS ? 0 : kk]; });
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        w[i] = __builtin_amdgcn_exp2f(fmaf(w[i], a.cs, -__shfl(l, 8 * (i / 4) + 4 * (lane >> 5) + i % 4, 64)));
                    if constexpr (DK) {
                        const pf16_t dp = pt_product<DT, D>(gb, a.g.st, j0, S.len, 0.0f, [&](int kk) { return R.v[kk]; });
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] *= (dp[i] + __shfl(d, 8 * (i / 4) + 4 * (lane >> 5) + i % 4, 64)) * up;
                    }
                    pt_add_terms<DT, D>(acc, w, DK ? qb : gb, DK ? a.q.st : a.g.st, j0, a.causal ? R.s : 0, S.len);
                }
            }
            pt_assign(sum, acc);
        };
        again(R.dk, std::true_type());
        again(R.dv, std::false_type());
    }
    // dk, then dv, of the upper half by way of the tiles' buffers, one a wave
    char *lds = kw == 0 ? q0 : kw == 1 ? q1 : kw == 2 ? g0 : g1;
    __syncthreads();
    if (upper) pt_give(lds, R.dk);
    __syncthreads();
    if (!upper) pt_take(lds, R.dk);
    __syncthreads();
    if (upper) pt_give(lds, R.dv);
    __syncthreads();
    if (upper || !live) return;
    pt_take(lds, R.dv);
    const bool mine = R.s < S.len;
    const float fk = a.scale / scale, fv = DT == OMNI_F16 ? 6.103515625e-5f : 1.0f;
    if (a.n_parts == 1) {
        pt_store<DT, D>(const_cast<char *>(a.dk.p) + (int64_t)(S.start + R.s) * a.dk.st + hk * a.dk.sh, R.dk, fk, mine);
        pt_store<DT, D>(const_cast<char *>(a.dv.p) + (int64_t)(S.start + R.s) * a.dv.st + hk * a.dv.sh, R.dv, fv, mine);
    } else if (mine) {
        float *p = a.parts + (((int64_t)part * 2 * a.N + S.start + R.s) * a.Hkv + hk) * D + 4 * (lane >> 5), *q = p + a.N * a.Hkv * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                *reinterpret_cast<float4 *>(p + 32 * d + 2 * i) = make_float4(R.dk[d][i] * fk, R.dk[d][i + 1] * fk, R.dk[d][i + 2] * fk, R.dk[d][i + 3] * fk);
                *reinterpret_cast<float4 *>(q + 32 * d + 2 * i) = make_float4(R.dv[d][i] * fv, R.dv[d][i + 1] * fv, R.dv[d][i + 2] * fv, R.dv[d][i + 3] * fv);
            }
    }
}

// dk and dv of the parts, added in their order: a thread for eight dims.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_parts_kernel(PromptArgs a) {
    const int64_t rows = min((int64_t)max(a.cu[a.B], 0), a.N), each = a.N * a.Hkv * D;
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    const int d = (int)(e % D), hk = (int)(e / D % a.Hkv);
    const int64_t t = e / D / a.Hkv;
    if (t >= rows) return;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        float x[8] = {};
        for (int p = 0; p < a.n_parts; ++p) {
            const float4 *src = reinterpret_cast<const float4 *>(a.parts + (2 * p + w) * each + e);
            const float4 u = src[0], v = src[1];
            x[0] += u.x; x[1] += u.y; x[2] += u.z; x[3] += u.w;
            x[4] += v.x; x[5] += v.y; x[6] += v.z; x[7] += v.w;
        }
        const PromptHeads &o = w ? a.dv : a.dk;
        *reinterpret_cast<uint4 *>(const_cast<char *>(o.p) + t * o.st + hk * o.sh + 2 * d) =
            make_uint4(pt_pack<DT>(x[0], x[1]), pt_pack<DT>(x[2], x[3]), pt_pack<DT>(x[4], x[5]), pt_pack<DT>(x[6], x[7]));
    }
}

// ── host ────────────────────────────────────────────────────────────────

static int prompt_heads(const char *who, const char *what, const void *p, const int64_t *s, PromptHeads &t) {
    OMNI_CHECK_ARG(p && s, "%s: NULL %s", who, what);
    OMNI_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0,
                   "%s: %s and its strides must be multiples of 16 bytes", who, what);
    // a tile's 64 rows are addressed with 32-bit offsets
    OMNI_CHECK_ARG(s[0] >= 0 && s[0] < (int64_t(1) << 24) && s[1] >= 0, "%s: %s: token stride out of range", who, what);
    t.p = static_cast<const char *>(p);
    t.st = 2 * s[0];
    t.sh = 2 * s[1];
    return OMNI_OK;
}

static int prompt_args(const char *who, int dtype, int64_t N, int Hq, int Hkv, int D, const int32_t *cu, int64_t B, float scale,
                       PromptArgs &a) {
    OMNI_CHECK_ARG(dtype == OMNI_F16 || dtype == OMNI_BF16, "%s: dtype must be f16 or bf16", who);
    OMNI_CHECK_ARG(D == 32 || D == 64 || D == 128, "%s: head_dim must be 32, 64 or 128, got %d", who, D);
    OMNI_CHECK_ARG(N >= 0 && B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "%s: bad shape (Hq must be a multiple of Hkv)", who);
    OMNI_CHECK_ARG(N < (int64_t(1) << 31) && N * Hq < (int64_t(1) << 31) - 1024 && B < (int64_t(1) << 30), "%s: shape too large", who);
    // times log2 e it stays finite
    OMNI_CHECK_ARG(scale == scale && fabsf(scale) <= 2.3e38f, "%s: scale must be finite and at most 2.3e38 in size", who);
    a.N = N;
    a.B = (int)B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.cu = cu;
    a.negate = scale < 0.0f;
    a.scale = scale;
    // a scale of 0 is next to 0 instead, so that hidden scores stay at -inf
    a.c = fmaxf(fabsf(scale) * 1.44269504088896f, 1.0e-37f);
    a.cs = scale < 0.0f ? -a.c : a.c;
    a.hide = scale < 0.0f ? INFINITY : -INFINITY;
    return OMNI_OK;
}

// Fewer than 2^32 threads in a dimension.
static bool prompt_grid(int64_t blocks, dim3 &grid) {
    const int64_t gx = blocks < (1 << 22) ? blocks : (1 << 22), gy = (blocks + gx - 1) / gx;
    grid = dim3((unsigned)gx, (unsigned)gy);
    return gy <= 65535;
}

}  // namespace omni

using namespace omni;

template <int DT, int D>
static void prompt_launch_forward(const PromptArgs &a, dim3 grid, hipStream_t st) {
    // Where all blocks start at once and rows are long, the longest block is the
    // launch's time: eight waves a block halve it.  Two waves of one block keep
    // step on their SIMD, though, where those of two blocks fill each other's
    // gaps, so that it pays up to two four-wave blocks a CU only, and not for
    // short sequences.  Four waves against eight, causal, head_dim 128, 32 heads
    // over 8: 1024 tokens 30 / 26 us, 1536 44 / 37, 1792 49 / 44, 2048 (two blocks
    // a CU) 55 / 51, 2304 62 / 67, 2560 71 / 78, 3000 86 / 98; 8 heads over 1:
    // 2048 46 / 36, 4096 88 / 66, 8192 (two blocks a CU) 189 / 147; 16 sequences of
    // 128 15 / 21; head_dim 32, 2048 tokens 27 / 23.  Lengths are known here by
    // their mean alone: 4096 tokens beside 30 single ones, 8 heads over 1, stay
    // with four waves, 88 / 65.
    const bool split = a.N * a.Hq / kPtRows <= 2 * device_cus() && a.N >= (int64_t)1024 * a.B;
    const dim3 one(64 * kPtWaves), two(2 * 64 * kPtWaves);
    if (a.olo.p && split) hipLaunchKernelGGL((prompt_forward_kernel<DT, D, true, 2>), grid, two, 0, st, a);
    else if (a.olo.p) hipLaunchKernelGGL((prompt_forward_kernel<DT, D, true, 1>), grid, one, 0, st, a);
    else if (split) hipLaunchKernelGGL((prompt_forward_kernel<DT, D, false, 2>), grid, two, 0, st, a);
    else hipLaunchKernelGGL((prompt_forward_kernel<DT, D, false, 1>), grid, one, 0, st, a);
}
template <int DT>
static void prompt_launch_forward(const PromptArgs &a, int D, dim3 grid, hipStream_t st) {
    if (D == 32) prompt_launch_forward<DT, 32>(a, grid, st);
    else if (D == 64) prompt_launch_forward<DT, 64>(a, grid, st);
    else prompt_launch_forward<DT, 128>(a, grid, st);
}

extern "C" int omni_prompt_attn(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v,
                                const int64_t *v_strides, int dtype, int64_t N, int Hq, int Hkv, int head_dim,
                                const int32_t *cu_seqlens, int64_t B, float scale, int causal, int fill_rest, void *out,
                                const int64_t *out_strides, float *lse, void *out_rest, const int64_t *out_rest_strides,
                                void *stream) {
    const char *who = "omni_prompt_attn";
    PromptArgs a = {};
    OMNI_TRY(prompt_args(who, dtype, N, Hq, Hkv, head_dim, cu_seqlens, B, scale, a));
    if (N == 0) return OMNI_OK;
    OMNI_TRY(prompt_heads(who, "q", q, q_strides, a.q));
    OMNI_TRY(prompt_heads(who, "k", k, k_strides, a.k));
    OMNI_TRY(prompt_heads(who, "v", v, v_strides, a.v));
    OMNI_TRY(prompt_heads(who, "out", out, out_strides, a.o));
    if (out_rest) OMNI_TRY(prompt_heads(who, "out_rest", out_rest, out_rest_strides, a.olo));
    OMNI_CHECK_ARG(cu_seqlens, "%s: NULL cu_seqlens", who);
    a.lse = lse;
    a.causal = causal != 0;
    a.fill = fill_rest != 0;
    dim3 grid;
    OMNI_CHECK_ARG(prompt_grid((N * a.G / kPtRows + B + 1) * Hkv, grid), "%s: grid too large", who);
    if (dtype == OMNI_F16) prompt_launch_forward<OMNI_F16>(a, head_dim, grid, as_stream(stream));
    else prompt_launch_forward<OMNI_BF16>(a, head_dim, grid, as_stream(stream));
    OMNI_CHECK_LAUNCH(who);
    return OMNI_OK;
}

template <int DT, int D>
static int prompt_launch_backward(const PromptArgs &a, hipStream_t st) {
    const char *who = "omni_prompt_attn_backward";
    dim3 rows, keys;
    OMNI_CHECK_ARG(prompt_grid((a.N * a.G / kPtRows + a.B + 1) * a.Hkv, rows) && prompt_grid((a.N / kPtKvKeys + a.B + 1) * a.Hkv * a.n_parts, keys),
                   "%s: grid too large", who);
    if constexpr (DT == OMNI_F16) {
        hipLaunchKernelGGL((prompt_peaks_kernel<D>), dim3(a.peak_rows), dim3(256), 0, st, a);
        OMNI_CHECK_LAUNCH(who);
    }
    hipLaunchKernelGGL((prompt_dq_kernel<DT, D>), rows, dim3(64 * kPtWaves), 0, st, a);
    OMNI_CHECK_LAUNCH(who);
    hipLaunchKernelGGL((prompt_dkv_kernel<DT, D>), keys, dim3(64 * kPtKvWaves), 0, st, a);
    OMNI_CHECK_LAUNCH(who);
    if (a.n_parts > 1) {
        // fewer than 2^24 rows of dk (prompt_parts)
        hipLaunchKernelGGL((prompt_parts_kernel<DT, D>), dim3((unsigned)((a.N * a.Hkv * D / 8 + 255) / 256)), dim3(256), 0, st, a);
        OMNI_CHECK_LAUNCH(who);
    }
    return OMNI_OK;
}

// Parts that the query heads of a kv head are dealt to in the launch for dk and
// dv, whose blocks each hold a CU: doubled while there are not two blocks for
// each CU, since a first key's block runs through every row of every head.  Each
// part writes its sums in fp32 and another launch adds them.  32 heads over 8 of
// 128, causal, the whole gradient, one part against this rule against four
// blocks a CU: 2048 tokens 283 / 185 / 185 us, 4096 628 / 508 / 528, nine
// sequences of 20 to 3000 tokens 498 / 451 / 499, 8192 1829 / 1832 / 1842;
// 4096 without a mask 893 / 916 / 939.
// Halves only: a group of 3, 5 or 7 heads stays whole, one of 6 is two parts.
static int prompt_parts(int64_t N, int64_t B, int Hq, int Hkv) {
    const int G = Hq / Hkv;
    const int64_t blocks = (N / kPtKvKeys + B) * Hkv;
    int parts = 1;
    while (G % (2 * parts) == 0 && blocks * parts < 2 * device_cus()) parts *= 2;
    return parts;
}

static size_t prompt_stats_bytes(int64_t N, int Hq) {
    return (((size_t)N * (size_t)Hq * 2 + 2 * kPtPeaks) * 4 + 15) / 16 * 16;
}

extern "C" size_t omni_prompt_attn_backward_workspace_size(int64_t N, int Hq, int Hkv, int head_dim, int64_t B) {
    if (N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || B < 0) return 0;
    const int parts = prompt_parts(N, B, Hq, Hkv);
    return prompt_stats_bytes(N, Hq) + (parts > 1 ? (size_t)parts * 2 * (size_t)N * (size_t)Hkv * (size_t)head_dim * 4 : 0);
}

extern "C" int omni_prompt_attn_backward(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides,
                                         const void *v, const int64_t *v_strides, int dtype, int64_t N, int Hq, int Hkv,
                                         int head_dim, const int32_t *cu_seqlens, int64_t B, float scale, int causal,
                                         const void *out, const int64_t *out_strides, const void *out_rest,
                                         const int64_t *out_rest_strides, const float *lse, const void *dout,
                                         const int64_t *dout_strides, void *dq, const int64_t *dq_strides, void *dk,
                                         const int64_t *dk_strides, void *dv, const int64_t *dv_strides, void *workspace,
                                         size_t workspace_bytes, void *stream) {
    const char *who = "omni_prompt_attn_backward";
    PromptArgs a = {};
    OMNI_TRY(prompt_args(who, dtype, N, Hq, Hkv, head_dim, cu_seqlens, B, scale, a));
    if (N == 0) return OMNI_OK;
    OMNI_TRY(prompt_heads(who, "q", q, q_strides, a.q));
    OMNI_TRY(prompt_heads(who, "k", k, k_strides, a.k));
    OMNI_TRY(prompt_heads(who, "v", v, v_strides, a.v));
    OMNI_TRY(prompt_heads(who, "out", out, out_strides, a.o));
    OMNI_TRY(prompt_heads(who, "out_rest", out_rest, out_rest_strides, a.olo));
    OMNI_TRY(prompt_heads(who, "dout", dout, dout_strides, a.g));
    OMNI_TRY(prompt_heads(who, "dq", dq, dq_strides, a.dq));
    OMNI_TRY(prompt_heads(who, "dk", dk, dk_strides, a.dk));
    OMNI_TRY(prompt_heads(who, "dv", dv, dv_strides, a.dv));
    OMNI_CHECK_ARG(cu_seqlens && lse, "%s: NULL cu_seqlens or lse", who);
    const size_t need = omni_prompt_attn_backward_workspace_size(N, Hq, Hkv, head_dim, B);
    if (!workspace || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes needed", who, need);
        return OMNI_EWORKSPACE;
    }
    OMNI_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: workspace must be 16-byte aligned", who);
    a.lse = const_cast<float *>(lse);
    a.peaks = static_cast<float *>(workspace);
    a.lse2 = a.peaks + 2 * kPtPeaks;
    a.delta = a.lse2 + (size_t)N * Hq;
    a.n_parts = prompt_parts(N, B, Hq, Hkv);
    a.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + prompt_stats_bytes(N, Hq));
    a.causal = causal != 0;
    a.peak_rows = (int)(N / 4 + 1 < kPtPeaks ? N / 4 + 1 : kPtPeaks);
    hipStream_t st = as_stream(stream);
    if (dtype == OMNI_F16) {
        if (head_dim == 32) return prompt_launch_backward<OMNI_F16, 32>(a, st);
        if (head_dim == 64) return prompt_launch_backward<OMNI_F16, 64>(a, st);
        return prompt_launch_backward<OMNI_F16, 128>(a, st);
    }
    if (head_dim == 32) return prompt_launch_backward<OMNI_BF16, 32>(a, st);
    if (head_dim == 64) return prompt_launch_backward<OMNI_BF16, 64>(a, st);
    return prompt_launch_backward<OMNI_BF16, 128>(a, st);
}
