// The paged INT4 + QJL cache's blocks (pages) on gfx950: the bounds of a
// block's key codes (omni_block_bounds), the selection of each query's blocks
// by a score that reads the bounds alone (omni_block_select), and the move of
// accepted drafted tokens within their sequence (omni_cache_keep).  head_dim
// 128.
//
// Bounds: byte d of (page, head) is lo | hi << 4, the least and the largest key
// code of dim d over the block's tokens.  Score of a block for the query heads
// of one kv head, with codebooks that ascend:
//   sum_h max_{lo <= code <= hi} q_h . c  =  sum_d Q+_d c[hi_d] - Q-_d c[lo_d],
//   Q+ = sum_h max(q_h, 0),  Q- = sum_h max(-q_h, 0)
// an upper bound of the group's summed scores q . c[code] (the residual signs
// are left out), here in whole numbers: Q and the head's centroids are each
// multiplied by the power of two that brings their largest into [64, 128) and
// rounded to the nearest int8 (127 at most), so that a score lies above or below
// the bound by what those roundings sum up to.  A sum of 256 products of int8
// lies below 2^22, so it does not depend on its order; equal scores are equal,
// and the lower block wins.  Q+ and Q- are summed in fp64 (rotated rows without
// the factor 1/sqrt(128), which does not change the order): exact for f16 (40
// bits a value, 47 a rotated one) of up to 1024 heads, 64 rotated, and for bf16
// (8 bits a value) where the exponents that meet in a sum span up to 45 bits
// less those that its number of terms adds; past that a sum is off by 2^-53 of
// itself, which can move a rounding to int8 at a tie only.
#include <math.h>

#include "omni_common.h"

namespace omni {

int check_pool(const char *who, int64_t n_pages, int Hkv, int page_size, int64_t max_pages, int &shift);

// ── bounds ──────────────────────────────────────────────────────────────

struct BoundsArgs {
    const uint8_t *k_nib;
    uint8_t *bounds;
    const int32_t *page_table, *start, *end;     // end NULL: start + count
    const int32_t *kept;                         // with it, count of them: the tokens that a move of drafted tokens leaves
    int64_t max_pages, n_pages, count;
    int64_t page0;                               // pages of each sequence that earlier launches took
    int Hkv, page_shift;
};

// One block per (sequence, page that holds a token of [start, end)): a wave
// per head; lane (c, k) reads code bytes 4 c .. + 3 of tokens k, k + 4, ...
// and keeps nibble minima and maxima in 16-bit lanes.  The page's first tokens
// up to `end` count, whatever start is, so what a page says does not depend on
// how it was filled.  Bound by latency where a decode step touches a page per
// sequence (4 to 6 us), else by 4-byte loads and 16 lane moves per KB of codes
// (8 x 131072 tokens, 537 MB: 153 to 174 us, 3.1 to 3.5 TB/s, 104 us at a copy's
// rate); wider loads have not been tried.
__global__ __launch_bounds__(256) void block_bounds_kernel(BoundsArgs a) {
    typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
    const int64_t b = blockIdx.y;
    const int64_t cap = a.max_pages << a.page_shift;
    int64_t s = a.start[b], e = a.end ? (int64_t)a.end[b] : s + a.count;
    if (a.kept) {
        // up to the last kept token; the page of the token before them, which
        // the dropped ones may have widened, also where none is kept
        e = s;
        for (int j = 0; j < a.count; ++j) e = (uint32_t)a.kept[b * a.count + j] < 64u ? s + j + 1 : e;
        --s;
    }
    s = s < 0 ? 0 : s;                           // rows outside the table are not written by an append either
    e = e > cap ? cap : e;
    if (s >= e) return;
    const int64_t pi = (s >> a.page_shift) + a.page0 + blockIdx.x;
    if (pi << a.page_shift >= e) return;
    const int32_t id = a.page_table[b * a.max_pages + pi];
    if (id < 0 || id >= a.n_pages) return;
    const int64_t left = e - (pi << a.page_shift);
    const int nv = left < (1 << a.page_shift) ? (int)left : 1 << a.page_shift;
    const int lane = threadIdx.x & 63, c = lane & 15, k = lane >> 4;
    for (int h = threadIdx.x >> 6; h < a.Hkv; h += 4) {
        const uint8_t *src = a.k_nib + (((int64_t)id * a.Hkv + h) << a.page_shift) * 64 + 4 * c;
        us2_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[j] = us2_t{15, 15};
            hi[j] = us2_t{0, 0};
        }
#pragma unroll 4
        for (int t = k; t < nv; t += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(src + (int64_t)t * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const us2_t v = __builtin_bit_cast(us2_t, (w >> (4 * j)) & 0x000F000Fu);
                lo[j] = __builtin_elementwise_min(lo[j], v);
                hi[j] = __builtin_elementwise_max(hi[j], v);
            }
        }
        uint32_t out[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int m = 16; m < 64; m <<= 1) {
                lo[j] = __builtin_elementwise_min(lo[j], __builtin_bit_cast(us2_t, __shfl_xor(__builtin_bit_cast(int, lo[j]), m)));
                hi[j] = __builtin_elementwise_max(hi[j], __builtin_bit_cast(us2_t, __shfl_xor(__builtin_bit_cast(int, hi[j]), m)));
            }
            // nibble j of the low half is dim 8 c + j, of the high half 8 c + 4 + j
            out[0] |= (uint32_t)(lo[j][0] | (hi[j][0] << 4)) << (8 * j);
            out[1] |= (uint32_t)(lo[j][1] | (hi[j][1] << 4)) << (8 * j);
        }
        if (k == 0) *reinterpret_cast<uint2 *>(a.bounds + ((int64_t)id * a.Hkv + h) * 128 + 8 * c) = make_uint2(out[0], out[1]);
    }
}

// ── scores ──────────────────────────────────────────────────────────────

struct SelectArgs {
    const void *q;
    const uint8_t *bounds;
    const int32_t *page_table, *seq_lens;
    const float *codebooks;
    const int8_t *sign_flip;
    int32_t *scores;             // [(b T + t) Hkv + hk][max_pages], as keys
    int32_t *blocks;             // (B, Hkv, T, top)
    int64_t max_pages, n_pages;
    int page_shift, per_head, Hq, Hkv, G, T, top, first, recent, rotate, f16;
    int per_block, heads;        // block_score_kernel: blocks and kv heads of a thread block
};

// Blocks that query (b, t) sees; 0 where the length does not fit the table.
__device__ __forceinline__ int64_t seen_blocks(const SelectArgs &a, int64_t b, int t) {
    const int64_t len = a.seq_lens[b], cap = a.max_pages << a.page_shift;
    const int64_t seen = len < 0 || len > cap ? 0 : len - a.T + t + 1;
    return seen <= 0 ? 0 : (seen + (1 << a.page_shift) - 1) >> a.page_shift;
}

// 2^k with most * 2^k in [64, 128)
__device__ __forceinline__ double whole_scale(double most) {
    const uint64_t e = (__builtin_bit_cast(uint64_t, most) >> 52) & 0x7ffu;
    return __builtin_bit_cast(double, (uint64_t)(e > 5 && e < 2047 ? 2 * 1023 + 6 - e : 1023) << 52);
}
__device__ __forceinline__ int whole(double x) { return (int)fmin(fmax(__builtin_rint(x), -127.0), 127.0); }

// Bits 0 .. 3 (NIBBLE 0) or 4 .. 7 of four bytes, codes, to four int8 centroids
// from the 16-byte table t: both halves of the table by the low three bits,
// then byte k of either by the fourth.
template <int NIBBLE>
__device__ __forceinline__ uint32_t four_centroids(uint32_t x, const uint32_t (&t)[4]) {
    const uint32_t sel = (NIBBLE ? x >> 4 : x) & 0x07070707u;
    const uint32_t low = __builtin_amdgcn_perm(t[1], t[0], sel), high = __builtin_amdgcn_perm(t[3], t[2], sel);
    return __builtin_amdgcn_perm(high, low, ((x >> (NIBBLE ? 5 : 1)) & 0x04040404u) | 0x03020100u);
}

constexpr int kSelWaves = 8;

struct ScoreLds {
    __attribute__((aligned(16))) double part[kSelWaves][256];
    __attribute__((aligned(16))) int8_t q[256];      // Q+, then -Q-
    __attribute__((aligned(16))) int8_t cent[16];
};

// x of lane c ^ m of a 16-lane row, m a power of two
__device__ __forceinline__ uint32_t sel_row_xor(uint32_t v, int m, int c) {
    if (m == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);             // quad_perm [1,0,3,2]
    if (m == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);             // quad_perm [2,3,0,1]
    if (m == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);            // row_ror:8
    const int up = __builtin_amdgcn_mov_dpp((int)v, 0x12C, 0xf, 0xf, true);                          // row_ror:12: lane c + 4
    const int dn = __builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true);                          // row_ror:4: lane c - 4
    return (uint32_t)(c & 4 ? dn : up);
}
__device__ __forceinline__ double sel_row_xor(double x, int m, int c) {
    const uint64_t v = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, ((uint64_t)sel_row_xor((uint32_t)(v >> 32), m, c) << 32) | sel_row_xor((uint32_t)v, m, c));
}

// A stage of the Hadamard sums over lanes l and l ^ HALF: the sum in the lower
// one, lower less upper in the other.
template <int HALF>
__device__ __forceinline__ double sel_stage(double x, int lane) {
    const uint64_t v = __builtin_bit_cast(uint64_t, x);
    uint64_t lower, upper;
    if constexpr (HALF == 16) {
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
        lower = ((uint64_t)hi[0] << 32) | lo[0];
        upper = ((uint64_t)hi[1] << 32) | lo[1];
    } else {
        const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
        lower = ((uint64_t)hi[0] << 32) | lo[0];
        upper = ((uint64_t)hi[1] << 32) | lo[1];
    }
    return __builtin_fma(lane & HALF ? -1.0 : 1.0, __builtin_bit_cast(double, upper), __builtin_bit_cast(double, lower));
}

// Q+ and -Q- of query (b, t)'s heads hk G .. + G - 1 and the centroids, as
// int8: a head a wave at a time, two dims a lane.  The constructor asks for the
// loads of head `first`.
struct WholeQuery {
    uint32_t raw, flip;
    float cent;
    __device__ __forceinline__ uint32_t head(const SelectArgs &a, int64_t b, int t, int hk, int h) const {
        return *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint16_t *>(a.q) +
                                                   ((b * a.Hq + hk * a.G + (h < a.G ? h : 0)) * a.T + t) * 128 + 2 * (threadIdx.x & 63));
    }
    __device__ __forceinline__ WholeQuery(const SelectArgs &a, int64_t b, int t, int hk, int first) {
        const int lane = threadIdx.x & 63;
        raw = head(a, b, t, hk, first);
        flip = 0u;
        if (a.sign_flip) flip = *reinterpret_cast<const uint16_t *>(a.sign_flip + 2 * lane);
        cent = (a.codebooks + (a.per_head ? hk * 16 : 0))[lane & 15];
    }
    // the wave's sums over heads first, first + stride, ..., N at a time (their
    // chains side by side): Q+, then -Q-
    template <int N>
    __device__ __forceinline__ void sums(const SelectArgs &a, double *part, int64_t b, int t, int hk, int first, int stride) const {
        const int lane = threadIdx.x & 63, c = lane & 15;
        double qp[2] = {0.0, 0.0}, qn[2] = {0.0, 0.0};
        for (int h0 = first; h0 < a.G; h0 += N * stride) {
            double x[2 * N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int h = h0 + k * stride;
                const uint32_t w = h == first ? raw : head(a, b, t, hk, h);
                const uint16_t u[2] = {(uint16_t)((w & 0xffffu) ^ ((flip & 0x80u) << 8)), (uint16_t)((w >> 16) ^ (flip & 0x8000u))};
#pragma unroll
                for (int j = 0; j < 2; ++j) x[2 * k + j] = h < a.G ? (double)(a.f16 ? f16_to_f32(u[j]) : bf16_to_f32(u[j])) : 0.0;
            }
            if (a.rotate) {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const double sum = x[2 * k] + x[2 * k + 1], less = x[2 * k] - x[2 * k + 1];
                    x[2 * k] = sum;
                    x[2 * k + 1] = less;
                }
#pragma unroll
                for (int m = 1; m < 16; m <<= 1)
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) x[j] = __builtin_fma(c & m ? -1.0 : 1.0, x[j], sel_row_xor(x[j], m, c));
#pragma unroll
                for (int j = 0; j < 2 * N; ++j) x[j] = sel_stage<32>(sel_stage<16>(x[j], lane), lane);
            }
#pragma unroll
            for (int j = 0; j < 2 * N; ++j) {
                qp[j & 1] += fmax(x[j], 0.0);
                qn[j & 1] += fmin(x[j], 0.0);
            }
        }
        *reinterpret_cast<double2 *>(part + 2 * lane) = make_double2(qp[0], qp[1]);
        *reinterpret_cast<double2 *>(part + 128 + 2 * lane) = make_double2(qn[0], qn[1]);
    }
    __device__ __forceinline__ int8_t centroid() const {          // lane l: of code l % 16
        const int c = threadIdx.x & 15;
        float cm = fabsf(cent);
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) cm = fmaxf(cm, __uint_as_float(sel_row_xor(__float_as_uint(cm), m, c)));
        return (int8_t)whole((double)cent * whole_scale((double)cm));
    }
    // v[k]: place 64 k + lane of the summed sums; each wave finds the largest, and stores the places that `mask` names
    __device__ __forceinline__ static void store(const double (&v)[4], int8_t *q, uint32_t mask) {
        const int lane = threadIdx.x & 63, c = lane & 15;
        double m = fmax(fmax(fabs(v[0]), fabs(v[1])), fmax(fabs(v[2]), fabs(v[3])));
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) m = fmax(m, sel_row_xor(m, k, c));
#pragma unroll
        for (int k = 16; k < 64; k <<= 1) m = fmax(m, __shfl_xor(m, k));
        const double scale = whole_scale(m);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((mask >> k) & 1u) q[64 * k + lane] = (int8_t)whole(v[k] * scale);
    }
    // one kv head by the whole block
    __device__ __forceinline__ void form(const SelectArgs &a, ScoreLds &sm, int64_t b, int t, int hk) const {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int waves = a.G < kSelWaves ? a.G : kSelWaves;
        if (wave < waves) sums<1>(a, sm.part[wave], b, t, hk, wave, kSelWaves);
        const int8_t ci = centroid();
        if (tid < 16) sm.cent[tid] = ci;
        __syncthreads();
        double v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = 0.0;
            for (int w = 0; w < waves; ++w) v[k] += sm.part[w][64 * k + lane];
        }
        if (wave < 4) store(v, sm.q, 1u << wave);
        __syncthreads();
    }
};

// The score of the block whose bounds the eight lanes of `lane`'s group hold 16
// dims each of, as an unsigned key that orders as it does.  A page outside the
// pool is selected first, so that its rows come out NaN.
__device__ __forceinline__ uint32_t block_key(const uint4 &w, int32_t id, int64_t n_pages, const uint32_t (&qp)[4],
                                              const uint32_t (&qn)[4], const uint32_t (&tab)[4], int lane) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    int s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s = __builtin_amdgcn_sdot4((int)four_centroids<1>(x[j], tab), (int)qp[j], s, false);
        s = __builtin_amdgcn_sdot4((int)four_centroids<0>(x[j], tab), (int)qn[j], s, false);
    }
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) s += (int)sel_row_xor((uint32_t)s, m, lane & 15);
    s += __builtin_amdgcn_mov_dpp(s, 0x141, 0xf, 0xf, true);      // row_half_mirror: the other quad's sum
    return id >= 0 && id < n_pages ? (uint32_t)s ^ 0x80000000u : 0xffffffffu;
}

// Scores of blocks from .. to - 1 by the block's eight waves, put(block, score
// as an unsigned key that orders as it does): eight lanes a block, 16 dims
// each; a wave has 32 blocks' bounds in flight (64 spill at two thread blocks a
// CU).  Bound by the chain of query, page table, bounds and digits: 32 x 8 rows
// of 512 blocks 10.7 us, choice included (16.8 MB of bounds: 3 us at a copy's
// rate; a launch for the scores and one for the choice 20); 312 rows of up to
// 939 blocks 15.4 us, 18 with one thread block a CU.
template <typename Put>
__device__ __forceinline__ void score_blocks(const SelectArgs &a, const WholeQuery &wq, ScoreLds &sm, int64_t b, int t, int hk, int from,
                                             int to, Put &&put) {
    constexpr int U = 4;                                          // loads in flight
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 7;
    const int32_t *pt = a.page_table + b * a.max_pages;
    int32_t id[U];
    uint4 w[U];
    auto ids = [&](int p0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + 8 * u + (lane >> 3);
            id[u] = p < to ? pt[p] : 0;
        }
    };
    auto bounds = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ok = id[u] >= 0 && id[u] < a.n_pages;
            w[u] = *reinterpret_cast<const uint4 *>(a.bounds + ((uint64_t)((uint32_t)(ok ? id[u] : 0) * (uint32_t)a.Hkv + (uint32_t)hk) * 128 + 16u * (uint32_t)c));
        }
    };
    int p0 = from + 8 * U * wave;
    ids(p0);
    bounds();
    wq.form(a, sm, b, t, hk);
    uint32_t qp[4], qn[4], tab[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        qp[j] = reinterpret_cast<const uint32_t *>(sm.q)[4 * c + j];
        qn[j] = reinterpret_cast<const uint32_t *>(sm.q)[32 + 4 * c + j];
        tab[j] = reinterpret_cast<const uint32_t *>(sm.cent)[j];
    }
    for (; p0 < to; p0 += 8 * U * kSelWaves) {
        uint32_t s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = block_key(w[u], id[u], a.n_pages, qp, qn, tab, lane);
        const int at = p0;
        ids(p0 + 8 * U * kSelWaves);
        if (p0 + 8 * U * kSelWaves < to) bounds();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = at + 8 * u + (lane >> 3);
            if (c == 0 && p < to) put(p, s[u]);
        }
    }
}

// ── selection ───────────────────────────────────────────────────────────
//
// One block per (b, t, hk): the score that the last of `need` blocks has, by
// digits of eight bits from the top of the scores' range (a histogram in LDS
// per digit), then the blocks above it and the first ones equal to it in
// ascending order.  SCORED: the scores are there already, by
// block_score_kernel; 64 rows of 8192 blocks 11.8 us, three digits of which
// each takes a pass over the keys in registers and three barriers.
constexpr int kPickLds = 14336;          // scores held in LDS (two blocks a CU); more are read again for every digit

// The key (at most `range`) that the `need`-th largest has, and of the equal
// ones how many are needed (in `need`).  each(shift, at, count) calls count(x)
// for every key x whose bits from `shift` up are `at`.
template <typename Each>
__device__ __forceinline__ uint32_t find_digits(uint32_t range, uint32_t &need, uint32_t *hist, uint32_t *sh, Each &&each) {
    const int tid = threadIdx.x, lane = tid & 63;
    int shift = range ? 32 - __builtin_clz(range) : 0;
    uint32_t prefix = 0u;
    while (shift > 0) {
        const int low = shift > 8 ? shift - 8 : 0, width = shift - low;
        if (tid < 256) hist[tid] = 0u;
        __syncthreads();
        each(shift, prefix, [&](uint32_t x) { atomicAdd(&hist[(x >> low) & ((1u << width) - 1u)], 1u); });
        __syncthreads();
        if (tid < 64) {
            // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
            const uint4 h4 = *reinterpret_cast<const uint4 *>(&hist[252 - 4 * lane]);
            const uint32_t c[4] = {h4.w, h4.z, h4.y, h4.x};
            const uint32_t sum = (c[0] + c[1]) + (c[2] + c[3]);
            uint32_t incl = sum;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t up = __shfl_up(incl, m);
                incl += lane >= m ? up : 0u;
            }
            uint32_t above = incl - sum;
            if (above < need && need <= incl) {                   // one lane
                bool found = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!found && need <= above + c[j]) {
                        sh[0] = (prefix << width) | (uint32_t)(255 - 4 * lane - j);
                        sh[1] = need - above;
                        found = true;
                    }
                    above += c[j];
                }
            }
        }
        __syncthreads();                                         // hist may be cleared again
        prefix = sh[0];
        need = sh[1];
        shift = low;
    }
    return prefix;
}

// The `need` largest of n <= R 512 keys (in LDS, from kmin to kmax), the first
// of equal ones: their places, counted from `first`, ascending.  Thread tid
// holds keys tid, tid + 512, ...
template <int R>
__device__ __forceinline__ void pick_held(uint32_t *keys, int n, uint32_t kmin, uint32_t kmax, uint32_t need, uint32_t *hist,
                                          uint32_t *sh, int first, int32_t *out) {
    constexpr int kThreads = 64 * kSelWaves;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t x[R];
#pragma unroll
    for (int j = 0; j < R; ++j) x[j] = j * kThreads + tid < n ? keys[j * kThreads + tid] - kmin : 0u;
    const uint32_t prefix = find_digits(kmax - kmin, need, hist, sh, [&](int shift, uint32_t at, auto &&count) {
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (j * kThreads + tid < n && (shift >= 32 || x[j] >> shift == at)) count(x[j]);
    });
    // counts of either kind by 64 consecutive keys, (j, wave)
    uint32_t *const cnt = keys;
    __syncthreads();                                             // keys are read
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const bool in = j * kThreads + tid < n;
        const uint64_t above = __builtin_amdgcn_ballot_w64(in && x[j] > prefix), equal = __builtin_amdgcn_ballot_w64(in && x[j] == prefix);
        if (lane == 0) cnt[j * kSelWaves + wave] = (uint32_t)__popcll(above) | ((uint32_t)__popcll(equal) << 16);
    }
    __syncthreads();
    // their exclusive sums, each wave for itself, two counts a lane (8192 of either kind at most: 16 bits hold them)
    const bool some = 2 * lane < R * kSelWaves;
    const uint2 two = *reinterpret_cast<const uint2 *>(&cnt[some ? 2 * lane : 0]);
    const uint32_t both = some ? two.x + two.y : 0u;
    uint32_t incl = both;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t up = __shfl_up(incl, m);
        incl += lane >= m ? up : 0u;
    }
    const uint32_t first_of = incl - both;
    const uint64_t before = ((uint64_t)1 << lane) - 1;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (j * kThreads >= n) break;                            // uniform
        const bool in = j * kThreads + tid < n;
        const uint64_t above = __builtin_amdgcn_ballot_w64(in && x[j] > prefix), equal = __builtin_amdgcn_ballot_w64(in && x[j] == prefix);
        const int item = j * kSelWaves + wave;
        const uint32_t base = (uint32_t)__builtin_amdgcn_readlane((int)first_of, item >> 1) +
                              (item & 1 ? (uint32_t)__builtin_amdgcn_readlane((int)two.x, item >> 1) : 0u);
        const uint32_t g = (base & 0xffffu) + (uint32_t)__popcll(above & before), e = (base >> 16) + (uint32_t)__popcll(equal & before);
        if (((above >> lane) & 1u) || (((equal >> lane) & 1u) && e < need)) out[g + (e < need ? e : need)] = first + j * kThreads + tid;
    }
}

// Scores where rows are fewer than CUs and long: the read of the bounds over
// the whole chip, `heads` kv heads (a divisor of 8, or 8) of a share of one
// query's blocks by a thread block, so that a wave's load is 8 / heads pages'
// neighbouring bounds, a KB.  8 x 8 rows of 8192 blocks (67 MB): 22 us, 3.0
// TB/s: 5 us of query, then some 90 vector instructions for eight bounds.
// Measured: two thread blocks a CU 21, one 24, four (two rounds) 27 us; eight
// loads in flight, which spill at two blocks, 22; query heads one after another
// instead of four side by side 27.
__global__ __launch_bounds__(64 * kSelWaves, 4) void block_score_kernel(SelectArgs a) {
    constexpr int U = 4;                                          // loads in flight
    __shared__ __attribute__((aligned(16))) int8_t qs[8][256];
    __shared__ __attribute__((aligned(16))) int8_t cs[8][16];
    __shared__ __attribute__((aligned(16))) double part[8][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 7;
    const int64_t b = blockIdx.z;
    const int sets = a.Hkv / a.heads, share = (int)(blockIdx.x / (unsigned)sets), h0 = ((int)blockIdx.x - share * sets) * a.heads;
    const int t = blockIdx.y;
    const int nb = (int)seen_blocks(a, b, t);
    const int from = a.first + share * a.per_block, last = nb - a.recent;
    if (nb <= a.top || from >= last) return;                     // block-uniform, before any barrier
    const int to = from + a.per_block < last ? from + a.per_block : last;
    const int32_t *pt = a.page_table + b * a.max_pages;
    const int per = 8 / a.heads, mine = (lane >> 3) / a.heads, hk = h0 + (lane >> 3) - mine * a.heads;     // pages a load; this lane's
    int32_t id[U];
    uint4 w[U];
    auto ids = [&](int p0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + per * u + mine;
            id[u] = p < to ? pt[p] : 0;
        }
    };
    auto bounds = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ok = id[u] >= 0 && id[u] < a.n_pages;
            w[u] = *reinterpret_cast<const uint4 *>(a.bounds + ((uint64_t)((uint32_t)(ok ? id[u] : 0) * (uint32_t)a.Hkv + (uint32_t)hk) * 128 + 16u * (uint32_t)c));
        }
    };
    const int step = per * U * kSelWaves;
    int p0 = from + per * U * wave;
    ids(p0);
    bounds();
    if (wave < a.heads) {                                        // a wave forms a head's query by itself
        const WholeQuery wq(a, b, t, h0 + wave, 0);
        wq.sums<4>(a, part[wave], b, t, h0 + wave, 0, 1);
        const int8_t ci = wq.centroid();
        if (lane < 16) cs[wave][lane] = ci;
        double v[4];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<volatile double *>(&part[wave][64 * k + lane]);
        WholeQuery::store(v, qs[wave], 15u);
    }
    __syncthreads();
    uint32_t qp[4], qn[4], tab[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        qp[j] = reinterpret_cast<const uint32_t *>(qs[hk - h0])[4 * c + j];
        qn[j] = reinterpret_cast<const uint32_t *>(qs[hk - h0])[32 + 4 * c + j];
        tab[j] = reinterpret_cast<const uint32_t *>(cs[hk - h0])[j];
    }
    uint32_t *out = reinterpret_cast<uint32_t *>(a.scores) + ((b * a.T + t) * a.Hkv + hk) * a.max_pages;
    for (; p0 < to; p0 += step) {
        uint32_t s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = block_key(w[u], id[u], a.n_pages, qp, qn, tab, lane);
        const int at = p0;
        ids(p0 + step);
        if (p0 + step < to) bounds();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = at + per * u + mine;
            if (c == 0 && p < to) out[p] = s[u];
        }
    }
}

template <bool SCORED>
__global__ __launch_bounds__(64 * kSelWaves, 4) void block_select_kernel(SelectArgs a) {
    constexpr int kThreads = 64 * kSelWaves;
    __shared__ uint32_t keys[kPickLds];
    __shared__ ScoreLds sm;
    __shared__ uint32_t hist[256];
    __shared__ uint32_t wred[2][kSelWaves];
    __shared__ uint32_t sh[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hk = blockIdx.x, t = blockIdx.y;
    const int64_t b = blockIdx.z, row = (b * a.T + t) * a.Hkv + hk;
    const WholeQuery wq(a, b, t, hk, (int)(threadIdx.x >> 6));
    const int64_t nb = seen_blocks(a, b, t);
    int32_t *out = a.blocks + ((b * a.Hkv + hk) * a.T + t) * a.top;
    if (nb <= a.top) {
        for (int i = tid; i < a.top; i += kThreads) out[i] = i < nb ? i : -1;
        return;
    }
    for (int i = tid; i < a.first + a.recent; i += kThreads)
        out[i < a.first ? i : a.top - a.recent + (i - a.first)] = (int32_t)(i < a.first ? i : nb - a.recent + (i - a.first));
    uint32_t need = (uint32_t)(a.top - a.first - a.recent);
    if (need == 0) return;                                       // uniform
    const int n = (int)(nb - a.first - a.recent);                // > need
    uint32_t *const src = reinterpret_cast<uint32_t *>(a.scores) + row * a.max_pages + a.first;
    const bool held = n <= kPickLds;
    uint32_t kmin = 0xffffffffu, kmax = 0u;
    if constexpr (SCORED) {
        for (int i0 = tid; i0 < n; i0 += 8 * kThreads) {          // eight loads in flight
            uint32_t k[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) k[j] = src[i0 + j * kThreads < n ? i0 + j * kThreads : i0];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (held && i0 + j * kThreads < n) keys[i0 + j * kThreads] = k[j];
                kmin = k[j] < kmin ? k[j] : kmin;
                kmax = k[j] > kmax ? k[j] : kmax;
            }
        }
    } else {
        score_blocks(a, wq, sm, b, t, hk, a.first, (int)nb - a.recent, [&](int p, uint32_t k) {
            if (held) keys[p - a.first] = k;
            else src[p - a.first] = k;
            kmin = k < kmin ? k : kmin;
            kmax = k > kmax ? k : kmax;
        });
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint32_t lo = __shfl_xor(kmin, m), hi = __shfl_xor(kmax, m);
        kmin = lo < kmin ? lo : kmin;
        kmax = hi > kmax ? hi : kmax;
    }
    if (lane == 0) {
        wred[0][wave] = kmin;
        wred[1][wave] = kmax;
    }
    __syncthreads();                                             // the keys too, in LDS or (block-wide) in memory
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
        kmin = wred[0][w] < kmin ? wred[0][w] : kmin;
        kmax = wred[1][w] > kmax ? wred[1][w] : kmax;
    }
    if (n <= 2 * kThreads) return pick_held<2>(keys, n, kmin, kmax, need, hist, sh, a.first, out + a.first);
    if (n <= 16 * kThreads) return pick_held<16>(keys, n, kmin, kmax, need, hist, sh, a.first, out + a.first);
    auto key = [&](int i) { return (held ? keys[i] : src[i]) - kmin; };
    const uint32_t prefix = find_digits(kmax - kmin, need, hist, sh, [&](int shift, uint32_t at, auto &&count) {
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t x = key(i);
            if (shift >= 32 || x >> shift == at) count(x);
        }
    });
    // ── the blocks above `prefix`, and the first `need` equal to it ──
    // each wave takes a share of consecutive blocks, 64 at a time: its count of
    // either kind first, then the places
    const int share = ((n + kSelWaves - 1) / kSelWaves + 63) & ~63, w0 = wave * share, w1 = w0 + share < n ? w0 + share : n;
    auto kinds = [&](int i0, uint64_t &above, uint64_t &equal) {
        const int i = i0 + lane;
        const uint32_t x = i < w1 ? key(i) : 0u;
        above = __builtin_amdgcn_ballot_w64(i < w1 && x > prefix);
        equal = __builtin_amdgcn_ballot_w64(i < w1 && x == prefix);
    };
    uint32_t pg = 0u, pe = 0u;
    for (int i0 = w0; i0 < w1; i0 += 64) {
        uint64_t above, equal;
        kinds(i0, above, equal);
        pg += (uint32_t)__popcll(above);
        pe += (uint32_t)__popcll(equal);
    }
    __syncthreads();                                             // wred is read
    if (lane == 0) {
        wred[0][wave] = pg;
        wred[1][wave] = pe;
    }
    __syncthreads();
    pg = pe = 0u;
    for (int w = 0; w < wave; ++w) {
        pg += wred[0][w];
        pe += wred[1][w];
    }
    const uint64_t before = ((uint64_t)1 << lane) - 1;
    for (int i0 = w0; i0 < w1; i0 += 64) {
        uint64_t above, equal;
        kinds(i0, above, equal);
        const uint32_t g = pg + (uint32_t)__popcll(above & before), e = pe + (uint32_t)__popcll(equal & before);
        if (((above >> lane) & 1u) || (((equal >> lane) & 1u) && e < need)) out[a.first + g + (e < need ? e : need)] = a.first + i0 + lane;
        pg += (uint32_t)__popcll(above);
        pe += (uint32_t)__popcll(equal);
    }
}

// ── accepted drafted tokens ─────────────────────────────────────────────

struct KeepArgs {
    uint8_t *k_nib, *k_qjl, *v_nib;
    float *k_norms;
    const int32_t *page_table, *positions, *kept;
    int64_t max_pages, n_pages;
    int Hkv, page_shift, K;
};

// One block per (head, sequence): token positions + kept[j] goes to positions
// + j.  All rows are read before any is written, so the order of `kept` does
// not matter.  Four threads a token, 16 code bytes of K and V each.  Bound by
// latency: 4 to 64 tokens of 8 to 64 sequences 3.2 us, then the bounds' launch.
__global__ __launch_bounds__(256) void cache_keep_kernel(KeepArgs a) {
    const int hk = blockIdx.x;
    const int64_t b = blockIdx.y;
    const int j = threadIdx.x >> 2, c = threadIdx.x & 3;
    const int64_t base = a.positions[b], cap = a.max_pages << a.page_shift;
    auto row = [&](int64_t pos) -> int64_t {
        if (pos < 0 || pos >= cap) return -1;
        const int32_t id = a.page_table[b * a.max_pages + (pos >> a.page_shift)];
        if (id < 0 || id >= a.n_pages) return -1;
        return (((int64_t)id * a.Hkv + hk) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
    };
    int64_t from = -1, to = -1;
    if (j < a.K && base >= 0) {
        const int32_t k = a.kept[b * a.K + j];
        if (k >= 0 && k < 64) {
            from = row(base + k);
            to = row(base + j);
        }
    }
    const bool move = from >= 0 && to >= 0;
    uint4 k4 = make_uint4(0u, 0u, 0u, 0u), v4 = k4;
    uint2 s2 = make_uint2(0u, 0u);
    float nr = 0.0f;
    if (move) {
        k4 = reinterpret_cast<const uint4 *>(a.k_nib + from * 64)[c];
        v4 = reinterpret_cast<const uint4 *>(a.v_nib + from * 64)[c];
        if (c == 0) {
            s2 = *reinterpret_cast<const uint2 *>(a.k_qjl + from * 8);
            nr = a.k_norms[from];
        }
    }
    __syncthreads();                     // waits for the reads of every wave
    if (move) {
        reinterpret_cast<uint4 *>(a.k_nib + to * 64)[c] = k4;
        reinterpret_cast<uint4 *>(a.v_nib + to * 64)[c] = v4;
        if (c == 0) {
            *reinterpret_cast<uint2 *>(a.k_qjl + to * 8) = s2;
            a.k_norms[to] = nr;
        }
    }
}

}  // namespace omni

using namespace omni;

extern "C" int omni_block_bounds(const uint8_t *k_nib, uint8_t *bounds, int64_t n_pages, int Hkv, int page_size,
                                 const int32_t *page_table, int64_t max_pages, const int32_t *start, const int32_t *end,
                                 int64_t count, int64_t B, void *stream) {
    int shift;
    OMNI_TRY(check_pool("omni_block_bounds", n_pages, Hkv, page_size, max_pages, shift));
    OMNI_CHECK_ARG(B >= 0 && B <= 65535 && count >= 0, "omni_block_bounds: need 0 <= B <= 65535 and count >= 0");
    if (B == 0 || (end == nullptr && count == 0)) return OMNI_OK;
    OMNI_CHECK_ARG(k_nib && bounds && page_table && start, "omni_block_bounds: NULL pointer");
    // pages that `count` tokens can touch (2^32 reach any table's end from any start)
    if (count > (int64_t(1) << 32)) count = int64_t(1) << 32;
    int64_t pages = end ? max_pages : (count + page_size - 2) / page_size + 1;
    if (pages > max_pages) pages = max_pages;
    BoundsArgs a{k_nib, bounds, page_table, start, end, nullptr, max_pages, n_pages, count, 0, Hkv, shift};
    // a grid of 2^32 threads and more would be cut to its low 32 bits without an error
    constexpr int64_t kMost = 1 << 20;
    for (; a.page0 < pages; a.page0 += kMost) {
        const int64_t n = pages - a.page0 < kMost ? pages - a.page0 : kMost;
        hipLaunchKernelGGL(block_bounds_kernel, dim3((unsigned)n, (unsigned)B), dim3(256), 0, as_stream(stream), a);
        OMNI_CHECK_LAUNCH("block_bounds_kernel");
    }
    return OMNI_OK;
}

// One launch where a row's blocks are few or the rows fill the chip (32 x 8
// rows of 512 blocks 10.7 us, 20 in two); else the scores over the whole chip
// first (8 x 8 rows of 8192 blocks 33 us, 44 with one kv head a thread block).
static bool score_first(int64_t rows, int64_t max_pages) { return max_pages > 1024 && 2 * rows <= device_cus(); }

extern "C" size_t omni_block_select_workspace_size(int64_t B, int Hkv, int64_t T, int64_t max_pages, int top) {
    if (B <= 0 || B > 65535 || Hkv <= 0 || Hkv > 65535 || T <= 0 || T > 64 || max_pages <= top || max_pages > (1 << 26)) return 0;
    if (max_pages <= kPickLds && !score_first(B * Hkv * T, max_pages)) return 0;      // a row's scores stay in LDS
    return (size_t)B * Hkv * T * max_pages * 4;
}

extern "C" int omni_block_select(const void *q, int q_dtype, const uint8_t *bounds, int64_t n_pages, int page_size,
                                 const int32_t *page_table, int64_t max_pages, const int32_t *seq_lens,
                                 const float *codebooks, int per_head_codebook, int64_t B, int Hq, int Hkv, int64_t T,
                                 int head_dim, int top, int first, int recent, int rotate_q, const int8_t *sign_flip,
                                 int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream) {
    int shift;
    OMNI_CHECK_ARG(q_dtype == OMNI_F16 || q_dtype == OMNI_BF16, "omni_block_select: q must be float16 or bfloat16");
    OMNI_CHECK_ARG(head_dim == 128, "omni_block_select: head_dim must be 128, got %d", head_dim);
    OMNI_CHECK_ARG(B >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0,
                   "omni_block_select: need B >= 0 and n_heads a multiple of n_kv_heads");
    OMNI_CHECK_ARG(T >= 1 && T <= 64 && B <= 65535 / T && Hkv <= 65535, "omni_block_select: 1 to 64 query tokens, B * T and n_kv_heads at most 65535");
    OMNI_CHECK_ARG(Hq / Hkv <= 1024, "omni_block_select: at most 1024 query heads per kv head");
    OMNI_TRY(check_pool("omni_block_select", n_pages, Hkv, page_size, max_pages, shift));
    OMNI_CHECK_ARG(first >= 0 && recent >= 1 && first <= top - recent, "omni_block_select: need first >= 0, recent >= 1 and first + recent <= top");
    OMNI_CHECK_ARG(top <= (1 << 30) / page_size, "omni_block_select: top must be at most 2^30 / page_size, got %d", top);
    if (B == 0) return OMNI_OK;
    OMNI_CHECK_ARG(q && bounds && page_table && seq_lens && codebooks && blocks, "omni_block_select: NULL pointer");
    const size_t ws = omni_block_select_workspace_size(B, Hkv, T, max_pages, top);
    if (ws > workspace_bytes || (ws && !workspace)) {
        set_error("omni_block_select: workspace of %zu bytes needed, %zu given", ws, workspace_bytes);
        return OMNI_EWORKSPACE;
    }
    SelectArgs a{q, bounds, page_table, seq_lens, codebooks, rotate_q ? sign_flip : nullptr, (int32_t *)workspace, blocks,
                 max_pages, n_pages, shift, per_head_codebook, Hq, Hkv, Hq / Hkv, (int)T, top, first, recent, rotate_q,
                 q_dtype == OMNI_F16, 0, 1};
    const int64_t rows = B * T * Hkv;
    const int64_t cus = device_cus();
    a.heads = Hkv % 8 == 0 ? 8 : 8 % Hkv == 0 ? Hkv : 1;
    if (max_pages > top && score_first(rows, max_pages)) {
        // about two thread blocks a CU, whole rounds of their waves
        const int64_t round = 8 / a.heads * 4 * kSelWaves;
        int64_t per = max_pages * (rows / a.heads) / (2 * cus) / round * round;
        per = per < round ? round : per;
        a.per_block = (int)per;
        const unsigned shares = (unsigned)((max_pages + per - 1) / per);
        hipLaunchKernelGGL(block_score_kernel, dim3(shares * (unsigned)(Hkv / a.heads), (unsigned)T, (unsigned)B), dim3(64 * kSelWaves),
                           0, as_stream(stream), a);
        OMNI_CHECK_LAUNCH("block_score_kernel");
        hipLaunchKernelGGL(block_select_kernel<true>, dim3((unsigned)Hkv, (unsigned)T, (unsigned)B), dim3(64 * kSelWaves), 0, as_stream(stream), a);
    } else {
        hipLaunchKernelGGL(block_select_kernel<false>, dim3((unsigned)Hkv, (unsigned)T, (unsigned)B), dim3(64 * kSelWaves), 0, as_stream(stream), a);
    }
    OMNI_CHECK_LAUNCH("block_select_kernel");
    return OMNI_OK;
}

extern "C" int omni_cache_keep(uint8_t *k_nib, uint8_t *k_qjl, float *k_norms, uint8_t *v_nib, uint8_t *bounds,
                               int64_t n_pages, int Hkv, int page_size, const int32_t *page_table, int64_t max_pages,
                               const int32_t *positions, const int32_t *kept, int64_t B, int K, void *stream) {
    int shift;
    OMNI_TRY(check_pool("omni_cache_keep", n_pages, Hkv, page_size, max_pages, shift));
    OMNI_CHECK_ARG(B >= 0 && B <= 65535 && K >= 0 && K <= 64, "omni_cache_keep: need 0 <= B <= 65535 and at most 64 kept tokens, got %d", K);
    if (B == 0 || K == 0) return OMNI_OK;
    OMNI_CHECK_ARG(k_nib && k_qjl && k_norms && v_nib && page_table && positions && kept, "omni_cache_keep: NULL pointer");
    const KeepArgs a{k_nib, k_qjl, v_nib, k_norms, page_table, positions, kept, max_pages, n_pages, Hkv, shift, K};
    hipLaunchKernelGGL(cache_keep_kernel, dim3((unsigned)Hkv, (unsigned)B), dim3(256), 0, as_stream(stream), a);
    OMNI_CHECK_LAUNCH("cache_keep_kernel");
    if (bounds) {
        int64_t pages = (K + 1 + page_size - 2) / page_size + 1;      // K tokens and the one before them
        if (pages > max_pages) pages = max_pages;
        const BoundsArgs ba{k_nib, bounds, page_table, positions, nullptr, kept, max_pages, n_pages, K, 0, Hkv, shift};
        hipLaunchKernelGGL(block_bounds_kernel, dim3((unsigned)pages, (unsigned)B), dim3(256), 0, as_stream(stream), ba);
        OMNI_CHECK_LAUNCH("block_bounds_kernel");
    }
    return OMNI_OK;
}
