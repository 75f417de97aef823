// Attention of 16-bit queries over lists of pages of the INT4 + QJL cache on
// gfx950: a tree of drafted tokens behind a cached sequence (omni_attn_tree)
// and the blocks (pages) that a score selected for each query
// (omni_attn_blocks).  head_dim 128.
//
//   k^_s = c[code_s] + n_s sqrt(2/pi)/128 (b_s G)      v^_s = c[vcode_s]
//   o_r  = sum_s p_rs v^_s / sum_s p_rs,   p_rs = exp(scale q_r . k^_s) over the visible s
//
// One block takes one list (a sequence, or the blocks of one query) of one kv
// head, a split of its 32-token tiles, and 16 NR query rows (the group's heads
// of one or more query tokens); its waves take the tiles in turn, each with
// its own running maximum and sum, and are merged at the end.  All products on
// v_mfma_f32_16x16x32_f16, tokens on M for the scores and dims on M for P V:
//   K pass    A = centroids of 16 tokens, looked up a code byte at a time in
//             an LDS table (64 KB: a private column per lane, so a byte and the
//             lane make the address with one v_perm and no bank is met twice);
//             B = the query rows.  Lane (n, g) reads bytes 16 g .. + 15 of
//             token n, so k-slot i of step s is dim 32 g + 8 s + i on both sides.
//   QJL pass  A = the signs as +-1, B = sqrt(2/pi)/128 G q as it leaves the
//             product G q (projections 16 cb + 4 g + i in lane (n, g)): the
//             sign nibbles are picked in that order.
//   P V       A = centroids again, two tokens' codes of one dim interleaved
//             into one table byte; B = P as it leaves the scores.
// Numbers: q rows times a power of two (largest in [2^14, 2^15)) and the head's
// centroids times one (largest in [2^9, 2^10)) are rounded to fp16.  bf16
// queries that the call does not rotate lose nothing; rotated ones and the
// centroids 2^-12 of themselves, P another 2^-12 (the same rounded P in
// numerator and denominator): below the 2^-9 of the bf16 output.  fp16 queries
// (HL) keep a second fp16 term of q and of the centroids in both products (22
// bits), which leaves P's 2^-12 against the output's 2^-12.  Scores, maxima,
// sums and accumulators are fp32.
#include <math.h>

#include <new>

#include "omni_common.h"

namespace omni {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

struct PageAttnArgs {
    const void *q;
    void *out;
    float *ws;                   // partials of the splits: [unit][split][row][kPartRow]
    const uint8_t *k_nib, *k_qjl, *v_nib;
    const float *k_norms, *codebooks;
    const uint32_t *g_bits;
    const int8_t *sign_flip;     // NULL: no flips
    const int32_t *page_table, *seq_lens;
    const int32_t *n_draft;      // tree: drafted tokens of each sequence (NULL: T)
    const int64_t *tree;         // tree: bit j of tree[b * tree_stride + t]: row t sees drafted token j
    const int32_t *blocks;       // blocks: (B, Hkv, T, top) block numbers, others are skipped
    int64_t max_pages, n_pages, tree_stride, units;
    int page_shift, per_head, Hq, Hkv, G, T, rows, chunks, splits, top, rotate;
    float qscale;                // scale log2 e
    float alpha, wht_scale;      // sqrt(2/pi) / 128, 1 / sqrt(128) as fp32
};

constexpr int kPgTile = 32;
constexpr int kPartRow = 128 + 4;            // floats of a split's row: O, then m and l
constexpr int kLutBytes = 65536;             // [byte][256 B]: 64 columns of 4 B (HL: 32 of 8 B)
constexpr int kSignOff = kLutBytes;          // [nibble][256 B]: 32 columns of four +-1.0 halves
constexpr int kQimgOff = kSignOff + 4096;

template <int NR, int NW, bool QJL, bool HL>
struct PgLds {
    static constexpr int kSteps = QJL ? 6 : 4;                               // B operands of a row group: q, then G q
    static constexpr int kQimg = NR * kSteps * (HL ? 2 : 1) * 1024;
    static constexpr int kCsc = kQimgOff + kQimg;                            // per row: score scale
    static constexpr int kBad = kCsc + NR * 16 * 4;                          // per wave: met a page outside the pool
    static constexpr int kUse = kBad + NW * 4;
    static constexpr int kSlabs = NW * 16 * kPartRow * 4;                    // epilogue: the waves' O of one row group
    static constexpr int kMl = kSlabs;                                       // then their m and l
    static constexpr int kTotal = kUse > kMl + NW * 32 * 4 + NW * 4 ? kUse : kMl + NW * 32 * 4 + NW * 4;
};

__device__ __forceinline__ uint32_t pg_pack(float x, float y) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){x, y}, half2_t));
}
__device__ __forceinline__ float pg_h_lo(uint32_t w) { return f16_to_f32((uint16_t)(w & 0xffffu)); }
__device__ __forceinline__ float pg_h_hi(uint32_t w) { return f16_to_f32((uint16_t)(w >> 16)); }
__device__ __forceinline__ half8_t pg_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8_t, make_uint4(a, b, c, d));
}
__device__ __forceinline__ float4_t pg_mfma(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float pg_max(float a, float b) {           // as fmaxf, without quieting its operands first
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float pg_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float pg_max_groups(float m) {
    auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = pg_max(__uint_as_float(t[0]), __uint_as_float(t[1]));
    auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return pg_max(__uint_as_float(u[0]), __uint_as_float(u[1]));
}
__device__ __forceinline__ float pg_sum_groups(float v) {
    auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(u[0]) + __uint_as_float(u[1]);
}

// The list that a unit (b, t, hk) or (b, hk) reads: `seen` tokens of sequence
// b, in tree calls the first `base` of them by every row.  Tiles are of the
// list's slots: positions in a sequence, or `top` blocks one after another.
struct PgList {
    int64_t b;
    int t, hk, nd;
    int64_t seen, base, tiles;
    bool bad;                    // a length that the table cannot hold, or more drafted tokens than there are
};
template <bool BLOCKS>
__device__ __forceinline__ PgList pg_list(const PageAttnArgs &a, int64_t unit) {
    PgList l;
    l.hk = (int)(unit % a.Hkv);
    const int64_t bt = unit / a.Hkv;
    l.b = BLOCKS ? bt / a.T : bt;
    l.t = BLOCKS ? (int)(bt - l.b * a.T) : 0;
    const int64_t len = a.seq_lens[l.b];
    l.bad = len < 0 || len > (a.max_pages << a.page_shift);
    if constexpr (BLOCKS) {
        l.nd = a.T;
        l.seen = l.bad ? 0 : len - a.T + l.t + 1 > 0 ? len - a.T + l.t + 1 : 0;
        l.base = 0;
        l.tiles = (((int64_t)a.top << (a.page_shift - 4)) + 1) >> 1;
    } else {
        l.nd = a.n_draft ? a.n_draft[l.b] : a.T;
        l.bad = l.bad || l.nd < 0 || l.nd > a.T || l.nd > len;
        l.seen = l.bad ? 0 : len;
        l.base = l.seen - l.nd;
        l.tiles = (l.seen + kPgTile - 1) / kPgTile;
    }
    return l;
}
// tiles of a split: even shares, so the splits of a short list are short
__device__ __forceinline__ int64_t pg_share(int64_t tiles, int splits) { return (tiles + splits - 1) / splits; }

struct PgTile {
    uint4 k[2];        // code bytes 16 g .. + 15 of token n of half u
    uint2 sg[2];       // its sign bytes
    float4 nr[2];      // norms of tokens 4 g .. + 3
    uint32_t v[8];     // code bytes 4 n .. + 3 of tokens 16 (i / 4) + 4 g + i % 4
    int nv[2];         // tokens of each half that the list holds (wave-uniform)
};

template <int NR, int NW, bool QJL, bool HL, bool BLOCKS>
__global__ __launch_bounds__(64 * NW) void page_attn_kernel(PageAttnArgs a) {
    using L = PgLds<NR, NW, QJL, HL>;
    constexpr bool F16 = HL;
    constexpr bool QREG = NR * (HL ? 2 : 1) <= 2;   // query operands in registers (else read from LDS in each tile)
    __shared__ __attribute__((aligned(16))) unsigned char smem[L::kTotal];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;

    // block -> (unit, split, row chunk): the chunks of one (unit, split) eight
    // blocks apart, so that they run on one XCD and share its L2
    const int64_t us_all = a.units * a.splits;
    const int64_t grp = blockIdx.x / (8 * a.chunks);
    const int rest = (int)(blockIdx.x - grp * 8 * a.chunks);
    const int64_t us = grp * 8 + (rest & 7);
    const int chunk = rest >> 3;
    if (us >= us_all) return;
    const int64_t unit = us / a.splits;
    const int split = (int)(us - unit * a.splits);
    const PgList li = pg_list<BLOCKS>(a, unit);
    const int hk = li.hk;
    const int64_t share = pg_share(li.tiles, a.splits);
    const int64_t t_begin = split * share, t_end = t_begin + share < li.tiles ? t_begin + share : li.tiles;
    if (split > 0 && t_begin >= li.tiles) return;           // the merge counts the splits that have tiles

    // ── the wave's tiles: pool rows of their halves, one tile a lane ──
    const int cnt = t_end - t_begin > wave ? (int)((t_end - t_begin - wave + NW - 1) / NW) : 0;
    uint32_t row0 = 0, row1 = 0, nvs = 0;
    bool page_bad = false;
    auto fetch = [&](int first) {
        uint32_t r[2], v[2];
        const int64_t tile = t_begin + wave + (int64_t)NW * (first + lane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t half = 2 * tile + u;
            int64_t pos = half << 4;                         // of its first token
            int64_t page = half >> (a.page_shift - 4);
            bool in = first + lane < cnt;
            if constexpr (BLOCKS) {
                const int64_t nb = (li.seen + (1 << a.page_shift) - 1) >> a.page_shift;
                in = in && page < a.top;
                const int64_t blk = in ? a.blocks[((li.b * a.Hkv + hk) * a.T + li.t) * a.top + page] : -1;
                in = in && blk >= 0 && blk < nb;
                pos = (blk << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
                page = blk;
            }
            const int64_t left = in ? li.seen - pos : 0;
            v[u] = left <= 0 ? 0u : left < 16 ? (uint32_t)left : 16u;
            const int32_t id = v[u] ? a.page_table[li.b * a.max_pages + page] : 0;
            const bool ok = id >= 0 && id < a.n_pages;
            page_bad = page_bad || !ok;
            r[u] = (((uint32_t)(ok ? id : 0) * (uint32_t)a.Hkv + (uint32_t)hk) << a.page_shift) +
                   (v[u] ? (uint32_t)(pos & ((1 << a.page_shift) - 1)) : 0u);
        }
        row0 = r[0];
        row1 = r[1];
        nvs = v[0] | (v[1] << 8);
    };
    fetch(0);
    auto load = [&](PgTile &R, int k) {
        if ((k & 63) == 0 && k > 0) fetch(k);
        const uint32_t r[2] = {(uint32_t)__builtin_amdgcn_readlane((int)row0, k & 63),
                               (uint32_t)__builtin_amdgcn_readlane((int)row1, k & 63)};
        const int v = __builtin_amdgcn_readlane((int)nvs, k & 63);
        R.nv[0] = v & 255;
        R.nv[1] = v >> 8;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            R.k[u] = *reinterpret_cast<const uint4 *>(a.k_nib + (uint64_t)r[u] * 64 + (uint32_t)(64 * n + 16 * g));
            if (QJL) {
                R.sg[u] = *reinterpret_cast<const uint2 *>(a.k_qjl + (uint64_t)r[u] * 8 + (uint32_t)(8 * n));
                R.nr[u] = *reinterpret_cast<const float4 *>(a.k_norms + (uint64_t)r[u] + (uint32_t)(4 * g));
            }
            const uint8_t *vp = a.v_nib + (uint64_t)r[u] * 64;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                R.v[4 * u + i] = *reinterpret_cast<const uint32_t *>(vp + (uint32_t)(64 * (4 * g + i) + 4 * n));
        }
    };
    PgTile R0, R1;
    if (cnt > 0) load(R0, 0);

    // ── tables ────────────────────────────────────────────────────────
    const float *cbp = a.codebooks + (a.per_head ? hk * 16 : 0);
    float cmax = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) cmax = fmaxf(cmax, fabsf(cbp[k]));
    int cexp = 0;
    if (cmax > 0.0f && cmax < INFINITY) frexpf(cmax, &cexp);
    cexp = cexp < -100 ? -100 : cexp;
    const float cmul = ldexpf(1.0f, 10 - cexp), cdiv = ldexpf(1.0f, cexp - 10);
    for (int m = tid; m < kLutBytes / 16; m += 64 * NW) {
        const int e = m >> 4;
        const float c0 = cbp[e & 15] * cmul, c1 = cbp[e >> 4] * cmul;
        const uint32_t hi = pg_pack(c0, c1);
        uint4 w = make_uint4(hi, hi, hi, hi);
        if (HL) w.y = w.w = pg_pack(c0 - pg_h_lo(hi), c1 - pg_h_hi(hi));
        *reinterpret_cast<uint4 *>(smem + 16 * m) = w;
    }
    if (QJL && tid < 512) {
        const uint32_t v = (uint32_t)tid >> 5;
        uint32_t w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            w[k] = (((v >> (2 * k)) & 1) ? 0x3C00u : 0xBC00u) | ((((v >> (2 * k + 1)) & 1) ? 0x3C00u : 0xBC00u) << 16);
        *reinterpret_cast<uint2 *>(smem + kSignOff + v * 256u + (tid & 31u) * 8u) = make_uint2(w[0], w[1]);
    }

    // ── query rows: wave w < NR turns row group w into MFMA operands ──
    uint4 *qimg = reinterpret_cast<uint4 *>(smem + kQimgOff);      // [rg][step][lane], HL: the remainders a plane on
    constexpr int kPlane = NR * L::kSteps * 64;
    float *csc_l = reinterpret_cast<float *>(smem + L::kCsc);
    if (wave < NR) {
        const int rho = (chunk * NR + wave) * 16 + n;
        const bool ok = rho < a.rows;
        const int rr = ok ? rho : 0;
        const int t = BLOCKS ? li.t : rr / a.G;
        const int hq = hk * a.G + (BLOCKS ? rr : rr - t * a.G);
        const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q) + ((li.b * a.Hq + hq) * a.T + t) * 128 + 32 * g;
        float x[4][8];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint4 w4 = reinterpret_cast<const uint4 *>(src)[s];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint16_t h = (uint16_t)((i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
                x[s][i] = ok ? (F16 ? f16_to_f32(h) : bf16_to_f32(h)) : 0.0f;
            }
        }
        if (a.rotate) {
            // the normalized WHT in stage order h = 1 .. 64; the row is not
            // rounded to q's type in between
            if (a.sign_flip) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const uint2 f = *reinterpret_cast<const uint2 *>(a.sign_flip + 32 * g + 8 * s);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        x[s][i] = __uint_as_float(__float_as_uint(x[s][i]) ^
                                                  (((i < 4 ? f.x >> (8 * i) : f.y >> (8 * i - 32)) & 0x80u) << 24));
                }
            }
#pragma unroll
            for (int h = 1; h < 8; h <<= 1)
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!(i & h)) {
                            const float u = x[s][i], l = x[s][i + h];
                            x[s][i] = u + l;
                            x[s][i + h] = u - l;
                        }
#pragma unroll
            for (int h = 1; h < 4; h <<= 1)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    if (!(s & h))
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float u = x[s][i], l = x[s + h][i];
                            x[s][i] = u + l;
                            x[s + h][i] = u - l;
                        }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 8; i += 2) xlane_pair_butterfly<16>(x[s][i], x[s][i + 1]);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 8; i += 2) xlane_pair_butterfly<32>(x[s][i], x[s][i + 1]);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] *= a.wht_scale;
        }
        float m = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[s][i]));
        m = pg_max_groups(m);
        int ex = 0;
        if (m > 0.0f && m < INFINITY) frexpf(m, &ex);
        ex = ex < -100 ? -100 : ex;
        const float sr = ldexpf(a.qscale < 0.0f ? -1.0f : 1.0f, 15 - ex);
        if (g == 0) csc_l[16 * wave + n] = fabsf(a.qscale) * ldexpf(cdiv, ex - 15);
        half8_t qh[4], ql[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint32_t hw[4], lw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v0 = x[s][2 * j] * sr, v1 = x[s][2 * j + 1] * sr;
                hw[j] = pg_pack(v0, v1);
                lw[j] = HL ? pg_pack(v0 - pg_h_lo(hw[j]), v1 - pg_h_hi(hw[j])) : 0u;
            }
            qh[s] = pg_half8(hw[0], hw[1], hw[2], hw[3]);
            ql[s] = pg_half8(lw[0], lw[1], lw[2], lw[3]);
            qimg[(wave * L::kSteps + s) * 64 + lane] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
            if (HL) qimg[kPlane + (wave * L::kSteps + s) * 64 + lane] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
        }
        if (QJL) {
            // G q: projections 16 cb + 4 g + i of row n
            float p[4][4];
#pragma unroll
            for (int cb = 0; cb < 4; ++cb) {
                const uint32_t w = a.g_bits[((int64_t)hk * 64 + 16 * cb + n) * 4 + g];
                float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t e[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t two = (w >> (8 * s + 2 * j)) & 3u;
                        e[j] = ((two & 1u) ? 0x3C00u : 0xBC00u) | ((two & 2u) ? 0x3C000000u : 0xBC000000u);
                    }
                    const half8_t ga = pg_half8(e[0], e[1], e[2], e[3]);
                    acc = pg_mfma(ga, qh[s], acc);
                    if (HL) acc = pg_mfma(ga, ql[s], acc);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) p[cb][i] = acc[i] * a.alpha;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t hw[4], lw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v0 = p[2 * s + (j >> 1)][2 * (j & 1)], v1 = p[2 * s + (j >> 1)][2 * (j & 1) + 1];
                    hw[j] = pg_pack(v0, v1);
                    lw[j] = HL ? pg_pack(v0 - pg_h_lo(hw[j]), v1 - pg_h_hi(hw[j])) : 0u;
                }
                qimg[(wave * L::kSteps + 4 + s) * 64 + lane] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                if (HL) qimg[kPlane + (wave * L::kSteps + 4 + s) * 64 + lane] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
            }
        }
    }
    __syncthreads();

    // ── main loop ─────────────────────────────────────────────────────
    auto qop = [&](int rg, int s, int plane) {
        return __builtin_bit_cast(half8_t, qimg[plane * kPlane + (rg * L::kSteps + s) * 64 + lane]);
    };
    half8_t qr[QREG ? NR : 1][L::kSteps][HL ? 2 : 1];
    if constexpr (QREG) {
#pragma unroll
        for (int rg = 0; rg < NR; ++rg)
#pragma unroll
            for (int s = 0; s < L::kSteps; ++s)
#pragma unroll
                for (int p = 0; p < (HL ? 2 : 1); ++p) qr[rg][s][p] = qop(rg, s, p);
    }
    auto q_at = [&](int rg, int s, int p) {
        if constexpr (QREG) return qr[rg][s][p];
        else return qop(rg, s, p);
    };
    float csc[NR], m_run[NR], l_run[NR];
    uint64_t sees[NR];
    float4_t oacc[NR][8];
#pragma unroll
    for (int rg = 0; rg < NR; ++rg) {
        csc[rg] = csc_l[16 * rg + n];
        m_run[rg] = -__FLT_MAX__;        // finite: a tile without a visible key leaves exp2(-inf) = 0
        l_run[rg] = 0.0f;
        sees[rg] = 0;
        if constexpr (!BLOCKS) {
            const int rho = (chunk * NR + rg) * 16 + n;
            if (rho < a.rows) sees[rg] = (uint64_t)a.tree[li.b * a.tree_stride + rho / a.G];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) oacc[rg][k] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const uint32_t laneoff = HL ? (lane & 31) * 8u : lane * 4u;
    const uint32_t slane = kSignOff + (lane & 31) * 8u;
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
    // table entry of byte k of w: (byte << 8) | the lane's column
    auto entry = [&](uint32_t w, int k) {
        const uint32_t at = __builtin_amdgcn_perm(w, laneoff, 0x0C0C0000u | ((uint32_t)(4 + k) << 8));
        if constexpr (HL) return *reinterpret_cast<const uint2 *>(smem + at);
        else return make_uint2(*reinterpret_cast<const uint32_t *>(smem + at), 0u);
    };
    auto step = [&](const PgTile &R, int64_t tile) {
        if (BLOCKS && R.nv[0] + R.nv[1] == 0) return;
        float4_t acc[NR][2], qacc[NR][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int rg = 0; rg < NR; ++rg) acc[rg][u] = qacc[rg][u] = float4_t{0.f, 0.f, 0.f, 0.f};
            const uint32_t kw[4] = {R.k[u].x, R.k[u].y, R.k[u].z, R.k[u].w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint2 e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = entry(kw[s], k);
                const half8_t ah = pg_half8(e[0].x, e[1].x, e[2].x, e[3].x);
#pragma unroll
                for (int rg = 0; rg < NR; ++rg) {
                    acc[rg][u] = pg_mfma(ah, q_at(rg, s, 0), acc[rg][u]);
                    if constexpr (HL) {
                        acc[rg][u] = pg_mfma(ah, q_at(rg, s, 1), acc[rg][u]);
                        acc[rg][u] = pg_mfma(pg_half8(e[0].y, e[1].y, e[2].y, e[3].y), q_at(rg, s, 0), acc[rg][u]);
                    }
                }
            }
            if constexpr (QJL) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t w = s ? R.sg[u].y : R.sg[u].x;
                    const uint2 e0 = *reinterpret_cast<const uint2 *>(smem + ((__builtin_amdgcn_ubfe(w, 4u * g, 4u) << 8) + slane));
                    const uint2 e1 = *reinterpret_cast<const uint2 *>(smem + ((__builtin_amdgcn_ubfe(w, 16u + 4u * g, 4u) << 8) + slane));
                    const half8_t sa = pg_half8(e0.x, e0.y, e1.x, e1.y);
#pragma unroll
                    for (int rg = 0; rg < NR; ++rg) {
                        qacc[rg][u] = pg_mfma(sa, q_at(rg, 4 + s, 0), qacc[rg][u]);
                        if constexpr (HL) qacc[rg][u] = pg_mfma(sa, q_at(rg, 4 + s, 1), qacc[rg][u]);
                    }
                }
            }
        }
        float nr[8];
        if constexpr (QJL) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                nr[4 * u] = R.nr[u].x * cmul;
                nr[4 * u + 1] = R.nr[u].y * cmul;
                nr[4 * u + 2] = R.nr[u].z * cmul;
                nr[4 * u + 3] = R.nr[u].w * cmul;
            }
        }
        const bool full = R.nv[0] == 16 && R.nv[1] == 16 && (BLOCKS || (tile + 1) * kPgTile <= li.base);
        half8_t pb[NR];
#pragma unroll
        for (int rg = 0; rg < NR; ++rg) {
            float sc[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = acc[rg][u][i];
                    if constexpr (QJL) v = __builtin_fmaf(nr[4 * u + i], qacc[rg][u][i], v);
                    sc[4 * u + i] = v * csc[rg];
                }
            if (!full) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = 4 * g + i;
                        bool vis = tok < R.nv[u];
                        if constexpr (!BLOCKS) {
                            const int64_t j = tile * kPgTile + 16 * u + tok - li.base;
                            vis = vis && (j < 0 || ((sees[rg] >> (j & 63)) & 1u));
                        }
                        sc[4 * u + i] = vis ? sc[4 * u + i] : -INFINITY;
                    }
            }
            // m_run is the same in a row's four lane groups: each lane tests its
            // own maximum, and the row's is formed only where some lane passes
            // the old one by 2^8 (P stays within fp16)
            float mt = pg_max3(pg_max3(sc[0], sc[1], sc[2]), pg_max3(sc[3], sc[4], sc[5]), pg_max(sc[6], sc[7]));
            if (__builtin_amdgcn_ballot_w64(mt > m_run[rg] + 8.0f)) {
                mt = pg_max_groups(mt);
                const bool need = mt > m_run[rg] + 8.0f;
                const float f = need ? __builtin_amdgcn_exp2f(m_run[rg] - mt) : 1.0f;
                m_run[rg] = need ? mt : m_run[rg];
                l_run[rg] *= f;
#pragma unroll
                for (int k = 0; k < 8; ++k) oacc[rg][k] *= f;
            }
            uint32_t p[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                p[k] = pg_pack(__builtin_amdgcn_exp2f(sc[2 * k] - m_run[rg]), __builtin_amdgcn_exp2f(sc[2 * k + 1] - m_run[rg]));
                l_run[rg] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, p[k]), ones, l_run[rg], false);
            }
            pb[rg] = pg_half8(p[0], p[1], p[2], p[3]);
        }
        uint32_t ev[4], od[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t va = R.v[2 * k], vb = R.v[2 * k + 1];
            ev[k] = ((vb << 4) & 0xF0F0F0F0u) | (va & 0x0F0F0F0Fu);
            od[k] = (vb & 0xF0F0F0F0u) | ((va >> 4) & 0x0F0F0F0Fu);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {                       // dims 8 m + k
            uint2 e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = entry(k & 1 ? od[j] : ev[j], k >> 1);
            const half8_t vh = pg_half8(e[0].x, e[1].x, e[2].x, e[3].x);
#pragma unroll
            for (int rg = 0; rg < NR; ++rg) {
                oacc[rg][k] = pg_mfma(vh, pb[rg], oacc[rg][k]);
                if constexpr (HL) oacc[rg][k] = pg_mfma(pg_half8(e[0].y, e[1].y, e[2].y, e[3].y), pb[rg], oacc[rg][k]);
            }
        }
    };
    if (cnt > 0) {
        const int64_t t0 = t_begin + wave;
        for (int k = 0;;) {
            load(R1, k + 1 < cnt ? k + 1 : cnt - 1);        // past the end: the last tile again, from cache
            __builtin_amdgcn_sched_barrier(0);
            step(R0, t0 + (int64_t)NW * k);
            if (++k >= cnt) break;
            load(R0, k + 1 < cnt ? k + 1 : cnt - 1);
            __builtin_amdgcn_sched_barrier(0);
            step(R1, t0 + (int64_t)NW * k);
            if (++k >= cnt) break;
        }
    }

    // ── merge of the waves, a row group at a time ─────────────────────
    const bool wave_bad = __builtin_amdgcn_ballot_w64(page_bad) != 0;
    const int64_t mine = t_end - t_begin;
    const int act = mine < 1 ? 1 : mine < NW ? (int)mine : NW;      // waves with tiles
    float *slab = reinterpret_cast<float *>(smem);
    float *ml = reinterpret_cast<float *>(smem + L::kMl);          // [wave][16][2], then a flag per wave
#pragma unroll
    for (int rg = 0; rg < NR; ++rg) {
        __syncthreads();                                           // the tables (or the last row group's slabs) are done with
        if ((chunk * NR + rg) * 16 >= a.rows) break;               // block-uniform
        if (wave < act) {
            const float l = pg_sum_groups(l_run[rg]);
            if (g == 0) {
                ml[(wave * 16 + n) * 2] = m_run[rg];
                ml[(wave * 16 + n) * 2 + 1] = l;
            }
            if (lane == 0) ml[NW * 32 + wave] = wave_bad ? 1.0f : 0.0f;
            float *dst = slab + (wave * 16 + n) * kPartRow;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float4 *d4 = reinterpret_cast<float4 *>(dst + 8 * (4 * g + i));
                d4[0] = make_float4(oacc[rg][0][i], oacc[rg][1][i], oacc[rg][2][i], oacc[rg][3][i]);
                d4[1] = make_float4(oacc[rg][4][i], oacc[rg][5][i], oacc[rg][6][i], oacc[rg][7][i]);
            }
        }
        __syncthreads();
        for (int e = tid; e < 16 * 32; e += 64 * NW) {
            const int r = e >> 5, d = 4 * (e & 31);
            const int rho = (chunk * NR + rg) * 16 + r;
            if (rho >= a.rows) break;
            float m = -__FLT_MAX__, l = 0.0f, nan = li.bad ? 1.0f : 0.0f;
            for (int w = 0; w < act; ++w) m = fmaxf(m, ml[(w * 16 + r) * 2]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < act; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[(w * 16 + r) * 2] - m);
                const float4 v = *reinterpret_cast<const float4 *>(slab + (w * 16 + r) * kPartRow + d);
                l = __builtin_fmaf(f, ml[(w * 16 + r) * 2 + 1], l);
                o.x = __builtin_fmaf(f, v.x, o.x);
                o.y = __builtin_fmaf(f, v.y, o.y);
                o.z = __builtin_fmaf(f, v.z, o.z);
                o.w = __builtin_fmaf(f, v.w, o.w);
                nan += ml[NW * 32 + w];
            }
            if (nan != 0.0f) l = __builtin_nanf("");
            const int t = BLOCKS ? li.t : rho / a.G;
            if (a.splits == 1) {
                const int hq = hk * a.G + (BLOCKS ? rho : rho - t * a.G);
                const float s = cdiv / l;
                float v[4] = {o.x * s, o.y * s, o.z * s, o.w * s};
                uint16_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!BLOCKS && !li.bad && t >= li.nd) v[i] = 0.0f;
                    h[i] = F16 ? f32_to_f16_rne(v[i]) : f32_to_bf16_rne(v[i]);
                }
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + ((li.b * a.Hq + hq) * a.T + t) * 128 + d) =
                    make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
            } else {
                float *p = a.ws + ((unit * a.splits + split) * a.rows + rho) * kPartRow;
                *reinterpret_cast<float4 *>(p + d) = make_float4(o.x * cdiv, o.y * cdiv, o.z * cdiv, o.w * cdiv);
                if (d == 0) {
                    p[128] = m;
                    p[129] = l;
                }
            }
        }
    }
}

// The splits' (m, l, O) of one row: 32 lanes, four dims each, eight splits'
// loads in flight.
template <bool F16, bool BLOCKS>
__global__ __launch_bounds__(256) void page_merge_kernel(PageAttnArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d = 4 * (threadIdx.x & 31);
    if (row >= a.units * a.rows) return;
    const int64_t unit = row / a.rows;
    const int rho = (int)(row - unit * a.rows);
    const PgList li = pg_list<BLOCKS>(a, unit);
    const int64_t share = pg_share(li.tiles, a.splits);
    const int act = li.tiles < 1 ? 1 : (int)((li.tiles + share - 1) / share);
    const float *base = a.ws + (unit * a.splits * a.rows + rho) * kPartRow;
    const int64_t stride = (int64_t)a.rows * kPartRow;
    float m = -__FLT_MAX__;
    for (int s0 = 0; s0 < act; s0 += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = base[(s0 + k < act ? s0 + k : act - 1) * stride + 128];
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, v[k]);
    }
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < act; s0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float *p = base + (s0 + k < act ? s0 + k : act - 1) * stride;
            ml[k] = *reinterpret_cast<const float2 *>(p + 128);
            v[k] = *reinterpret_cast<const float4 *>(p + d);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < act) {
                const float f = __builtin_amdgcn_exp2f(ml[k].x - m);
                l = __builtin_fmaf(f, ml[k].y, l);
                o.x = __builtin_fmaf(f, v[k].x, o.x);
                o.y = __builtin_fmaf(f, v[k].y, o.y);
                o.z = __builtin_fmaf(f, v[k].z, o.z);
                o.w = __builtin_fmaf(f, v[k].w, o.w);
            }
    }
    const int t = BLOCKS ? li.t : rho / a.G;
    const int hq = li.hk * a.G + (BLOCKS ? rho : rho - t * a.G);
    const float s = 1.0f / l;
    float v[4] = {o.x * s, o.y * s, o.z * s, o.w * s};
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!BLOCKS && !li.bad && t >= li.nd) v[i] = 0.0f;
        h[i] = F16 ? f32_to_f16_rne(v[i]) : f32_to_bf16_rne(v[i]);
    }
    *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + ((li.b * a.Hq + hq) * a.T + t) * 128 + d) =
        make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
}

// ── host ────────────────────────────────────────────────────────────────

struct PagePlan {
    int nr, chunks, splits;
    size_t ws;
};

// Row groups per block and splits of a call: `units` lists of at most `tiles`
// tiles, `rows` query rows each.
static PagePlan page_plan(int64_t units, int rows, int64_t tiles, bool hl) {
    PagePlan p;
    p.nr = rows <= 16 ? 1 : 2;
    p.chunks = (rows + 16 * p.nr - 1) / (16 * p.nr);
    const int64_t cus = device_cus(), blocks = units * p.chunks;
    const double tile = (p.nr == 1 ? 0.21 : 0.27) * (hl ? 1.6 : 1.0);
    double best = 1e30;
    p.splits = 1;
    auto consider = [&](int64_t s) {
        if (s < 1 || s > 256 || (s > 1 && tiles / s < 8)) return;
        const double t = (double)((blocks * s + cus - 1) / cus) * (5.0 + tile * (double)((tiles + s - 1) / s)) +
                         (s > 1 ? 3.0 + 0.03 * (double)s : 0.0);
        if (t < best) {
            best = t;
            p.splits = (int)s;
        }
    };
    consider(1);
    if (blocks > 0)
        for (int r = 1; r <= 4; ++r)
            for (int k = 0; k < 3; ++k) consider(r * cus / (blocks << k));
    p.ws = p.splits > 1 ? (size_t)units * p.splits * rows * kPartRow * 4 : 0;
    return p;
}

template <int NR, int NW, bool QJL, bool HL, bool BLOCKS>
static void page_launch(const PageAttnArgs &a, hipStream_t s) {
    const int64_t us = (a.units * a.splits + 7) / 8 * 8;
    hipLaunchKernelGGL((page_attn_kernel<NR, NW, QJL, HL, BLOCKS>), dim3((unsigned)(us * a.chunks)), dim3(64 * NW), 0, s, a);
}

template <bool BLOCKS>
static int page_run(PageAttnArgs &a, int q_dtype, bool qjl, int nr, hipStream_t s) {
    const bool hl = q_dtype == OMNI_F16;
    if (nr == 1) {
        if (hl) qjl ? page_launch<1, 8, true, true, BLOCKS>(a, s) : page_launch<1, 8, false, true, BLOCKS>(a, s);
        else qjl ? page_launch<1, 12, true, false, BLOCKS>(a, s) : page_launch<1, 12, false, false, BLOCKS>(a, s);
    } else {
        if (hl) qjl ? page_launch<2, 8, true, true, BLOCKS>(a, s) : page_launch<2, 8, false, true, BLOCKS>(a, s);
        else qjl ? page_launch<2, 8, true, false, BLOCKS>(a, s) : page_launch<2, 8, false, false, BLOCKS>(a, s);
    }
    OMNI_CHECK_LAUNCH("page_attn_kernel");
    if (a.splits > 1) {
        const unsigned blocks = (unsigned)((a.units * a.rows + 7) / 8);
        if (hl) hipLaunchKernelGGL((page_merge_kernel<true, BLOCKS>), dim3(blocks), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((page_merge_kernel<false, BLOCKS>), dim3(blocks), dim3(256), 0, s, a);
        OMNI_CHECK_LAUNCH("page_merge_kernel");
    }
    return OMNI_OK;
}

// The pool's geometry: page_size a power of two, every token row of the pool
// (page, head, slot) numbered below 2^31, positions in 32 bits.
int check_pool(const char *who, int64_t n_pages, int Hkv, int page_size, int64_t max_pages, int &shift) {
    shift = 0;
    while (shift < 11 && (1 << shift) < page_size) ++shift;
    OMNI_CHECK_ARG(page_size >= 16 && page_size <= 1024 && (1 << shift) == page_size,
                   "%s: page_size must be a power of two in [16, 1024], got %d", who, page_size);
    OMNI_CHECK_ARG(n_pages >= 1 && max_pages >= 1 && Hkv >= 1, "%s: need n_pages, max_pages and n_kv_heads >= 1", who);
    OMNI_CHECK_ARG(n_pages <= (int64_t(1) << 31) / Hkv / page_size,
                   "%s: pool too large (n_pages * n_kv_heads * page_size must be at most 2^31 tokens)", who);
    OMNI_CHECK_ARG(max_pages <= (int64_t(1) << 30) / page_size, "%s: max_pages * page_size must be at most 2^30", who);
    return OMNI_OK;
}

static int page_check(const char *who, const void *q, int q_dtype, const void *k_nib, const void *k_qjl, const void *k_norms,
                      const void *v_nib, const void *codebooks, const void *g_bits, int64_t B, int Hq, int Hkv, int64_t T,
                      int head_dim, float scale, int with_qjl, const void *out) {
    OMNI_CHECK_ARG(q_dtype == OMNI_F16 || q_dtype == OMNI_BF16, "%s: q must be float16 or bfloat16", who);
    OMNI_CHECK_ARG(head_dim == 128, "%s: head_dim must be 128, got %d", who, head_dim);
    OMNI_CHECK_ARG(B >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "%s: need B >= 0 and n_heads a multiple of n_kv_heads", who);
    OMNI_CHECK_ARG(T >= 1 && T <= 64, "%s: 1 to 64 query tokens, got %lld", who, (long long)T);
    OMNI_CHECK_ARG(Hq / Hkv <= 1024, "%s: at most 1024 query heads per kv head", who);
    OMNI_CHECK_ARG(B <= (int64_t(1) << 22) / Hkv / T, "%s: batch too large", who);
    OMNI_CHECK_ARG(fabsf(scale) <= 2.3e38f, "%s: scale must be finite and at most 2.3e38 in size", who);
    if (B == 0) return OMNI_OK;
    OMNI_CHECK_ARG(q && k_nib && v_nib && codebooks && out, "%s: NULL pointer", who);
    OMNI_CHECK_ARG(!with_qjl || (k_qjl && k_norms && g_bits), "%s: with_qjl needs signs, norms and G bits", who);
    return OMNI_OK;
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_attn_tree_workspace_size(int64_t B, int Hq, int Hkv, int64_t T, int64_t max_pages, int page_size,
                                                int q_dtype) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || T <= 0 || T > 64 || max_pages <= 0 || page_size < 16) return 0;
    return page_plan(B * Hkv, (int)T * (Hq / Hkv), (max_pages * page_size + kPgTile - 1) / kPgTile, q_dtype == OMNI_F16).ws;
}

extern "C" int omni_attn_tree(const void *q, int q_dtype, const uint8_t *k_nib, const uint8_t *k_qjl, const float *k_norms,
                              const uint8_t *v_nib, int64_t n_pages, int page_size, const int32_t *page_table,
                              int64_t max_pages, const int32_t *seq_lens, const int32_t *n_draft, const int64_t *tree,
                              int64_t tree_stride, const float *codebooks, int per_head_codebook, const uint32_t *g_bits,
                              int64_t B, int Hq, int Hkv, int64_t T, int head_dim, float scale, int with_qjl, int rotate_q,
                              const int8_t *sign_flip, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    int shift;
    OMNI_TRY(page_check("omni_attn_tree", q, q_dtype, k_nib, k_qjl, k_norms, v_nib, codebooks, g_bits, B, Hq, Hkv, T, head_dim,
                        scale, with_qjl, out));
    OMNI_TRY(check_pool("omni_attn_tree", n_pages, Hkv, page_size, max_pages, shift));
    if (B == 0) return OMNI_OK;
    OMNI_CHECK_ARG(page_table && seq_lens && tree, "omni_attn_tree: NULL page table, lengths or tree");
    OMNI_CHECK_ARG(tree_stride == 0 || tree_stride >= T, "omni_attn_tree: tree_stride must be 0 or at least T");
    const int G = Hq / Hkv;
    const PagePlan p = page_plan(B * Hkv, (int)T * G, (max_pages * page_size + kPgTile - 1) / kPgTile, q_dtype == OMNI_F16);
    if (p.ws > workspace_bytes || (p.ws && !workspace)) {
        set_error("omni_attn_tree: workspace of %zu bytes needed, %zu given", p.ws, workspace_bytes);
        return OMNI_EWORKSPACE;
    }
    PageAttnArgs a{q, out, (float *)workspace, k_nib, k_qjl, v_nib, k_norms, codebooks, g_bits, rotate_q ? sign_flip : nullptr,
                   page_table, seq_lens, n_draft, tree, nullptr, max_pages, n_pages, tree_stride, B * Hkv, shift,
                   per_head_codebook, Hq, Hkv, G, (int)T, (int)T * G, p.chunks, p.splits, 0, rotate_q,
                   (float)((double)scale * 1.4426950408889634), (float)(sqrt(2.0 / M_PI) / 128.0), inv_sqrt_dim_f32(128)};
    return page_run<false>(a, q_dtype, with_qjl != 0, p.nr, as_stream(stream));
}

extern "C" size_t omni_attn_blocks_workspace_size(int64_t B, int Hq, int Hkv, int64_t T, int top, int page_size, int q_dtype) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || T <= 0 || T > 64 || top <= 0 || page_size < 16) return 0;
    return page_plan(B * T * Hkv, Hq / Hkv, ((int64_t)top * page_size + kPgTile - 1) / kPgTile, q_dtype == OMNI_F16).ws;
}

extern "C" int omni_attn_blocks(const void *q, int q_dtype, const uint8_t *k_nib, const uint8_t *k_qjl, const float *k_norms,
                                const uint8_t *v_nib, int64_t n_pages, int page_size, const int32_t *page_table,
                                int64_t max_pages, const int32_t *seq_lens, const int32_t *blocks, int top,
                                const float *codebooks, int per_head_codebook, const uint32_t *g_bits, int64_t B, int Hq,
                                int Hkv, int64_t T, int head_dim, float scale, int with_qjl, int rotate_q,
                                const int8_t *sign_flip, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    int shift;
    OMNI_TRY(page_check("omni_attn_blocks", q, q_dtype, k_nib, k_qjl, k_norms, v_nib, codebooks, g_bits, B, Hq, Hkv, T,
                        head_dim, scale, with_qjl, out));
    OMNI_TRY(check_pool("omni_attn_blocks", n_pages, Hkv, page_size, max_pages, shift));
    OMNI_CHECK_ARG(top >= 1 && top <= (1 << 30) / page_size, "omni_attn_blocks: top must lie in [1, 2^30 / page_size], got %d", top);
    if (B == 0) return OMNI_OK;
    OMNI_CHECK_ARG(page_table && seq_lens && blocks, "omni_attn_blocks: NULL page table, lengths or blocks");
    const int G = Hq / Hkv;
    const PagePlan p = page_plan(B * T * Hkv, G, ((int64_t)top * page_size + kPgTile - 1) / kPgTile, q_dtype == OMNI_F16);
    if (p.ws > workspace_bytes || (p.ws && !workspace)) {
        set_error("omni_attn_blocks: workspace of %zu bytes needed, %zu given", p.ws, workspace_bytes);
        return OMNI_EWORKSPACE;
    }
    PageAttnArgs a{q, out, (float *)workspace, k_nib, k_qjl, v_nib, k_norms, codebooks, g_bits, rotate_q ? sign_flip : nullptr,
                   page_table, seq_lens, nullptr, nullptr, blocks, max_pages, n_pages, 0, B * T * Hkv, shift,
                   per_head_codebook, Hq, Hkv, G, (int)T, G, p.chunks, p.splits, top, rotate_q,
                   (float)((double)scale * 1.4426950408889634), (float)(sqrt(2.0 / M_PI) / 128.0), inv_sqrt_dim_f32(128)};
    return page_run<true>(a, q_dtype, with_qjl != 0, p.nr, as_stream(stream));
}

// ── prepared calls (PagedTreeAttention, PagedBlockAttention) ────────────
//
// The arguments that stay fixed across a serving loop, stored once; the plan
// holds pointers only, which must outlive it.
struct omni_attn_pages_plan {
    int q_dtype;
    const uint8_t *k_nib, *k_qjl, *v_nib, *bounds;      // bounds NULL: a tree plan
    const float *k_norms;
    int64_t n_pages;
    int page_size;
    int64_t max_pages;
    int32_t *blocks;
    int top, first, recent;
    const float *codebooks;
    int per_head_codebook;
    const uint32_t *g_bits;
    int64_t B;
    int Hq, Hkv;
    int64_t T;
    float scale;
    int with_qjl, rotate_q;
    const int8_t *sign_flip;
    void *out, *workspace;
    size_t workspace_bytes;
};

extern "C" int omni_attn_pages_plan_create(int q_dtype, const uint8_t *k_nib, const uint8_t *k_qjl, const float *k_norms,
                                           const uint8_t *v_nib, const uint8_t *bounds, int64_t n_pages, int page_size,
                                           int64_t max_pages, int32_t *blocks, int top, int first, int recent,
                                           const float *codebooks, int per_head_codebook, const uint32_t *g_bits, int64_t B,
                                           int Hq, int Hkv, int64_t T, float scale, int with_qjl, int rotate_q,
                                           const int8_t *sign_flip, void *out, void *workspace, size_t workspace_bytes,
                                           omni_attn_pages_plan **plan) {
    OMNI_CHECK_ARG(plan != nullptr, "omni_attn_pages_plan_create: NULL plan pointer");
    *plan = nullptr;
    int shift;
    OMNI_TRY(check_pool("omni_attn_pages_plan_create", n_pages, Hkv, page_size, max_pages, shift));
    omni_attn_pages_plan *p = new (std::nothrow) omni_attn_pages_plan;
    if (p == nullptr) {
        set_error("omni_attn_pages_plan_create: out of host memory");
        return OMNI_ERUNTIME;
    }
    *p = omni_attn_pages_plan{q_dtype, k_nib, k_qjl, v_nib, bounds, k_norms, n_pages, page_size, max_pages, blocks, top, first,
                              recent, codebooks, per_head_codebook, g_bits, B, Hq, Hkv, T, scale, with_qjl, rotate_q,
                              sign_flip, out, workspace, workspace_bytes};
    *plan = p;
    return OMNI_OK;
}

extern "C" int omni_attn_tree_plan_run(const omni_attn_pages_plan *p, const void *q, const int32_t *page_table,
                                       const int32_t *seq_lens, const int64_t *tree, int64_t tree_stride,
                                       const int32_t *n_draft, void *stream) {
    OMNI_CHECK_ARG(p != nullptr && p->bounds == nullptr, "omni_attn_tree_plan_run: not a tree plan");
    return omni_attn_tree(q, p->q_dtype, p->k_nib, p->k_qjl, p->k_norms, p->v_nib, p->n_pages, p->page_size, page_table,
                          p->max_pages, seq_lens, n_draft, tree, tree_stride, p->codebooks, p->per_head_codebook, p->g_bits,
                          p->B, p->Hq, p->Hkv, p->T, 128, p->scale, p->with_qjl, p->rotate_q, p->sign_flip, p->out,
                          p->workspace, p->workspace_bytes, stream);
}

extern "C" int omni_attn_blocks_plan_run(const omni_attn_pages_plan *p, const void *q, const int32_t *page_table,
                                         const int32_t *seq_lens, void *stream) {
    OMNI_CHECK_ARG(p != nullptr && p->bounds != nullptr, "omni_attn_blocks_plan_run: not a plan of blocks");
    // the selection's scores are read before the attention writes its partials
    OMNI_TRY(omni_block_select(q, p->q_dtype, p->bounds, p->n_pages, p->page_size, page_table, p->max_pages, seq_lens,
                               p->codebooks, p->per_head_codebook, p->B, p->Hq, p->Hkv, p->T, 128, p->top, p->first, p->recent,
                               p->rotate_q, p->sign_flip, p->blocks, p->workspace, p->workspace_bytes, stream));
    return omni_attn_blocks(q, p->q_dtype, p->k_nib, p->k_qjl, p->k_norms, p->v_nib, p->n_pages, p->page_size, page_table,
                            p->max_pages, seq_lens, p->blocks, p->top, p->codebooks, p->per_head_codebook, p->g_bits, p->B,
                            p->Hq, p->Hkv, p->T, 128, p->scale, p->with_qjl, p->rotate_q, p->sign_flip, p->out, p->workspace,
                            p->workspace_bytes, stream);
}

extern "C" void omni_attn_pages_plan_destroy(omni_attn_pages_plan *p) { delete p; }
