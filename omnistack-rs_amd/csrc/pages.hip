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
// its own running reference and sum, and are merged at the end.  All products on
// v_mfma_f32_16x16x32_f16, tokens on M for the scores and dims on M for P V:
//   table     64 KB of LDS, a row of 256 bytes for every code byte: in 32
//             columns its two centroids in fp16 and their remainders, 8 bytes.
//             A lane reads its own column, so a byte and the lane make the
//             address with one v_perm, and 32 lanes meet no bank twice.
//   K pass    A = centroids of 16 tokens (fp16 calls: and remainders); B = the
//             query rows.  Lane (n, g) reads bytes 16 g .. + 15 of token n, so
//             k-slot i of step s is dim 32 g + 8 s + i on both sides.
//   QJL pass  A = the signs, made from the sign words by shift, mask and xor
//             (with the norm in bf16 calls, as 1 in fp16 ones); B =
//             sqrt(2/pi)/128 G q, in the order of the sign bits that a lane
//             takes: projections 32 s + 4 g + j and 16 on.
//   P V       A = centroids and remainders side by side, two tokens' codes of
//             one dim interleaved into one table byte; B = P, each value twice.
// Numbers: q rows times a power of two (largest in [2^14, 2^15)) and the head's
// centroids times one are rounded to fp16.  bf16 queries that the call does not
// rotate lose nothing; rotated ones, K's centroids (less what is common to them,
// see `fit`), norms and G q lose 2^-12 of themselves, P another 2^-12 down to
// 2^-22 of the largest (the same rounded P in numerator and denominator): below
// the 2^-9 of the bf16 output.  V's centroids keep a second fp16 term in either
// type: their roundings do not average out over a long list as P's do.  fp16
// queries (HL) keep a second term of q, of G q and of K's centroids too (22
// bits), which leaves P's 2^-12 against the output's 2^-12.
// Scores, references, sums and accumulators are fp32.
//
// What bounds it: many rows, the matrix and the vector units in turn (32
// sequences of 8192 tokens and 16 drafted, 64 rows a list: 124 us, 690 TFLOP/s
// of the 1200 to 1550 that large products reach by their layout; matrix units
// busy in 42 % of the cycles, vector instructions issuing in 45 %, 256 registers
// hold a SIMD at two waves).  Few rows, the cache's read and the vector work per
// tile (16 rows 52 us, 294 MB at 5.7 TB/s; a plain read reaches 7.1).  Short
// lists, a block's chain of dependent accesses, 7 to 8 us: lengths, page ids,
// tiles and q one after another, the table (0.7 us), G q, and the waves' merge
// (1.5 us).
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
    uint64_t hkv_magic, t_magic, g_magic;        // pg_div by Hkv, T and G
    float qscale;                // scale log2 e
    float alpha, wht_scale;      // sqrt(2/pi) / 128, 1 / sqrt(128) as fp32
};

constexpr int kPgTile = 32;
constexpr int kPartRow = 128 + 4;            // floats of a split's row: O, then m and l
constexpr int kLutBytes = 65536;             // the table
constexpr int kQimgOff = kLutBytes;
constexpr int kBufWord3 = 0x00020000;        // raw buffer, gfx9 descriptor dword 3
constexpr float kLag = 13.0f, kBelow = 8.0f; // of the softmax's reference, base 2: see `settle`

// What a variant keeps where.  NR: groups of 16 query rows a block; HL: fp16
// queries; PAIR: two blocks a CU (128 registers a lane), else one.
template <int NR, bool QJL, bool HL, int WAVES, bool PAIR>
struct Pg {
    static constexpr int NW = WAVES;
    // steps whose B operands stay in registers; the others are read from LDS for every tile
    static constexpr int kQKept = NR > 2 || PAIR ? 0 : HL && NR == 2 ? 8 : 99;
    static constexpr int kQSteps = HL ? 8 : 4;                               // B operands of a row group: q (HL: twice four),
    static constexpr int kGSteps = QJL ? (HL ? 4 : 2) : 0;                   // then G q (HL: twice two)
    static constexpr int kSteps = kQSteps + kGSteps;
    static constexpr int kQimg = NR * kSteps * 1024;
    static constexpr int kCsc = kQimgOff + kQimg;                            // per row: score scale
    static constexpr int kSees = kCsc + NR * 16 * 4;                         // per row: its tree mask
    static constexpr int kM = kSees + NR * 16 * 8;                           // [row][wave]: references, then sums
    static constexpr int kFlags = kM + 2 * NR * 16 * NW * 4;                 // per wave: met a page outside the pool
    static constexpr int kUse = kFlags + 16 * 4;
    // the merge: the waves' O of MR row groups at a time, from 0 on (over the tables and the query rows)
    static constexpr int MR = NR % 2 == 0 && NW <= 8 && !PAIR ? 2 : 1;
    static constexpr int kSlabs = NW * MR * 16 * kPartRow * 4;
    static constexpr int kMoved = kSlabs > kCsc ? kSlabs - kCsc : 0;         // what lies behind them moves up
    static constexpr int kLds = kUse + kMoved;
    static_assert(kLds <= (PAIR ? 81920 : 163840), "LDS of a CU");
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
// x of lane c ^ m of a 16-lane row, m a power of two
__device__ __forceinline__ float pg_row_xor(float x, int m, int c) {
    const int v = __float_as_int(x);
    if (m == 1) return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true));            // quad_perm [1,0,3,2]
    if (m == 2) return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true));            // quad_perm [2,3,0,1]
    if (m == 8) return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true));           // row_ror:8
    const int up = __builtin_amdgcn_mov_dpp(v, 0x12C, 0xf, 0xf, true);                               // row_ror:12: lane c + 4
    const int dn = __builtin_amdgcn_mov_dpp(v, 0x124, 0xf, 0xf, true);                               // row_ror:4: lane c - 4
    return __int_as_float(c & 4 ? dn : up);
}
// The larger, or NaN if one is: single instructions (fmaxf quiets operands
// first that the compiler cannot prove quiet, such as a matrix product's).
__device__ __forceinline__ float pg_max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float pg_max_groups(float m) {
    auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
    auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1]));
}
__device__ __forceinline__ float pg_sum_groups(float v) {
    auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(u[0]) + __uint_as_float(u[1]);
}

// floor(x / d) as (x (floor(2^32 / d) + 1)) >> 32: exact for x d < 2^32
__device__ __forceinline__ uint32_t pg_div(uint32_t x, uint64_t magic) { return (uint32_t)(((uint64_t)x * magic) >> 32); }

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
__device__ __forceinline__ PgList pg_list(const PageAttnArgs &a, uint32_t unit) {
    PgList l;
    const uint32_t bt = pg_div(unit, a.hkv_magic);
    l.hk = (int)(unit - bt * (uint32_t)a.Hkv);
    l.b = BLOCKS ? pg_div(bt, a.t_magic) : bt;
    l.t = BLOCKS ? (int)(bt - (uint32_t)l.b * (uint32_t)a.T) : 0;
    return l;
}
template <bool BLOCKS>
__device__ __forceinline__ void pg_length(const PageAttnArgs &a, PgList &l) {
    const int64_t len = a.seq_lens[l.b];
    l.bad = len < 0 || len > (a.max_pages << a.page_shift);
    if constexpr (BLOCKS) {
        l.nd = a.T;
        l.seen = l.bad || len - a.T + l.t + 1 < 0 ? 0 : len - a.T + l.t + 1;
        l.base = 0;
        l.tiles = (((int64_t)a.top << (a.page_shift - 4)) + 1) >> 1;
    } else {
        l.nd = a.n_draft ? a.n_draft[l.b] : a.T;
        l.bad = l.bad || l.nd < 0 || l.nd > a.T || l.nd > len;
        l.seen = l.bad ? 0 : len;
        l.base = l.seen - l.nd;
        l.tiles = (l.seen + kPgTile - 1) / kPgTile;
    }
}
// tiles of a split: even shares, so the splits of a short list are short
__device__ __forceinline__ int64_t pg_share(int64_t tiles, int splits) {
    return (int64_t)(((uint32_t)tiles + (uint32_t)splits - 1) / (uint32_t)splits);
}

template <bool HL>
struct PgKeys {
    uint4 k[2];                  // code bytes 16 g .. + 15 of token n of half u
    uint2 sg[2];                 // its sign bytes
    float nr[2][HL ? 4 : 1];     // its norm; HL: the norms of tokens 4 g .. + 3
};
struct PgValues {
    uint32_t v[8];               // code bytes 4 n .. + 3 of tokens 16 (i / 4) + 4 g + i % 4
};

template <int NR, bool QJL, bool HL, bool BLOCKS, int NW, bool PAIR>
__global__ __launch_bounds__(64 * NW, (PAIR ? 4 : NW / 4)) void page_attn_kernel(PageAttnArgs a) {
    using L = Pg<NR, QJL, HL, NW, PAIR>;
    __shared__ __attribute__((aligned(16))) unsigned char smem[L::kLds];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;

    // x: eight units, then row chunks; y: splits; z: groups of eight units.  The
    // chunks of one (unit, split) are eight blocks apart: they run on one XCD
    // and share its L2.
    const uint32_t unit = blockIdx.z * 8u + (blockIdx.x & 7u);
    const int chunk = (int)(blockIdx.x >> 3), split = (int)blockIdx.y;
    if (unit >= (uint32_t)a.units) return;
    PgList li = pg_list<BLOCKS>(a, unit);
    const int hk = li.hk;

    // ── query rows, four a wave, on their way: 16 lanes a row, eight dims a lane ──
    constexpr int kPasses = NR * 4 / NW + (NR * 4 % NW ? 1 : 0);
    const int c = lane & 15;                                // dims 8 c .. + 7
    uint4 q_raw[kPasses];
    uint2 q_flip = make_uint2(0u, 0u);
    bool q_ok[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int rl = 4 * (wave + i * NW) + g, rho = chunk * NR * 16 + rl;     // row of the block, of the unit
        q_ok[i] = rl < NR * 16 && rho < a.rows;
        const int rr = q_ok[i] ? rho : 0;
        const int t = BLOCKS ? li.t : (int)pg_div((uint32_t)rr, a.g_magic);
        const int hq = hk * a.G + (BLOCKS ? rr : rr - t * a.G);
        q_raw[i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.q) + ((li.b * a.Hq + hq) * a.T + t) * 128 + 8 * c);
    }
    if (a.sign_flip) q_flip = *reinterpret_cast<const uint2 *>(a.sign_flip + 8 * c);
    // G rows 16 cb + n, word g, for the product of row group rg that this wave forms
    constexpr int kGPasses = QJL ? kPasses : 0;
    uint32_t g_word[QJL ? kPasses : 1];
#pragma unroll
    for (int i = 0; i < kGPasses; ++i) g_word[i] = a.g_bits[((int64_t)hk * 64 + 16 * ((wave + i * NW) & 3) + n) * 4 + g];
    uint64_t sees_row = 0;
    if (!BLOCKS && tid < NR * 16 && chunk * NR * 16 + tid < a.rows)
        sees_row = (uint64_t)a.tree[li.b * a.tree_stride + pg_div((uint32_t)(chunk * NR * 16 + tid), a.g_magic)];
    const float cent = (a.codebooks + (a.per_head ? hk * 16 : 0))[c];      // lane l: centroid l % 16

    pg_length<BLOCKS>(a, li);
    const int64_t share = pg_share(li.tiles, a.splits);
    const int64_t t_begin = split * share, t_end = t_begin + share < li.tiles ? t_begin + share : li.tiles;
    if (split > 0 && t_begin >= li.tiles) return;           // the merge counts the splits that have tiles

    // ── the wave's tiles: pool rows of their halves, one tile a lane ──
    const int cnt = t_end - t_begin > wave ? (int)((t_end - t_begin - wave + NW - 1) / NW) : 0;
    uint32_t row0 = 0, row1 = 0, nvs = 0;
    bool page_bad = false;
    int64_t slot_pos[2], slot_page[2];
    int32_t slot_id[2];
    auto fetch_slots = [&](int first) {                      // which tokens, and their page table entries
        const int64_t tile = t_begin + wave + (int64_t)NW * (first + lane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t half = 2 * tile + u;
            slot_pos[u] = half << 4;                         // of its first token
            slot_page[u] = half >> (a.page_shift - 4);
            bool in = first + lane < cnt;
            if constexpr (BLOCKS) {
                const int64_t nb = (li.seen + (1 << a.page_shift) - 1) >> a.page_shift;
                in = in && slot_page[u] < a.top;
                const int64_t blk = in ? a.blocks[((li.b * a.Hkv + hk) * a.T + li.t) * a.top + slot_page[u]] : -1;
                in = blk >= 0 && blk < nb;
                slot_pos[u] = (blk << a.page_shift) + (slot_pos[u] & ((1 << a.page_shift) - 1));
                slot_page[u] = blk;
            }
            in = in && slot_pos[u] < li.seen;
            if (!in) slot_pos[u] = li.seen;
            slot_id[u] = in ? a.page_table[li.b * a.max_pages + slot_page[u]] : 0;
        }
    };
    auto fetch_rows = [&]() {
        uint32_t r[2], v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t left = li.seen - slot_pos[u];
            v[u] = left < 16 ? (uint32_t)left : 16u;
            const bool ok = slot_id[u] >= 0 && slot_id[u] < a.n_pages;
            page_bad = page_bad || !ok;
            r[u] = (((uint32_t)(ok ? slot_id[u] : 0) * (uint32_t)a.Hkv + (uint32_t)hk) << a.page_shift) +
                   (v[u] ? (uint32_t)(slot_pos[u] & ((1 << a.page_shift) - 1)) : 0u);
        }
        row0 = r[0];
        row1 = r[1];
        nvs = v[0] | (v[1] << 8);
    };
    auto rows_at = [&](int k, uint32_t (&r)[2], int &v) {
        if ((k & 63) == 0 && k > 0) {
            fetch_slots(k);
            fetch_rows();
        }
        r[0] = (uint32_t)__builtin_amdgcn_readlane((int)row0, k & 63);
        r[1] = (uint32_t)__builtin_amdgcn_readlane((int)row1, k & 63);
        v = __builtin_amdgcn_readlane((int)nvs, k & 63);
    };
    // a half's 16 tokens of one array: the descriptor starts at its row, so a
    // lane's offset is the same for every tile
    auto half_of = [&](const void *base, uint32_t r, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)(reinterpret_cast<const char *>(base) + (uint64_t)r * bytes), (short)0,
                                                 (int)(16 * bytes), kBufWord3);
    };
    auto load_k = [&](PgKeys<HL> &R, const uint32_t (&r)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            R.k[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(half_of(a.k_nib, r[u], 64), 64 * n + 16 * g, 0, 0));
            if constexpr (QJL) {
                R.sg[u] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(half_of(a.k_qjl, r[u], 8), 8 * n, 0, 0));
                if constexpr (HL) {
                    const float4 f = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(half_of(a.k_norms, r[u], 4), 16 * g, 0, 0));
                    R.nr[u][0] = f.x;
                    R.nr[u][1] = f.y;
                    R.nr[u][2] = f.z;
                    R.nr[u][3] = f.w;
                } else {
                    R.nr[u][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(half_of(a.k_norms, r[u], 4), 4 * n, 0, 0));
                }
            }
        }
    };
    auto load_v = [&](PgValues &R, const uint32_t (&r)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const auto V = half_of(a.v_nib, r[u], 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) R.v[4 * u + i] = __builtin_amdgcn_raw_buffer_load_b32(V, 256 * g + 4 * n + 64 * i, 0, 0);
        }
    };
    auto clamp = [&](int k) { return k < cnt ? k : cnt - 1; };     // past the end: the last tile again, from cache
    fetch_slots(0);

    // ── tables ────────────────────────────────────────────────────────
    float cmax = fabsf(cent);
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) cmax = fmaxf(cmax, pg_row_xor(cmax, m, c));
    cmax = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(cmax)));
    int cexp = 0;
    if (cmax > 0.0f && cmax < INFINITY) frexpf(cmax, &cexp);
    cexp = cexp < -100 ? -100 : cexp;
    // largest centroid in [2^(kc - 1), 2^kc): HL up to 2^10, for the remainders
    // of small ones; else 1, for norms, which follow them: up to 65504 of it in
    // the fast way
    constexpr int kc = HL ? 10 : 0;
    const float cmul = ldexpf(1.0f, kc - cexp), cdiv = ldexpf(1.0f, cexp - kc);
    {
        const uint16_t h = f32_to_f16_rne(cent * cmul);
        const uint32_t both = (uint32_t)h | ((uint32_t)f32_to_f16_rne(cent * cmul - f16_to_f32(h)) << 16);
#pragma unroll
        for (int i = 0; i < (4096 + 64 * NW - 1) / (64 * NW); ++i) {
            const int m = tid + 64 * NW * i, e = m >> 4;           // 16 threads a byte
            const uint32_t w0 = __shfl(both, e & 15), w1 = __shfl(both, (e >> 4) & 15);
            const uint32_t hi = __builtin_amdgcn_perm(w1, w0, 0x05040100u), lo = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
            if (m < 4096) *reinterpret_cast<uint4 *>(smem + 16 * m) = make_uint4(hi, lo, hi, lo);
        }
    }

    // ── the first tiles, on their way ─────────────────────────────────
    fetch_rows();
    PgKeys<HL> K;
    PgValues V;
    int nv = 0;                                   // tokens of each half that the list holds: low byte, next byte
    if (cnt > 0) {
        uint32_t r[2];
        rows_at(0, r, nv);
        load_k(K, r);
        load_v(V, r);
    }
    __builtin_amdgcn_sched_barrier(0);

    // The part of the centroids' rounding that is common to keys: where a row
    // leans on a key along itself, its score is off by sum f c (h - c) / sum f c^2
    // of itself, f the codes' frequencies; the score scale takes that back.  A
    // calibrated codebook's codes come about as often as 1 / spacing^2 (points
    // lie as density^(1/3)).  Score error of such rows 1e-4 to 3e-4 without,
    // 2e-5 to 6e-5 with it; other codebooks: a weighted mean of the roundings.
    float fit = 1.0f;
    if constexpr (!HL) {
        const float x = cent * cmul;
        const float up = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x101, 0xf, 0xf, true));      // row_shl:1: lane c + 1
        const float dn = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x111, 0xf, 0xf, true));      // row_shr:1: lane c - 1
        const float gap = c == 0 ? up - x : c == 15 ? x - dn : 0.5f * (up - dn), w = __builtin_amdgcn_rcpf(gap * gap + 0x1p-20f);
        float over = w * x * (f16_to_f32(f32_to_f16_rne(x)) - x), of = w * x * x;
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) {
            over += pg_row_xor(over, m, c);
            of += pg_row_xor(of, m, c);
        }
        fit = of > 0.0f ? 1.0f - over / of : 1.0f;
    }

    // ── query rows into MFMA operands ─────────────────────────────────
    uint4 *qimg = reinterpret_cast<uint4 *>(smem + kQimgOff);      // [rg][step][lane]
    float *csc_l = reinterpret_cast<float *>(smem + L::kMoved + L::kCsc);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int rl = 4 * (wave + i * NW) + g, rg = rl >> 4;
        if (4 * (wave + i * NW) >= NR * 16) break;                 // wave-uniform
        float x[8];
        {
            const uint32_t w[4] = {q_raw[i].x, q_raw[i].y, q_raw[i].z, q_raw[i].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint16_t h = (uint16_t)((j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
                x[j] = q_ok[i] ? (HL ? f16_to_f32(h) : bf16_to_f32(h)) : 0.0f;
            }
        }
        if (a.rotate) {
            // the normalized WHT in stage order h = 1 .. 64, not rounded to
            // q's type in between
            if (a.sign_flip) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = __uint_as_float(__float_as_uint(x[j]) ^
                                           (((j < 4 ? q_flip.x >> (8 * j) : q_flip.y >> (8 * j - 32)) & 0x80u) << 24));
            }
#pragma unroll
            for (int h = 1; h < 8; h <<= 1)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(j & h)) {
                        const float u = x[j], l = x[j + h];
                        x[j] = u + l;
                        x[j + h] = u - l;
                    }
            // stages 8 .. 64: lanes c ^ 1, 2, 4, 8 (an fma with +-1 rounds as the sum)
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) {
                const float sgn = c & m ? -1.0f : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf(sgn, x[j], pg_row_xor(x[j], m, c));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= a.wht_scale;
        }
        float m = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                        fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7]))));
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) m = fmaxf(m, pg_row_xor(m, k, c));
        int ex = 0;
        if (m > 0.0f && m < INFINITY) frexpf(m, &ex);
        ex = ex < -100 ? -100 : ex;
        const float sr = ldexpf(a.qscale < 0.0f ? -1.0f : 1.0f, 15 - ex);
        // at least FLT_MIN (scores are as good as 0 either way), so that a hidden score's -inf stays one
        if (c == 0) csc_l[rl] = fmaxf(fabsf(a.qscale) * fit * ldexpf(cdiv, ex - 15), __FLT_MIN__);
        uint32_t hw[4], lw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v0 = x[2 * j] * sr, v1 = x[2 * j + 1] * sr;
            hw[j] = pg_pack(v0, v1);
            lw[j] = HL ? pg_pack(v0 - pg_h_lo(hw[j]), v1 - pg_h_hi(hw[j])) : 0u;
        }
        // dims 8 c .. + 7 are step c % 4 of lane (row, c / 4)
        uint4 *dst = qimg + rg * L::kSteps * 64 + 16 * (c >> 2) + (rl & 15);
        const int s = c & 3;
        dst[64 * s] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
        if constexpr (HL) dst[64 * (4 + s)] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
    }
    uint64_t *sees_l = reinterpret_cast<uint64_t *>(smem + L::kMoved + L::kSees);    // per row: the drafted tokens that it sees
    if (!BLOCKS && tid < NR * 16) sees_l[tid] = sees_row;
    __syncthreads();
    if constexpr (QJL) {
        // G q: projections 16 cb + 4 g + i of row n of group rg, a wave for each (rg, cb)
#pragma unroll
        for (int i = 0; i < kGPasses; ++i) {
            const int item = wave + i * NW, rg = item >> 2, cb = item & 3;
            if (item >= NR * 4) break;                             // wave-uniform
            const uint4 *img = qimg + rg * L::kSteps * 64 + lane;
            float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < L::kQSteps; ++s) {
                uint32_t e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t not2 = ~g_word[i] >> (8 * (s & 3) + 2 * j);
                    e[j] = 0x3C003C00u | ((not2 & 1u) << 15) | ((not2 & 2u) << 30);
                }
                acc = pg_mfma(pg_half8(e[0], e[1], e[2], e[3]), __builtin_bit_cast(half8_t, img[64 * s]), acc);
            }
            // slots 2 j and 2 j + 1 of step s: projections 32 s + 4 g + j and 16 on, whose signs lie 16 bits apart
            uint16_t *dst = reinterpret_cast<uint16_t *>(qimg + (rg * L::kSteps + L::kQSteps + (cb >> 1)) * 64 + lane) + (cb & 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = acc[j] * a.alpha;
                const uint16_t h = f32_to_f16_rne(p);
                dst[2 * j] = h;
                if constexpr (HL) dst[2 * 64 * 8 + 2 * j] = f32_to_f16_rne(p - f16_to_f32(h));
            }
        }
        __syncthreads();
    }

    // ── main loop ─────────────────────────────────────────────────────
    uint32_t q_off = kQimgOff + 16 * lane;
    constexpr int kKept = L::kQKept < L::kSteps ? L::kQKept : L::kSteps;
    half8_t qr[NR][kKept + 1];
    {
#pragma unroll
        for (int rg = 0; rg < NR; ++rg)
#pragma unroll
            for (int s = 0; s < kKept; ++s) qr[rg][s] = *reinterpret_cast<const half8_t *>(smem + q_off + (rg * L::kSteps + s) * 1024);
    }
    auto q_at = [&](int rg, int s) {
        if (s < kKept) return qr[rg][s];
        else return *reinterpret_cast<const half8_t *>(smem + q_off + (rg * L::kSteps + s) * 1024);
    };
    float csc[NR], m_run[NR], l_run[NR];
    float4_t oacc[NR][8];
#pragma unroll
    for (int rg = 0; rg < NR; ++rg) {
        csc[rg] = csc_l[16 * rg + n];
        m_run[rg] = -__FLT_MAX__;        // finite: a tile without a visible key leaves exp2(-inf) = 0
        l_run[rg] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) oacc[rg][k] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const uint32_t laneoff = (lane & 31) * 8u;
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
    // table address of byte k of w: (byte << 8) | the lane's column
    auto entry = [&](uint32_t w, int k) {
        return smem + __builtin_amdgcn_perm(w, laneoff, 0x0C0C0000u | ((uint32_t)(4 + k) << 8));
    };
    // the fp16 centroids of a word's four bytes
    auto four_bytes = [&](uint32_t w) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = *reinterpret_cast<const uint32_t *>(entry(w, j));
        return pg_half8(h[0], h[1], h[2], h[3]);
    };
    // HL: and their remainders
    auto four_pairs = [&](uint32_t w, half8_t &hi, half8_t &lo) {
        uint2 e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = *reinterpret_cast<const uint2 *>(entry(w, j));
        hi = pg_half8(e[0].x, e[1].x, e[2].x, e[3].x);
        lo = pg_half8(e[0].y, e[1].y, e[2].y, e[3].y);
    };
    // centroids and remainders of byte i of x and byte j of y
    auto two_bytes = [&](uint32_t x, int i, uint32_t y, int j) {
        const uint2 e0 = *reinterpret_cast<const uint2 *>(entry(x, i)), e1 = *reinterpret_cast<const uint2 *>(entry(y, j));
        return pg_half8(e0.x, e0.y, e1.x, e1.y);
    };
    // scores of a tile, raw: lane (n, g) holds tokens 16 u + 4 g + i of row n
    auto scores = [&](const PgKeys<HL> &R, float4_t (&acc)[NR][2], uint64_t &large) {
        if constexpr (kKept < L::kSteps) asm volatile("" : "+v"(q_off));       // read again for each tile, not kept (and spilled)
#pragma unroll
        for (int rg = 0; rg < NR; ++rg)
#pragma unroll
            for (int u = 0; u < 2; ++u) acc[rg][u] = float4_t{0.f, 0.f, 0.f, 0.f};
        // norms beyond fp16 count as 0 here, and in `large_signs`
        float nrm[2] = {0.0f, 0.0f};
        if constexpr (QJL && !HL) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float x = -cmul * R.nr[u][0];
                const bool over = fabsf(x) > 65504.0f;
                large |= __builtin_amdgcn_ballot_w64(over);
                nrm[u] = over ? 0.0f : x;
            }
        }
        if constexpr (QJL) {
            // the signs' part.  The norm rides on the signs (fp16, 2^-12 of a
            // small term); HL: +-1, and the sums times the norms
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                half8_t A[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t nh = HL ? 0xBC00BC00u : pg_pack(nrm[u], nrm[u]);
                    const uint32_t w = (s ? R.sg[u].y : R.sg[u].x) >> (4 * g);
                    uint32_t e[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) e[j] = ((w << (15 - j)) & 0x80008000u) ^ nh;
                    A[u] = pg_half8(e[0], e[1], e[2], e[3]);
                }
#pragma unroll
                for (int rg = 0; rg < NR; ++rg)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        acc[rg][u] = pg_mfma(A[u], q_at(rg, L::kQSteps + s), acc[rg][u]);
                        if constexpr (HL) acc[rg][u] = pg_mfma(A[u], q_at(rg, L::kQSteps + 2 + s), acc[rg][u]);
                    }
            }
            if constexpr (HL) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float ni = R.nr[u][i] * cmul;
#pragma unroll
                        for (int rg = 0; rg < NR; ++rg) acc[rg][u][i] *= ni;
                    }
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            half8_t A[2], Al[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t kw[4] = {R.k[u].x, R.k[u].y, R.k[u].z, R.k[u].w};
                if constexpr (HL) four_pairs(kw[s], A[u], Al[u]);
                else A[u] = four_bytes(kw[s]);
            }
#pragma unroll
            for (int rg = 0; rg < NR; ++rg)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    acc[rg][u] = pg_mfma(A[u], q_at(rg, s), acc[rg][u]);
                    if constexpr (HL) {                     // without remainder times remainder, 2^-24 of it
                        acc[rg][u] = pg_mfma(A[u], q_at(rg, 4 + s), acc[rg][u]);
                        acc[rg][u] = pg_mfma(Al[u], q_at(rg, s), acc[rg][u]);
                    }
                }
        }
    };
    // bf16 calls: the signs' part of tokens whose norm lies beyond 65504 of the
    // table's unit, the norm less a power of two in fp16 and the sums times that;
    // the other tokens of the tile add 0 and keep their bits.  From memory again,
    // so that nothing waits in registers for what a calibrated cache does not
    // hold (two comparisons a tile: 64 rows 1 to 4 %, 32 rows at two blocks a CU
    // 2 to 3 %, others up to 1 %; with both ways inside `scores` 48 rows 7 %).
    auto large_signs = [&](const uint32_t (&r)[2], float4_t (&acc)[NR][2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint2 sg = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(half_of(a.k_qjl, r[u], 8), 8 * n, 0, 0));
            const float x = -cmul * __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(half_of(a.k_norms, r[u], 4), 4 * n, 0, 0));
            const bool over = fabsf(x) > 65504.0f;
            const int e = over ? __builtin_amdgcn_frexp_expf(x) - 15 : 0;
            const float m = over ? __builtin_amdgcn_ldexpf(x, -e) : 0.0f;
            const uint32_t nh = pg_pack(m, m);
            half8_t A[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t w = (s ? sg.y : sg.x) >> (4 * g);
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = ((w << (15 - j)) & 0x80008000u) ^ nh;
                A[s] = pg_half8(h[0], h[1], h[2], h[3]);
            }
            int ei[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ei[i] = __shfl(e, 4 * g + i);
#pragma unroll
            for (int rg = 0; rg < NR; ++rg) {
                float4_t t = pg_mfma(A[0], q_at(rg, L::kQSteps), float4_t{0.f, 0.f, 0.f, 0.f});
                t = pg_mfma(A[1], q_at(rg, L::kQSteps + 1), t);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[rg][u][i] += __builtin_amdgcn_ldexpf(t[i], ei[i]);
            }
        }
    };
    // Masks, and a row's reference m_run raised where some lane's maximum passes
    // it by 2^13, to 2^8 below that maximum: P reaches 2^13 (2^15 with the
    // roundings of scores below 2^25, base 2), near fp16's 65504, so that it
    // loses the weights below 2^-33 of the largest and rounds those below 2^-22
    // of it as subnormals.  (With the maximum itself as the reference, weights
    // below 2^-25 were lost: 16384 of them a wave beside one key, 2.5 half steps
    // of an fp16 output.)  m_run is the same in a row's four lane groups: each
    // lane tests its own maximum, and the row's is formed only where one does.
    auto settle = [&](float4_t (&acc)[NR][2], int64_t tile, int v) {
        const int nv[2] = {v & 255, v >> 8};
        if (!(v == 16 * 257 && (BLOCKS || (tile + 1) * kPgTile <= li.base))) {
#pragma unroll
            for (int rg = 0; rg < NR; ++rg) {
                const uint64_t sees = BLOCKS ? 0u : sees_l[16 * rg + n];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = 4 * g + i;
                        bool vis = tok < nv[u];
                        if constexpr (!BLOCKS) {
                            const int64_t j = tile * kPgTile + 16 * u + tok - li.base;
                            vis = vis && (j < 0 || ((sees >> (j & 63)) & 1u));
                        }
                        acc[rg][u][i] = vis ? acc[rg][u][i] : -INFINITY;
                    }
            }
        }
        float mt[NR];
        bool any = false;
#pragma unroll
        for (int rg = 0; rg < NR; ++rg) {
            mt[rg] = pg_max3(pg_max3(acc[rg][0][0], acc[rg][0][1], acc[rg][0][2]), pg_max3(acc[rg][0][3], acc[rg][1][0], acc[rg][1][1]),
                             __builtin_elementwise_maximum(acc[rg][1][2], acc[rg][1][3])) * csc[rg];
            any = any || mt[rg] > m_run[rg] + kLag;
        }
        if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
            for (int rg = 0; rg < NR; ++rg) {
                mt[rg] = pg_max_groups(mt[rg]);
                const float to = mt[rg] > m_run[rg] + kLag ? mt[rg] - kBelow : m_run[rg];
                const float f = __builtin_amdgcn_exp2f(m_run[rg] - to);
                m_run[rg] = to;
                l_run[rg] *= f;
#pragma unroll
                for (int k = 0; k < 8; ++k) oacc[rg][k] *= f;
            }
        }
    };
    // P and its sums.  Exponents are formed from the raw scores: m_run's own
    // rounding cancels between numerator and denominator.
    auto weights = [&](const float4_t (&acc)[NR][2], half8_t (&pb)[NR][2]) {
#pragma unroll
        for (int rg = 0; rg < NR; ++rg)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t p[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    p[k] = pg_pack(__builtin_amdgcn_exp2f(__builtin_fmaf(acc[rg][u][2 * k], csc[rg], -m_run[rg])),
                                   __builtin_amdgcn_exp2f(__builtin_fmaf(acc[rg][u][2 * k + 1], csc[rg], -m_run[rg])));
                    l_run[rg] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, p[k]), ones, l_run[rg], false);
                }
                pb[rg][u] = pg_half8(p[0], p[0], p[1], p[1]);       // against centroids and remainders
            }
    };
    auto products = [&](const uint32_t (&ev)[4], const uint32_t (&od)[4], const half8_t (&pb)[NR][2]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {                       // dims 8 m + k
            const uint32_t (&w)[4] = k & 1 ? od : ev;
            half8_t A[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) A[u] = two_bytes(w[2 * u], k >> 1, w[2 * u + 1], k >> 1);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int rg = 0; rg < NR; ++rg) oacc[rg][k] = pg_mfma(A[u], pb[rg][u], oacc[rg][k]);
        }
    };
    // two tokens' codes of one dim as one table byte: even dims, odd dims
    auto pair_codes = [&](const PgValues &V, uint32_t (&ev)[4], uint32_t (&od)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t va = V.v[2 * j], vb = V.v[2 * j + 1];
            ev[j] = ((vb << 4) & 0xF0F0F0F0u) | (va & 0x0F0F0F0Fu);
            od[j] = (vb & 0xF0F0F0F0u) | ((va >> 4) & 0x0F0F0F0Fu);
        }
    };
    if (cnt > 0) {
        const int64_t t0 = t_begin + wave;
        uint32_t r[2];
        int next;
        rows_at(0, r, next);                     // of the tile at hand (kept from above, two row groups spill more)
        half8_t pb[NR][2];
        uint32_t ev[4], od[4];
        // The next tile is asked for as its registers come free (two tiles
        // ahead: 54 instead of 51 us at 16 rows).  Waves in a matrix phase
        // issue first: of a SIMD's, others then work on their weights (without:
        // 56 instead of 54 us, 127 instead of 125 at 64 rows).
        // As a function of its operands: written out in the loop, 64 rows spill
        // more (now 3 to 5 registers with signs) and 48 and 64 take 2 to 5 % longer.
        auto step = [&](PgKeys<HL> &K, PgValues &V, int &nv, int k) {
            float4_t S[NR][2];
            const uint32_t now[2] = {r[0], r[1]};
            uint64_t large = 0;
            rows_at(clamp(k + 1), r, next);
            __builtin_amdgcn_s_setprio(1);
            scores(K, S, large);
            __builtin_amdgcn_s_setprio(0);
            load_k(K, r);
            if constexpr (QJL && !HL) {
                if (large) large_signs(now, S);
            }
            settle(S, t0 + (int64_t)NW * k, nv);
            nv = next;
            weights(S, pb);
            pair_codes(V, ev, od);
            load_v(V, r);
            __builtin_amdgcn_s_setprio(1);
            products(ev, od, pb);
            __builtin_amdgcn_s_setprio(0);
        };
        for (int k = 0; k < cnt; ++k) step(K, V, nv, k);
    }

    // ── merge of the waves ────────────────────────────────────────────
    // Every wave scales its O by 2^(m - the row's largest m) and adds up the
    // row's sum; the slabs are then summed.
    const bool wave_bad = __builtin_amdgcn_ballot_w64(page_bad) != 0;
    const int64_t mine = t_end - t_begin;
    const int act = mine < 1 ? 1 : mine < NW ? (int)mine : NW;      // waves with tiles
    float *slab = reinterpret_cast<float *>(smem);
    float *m_l = reinterpret_cast<float *>(smem + L::kMoved + L::kM), *l_l = m_l + NR * 16 * NW;
    float *flags = reinterpret_cast<float *>(smem + L::kMoved + L::kFlags);
#pragma unroll
    for (int rg = 0; rg < NR; ++rg) {
        const float l = pg_sum_groups(l_run[rg]);
        if (g == 0) {
            m_l[(rg * 16 + n) * NW + wave] = m_run[rg];
            l_l[(rg * 16 + n) * NW + wave] = l;
        }
    }
    if (lane == 0) flags[wave] = wave_bad ? 1.0f : 0.0f;
    __syncthreads();                                               // and the tables are done with
    float row_l[NR];
    float nan = li.bad ? 1.0f : 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(flags + w);
        nan += (f.x + f.y) + (f.z + f.w);
    }
#pragma unroll
    for (int rg = 0; rg < NR; ++rg) {
        float4 mw[NW / 4], lw[NW / 4];
#pragma unroll
        for (int w = 0; w < NW / 4; ++w) {
            mw[w] = *reinterpret_cast<const float4 *>(m_l + (rg * 16 + n) * NW + 4 * w);
            lw[w] = *reinterpret_cast<const float4 *>(l_l + (rg * 16 + n) * NW + 4 * w);
        }
        float m = -__FLT_MAX__;
#pragma unroll
        for (int w = 0; w < NW / 4; ++w) m = fmaxf(m, fmaxf(fmaxf(mw[w].x, mw[w].y), fmaxf(mw[w].z, mw[w].w)));
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW / 4; ++w) {
            l = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w].x - m), lw[w].x, l);
            l = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w].y - m), lw[w].y, l);
            l = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w].z - m), lw[w].z, l);
            l = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w].w - m), lw[w].w, l);
        }
        row_l[rg] = nan != 0.0f ? __builtin_nanf("") : l;
        const float f = __builtin_amdgcn_exp2f(m_run[rg] - m);
#pragma unroll
        for (int k = 0; k < 8; ++k) oacc[rg][k] *= f;
        m_run[rg] = m;
    }
    __syncthreads();                                               // m_l and l_l are read
    if (wave == 0 && g == 0) {
#pragma unroll
        for (int rg = 0; rg < NR; ++rg) {
            m_l[rg * 16 + n] = m_run[rg];
            l_l[rg * 16 + n] = row_l[rg];
        }
    }
#pragma unroll
    for (int r0 = 0; r0 < NR; r0 += L::MR) {
        if (r0) __syncthreads();                                   // the last slabs are read
        if ((chunk * NR + r0) * 16 >= a.rows) break;               // block-uniform
        if (wave < act) {
#pragma unroll
            for (int rg = r0; rg < r0 + L::MR; ++rg) {
                float *dst = slab + ((wave * L::MR + rg - r0) * 16 + n) * kPartRow;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 *d4 = reinterpret_cast<float4 *>(dst + 8 * (4 * g + i));
                    d4[0] = make_float4(oacc[rg][0][i], oacc[rg][1][i], oacc[rg][2][i], oacc[rg][3][i]);
                    d4[1] = make_float4(oacc[rg][4][i], oacc[rg][5][i], oacc[rg][6][i], oacc[rg][7][i]);
                }
            }
        }
        __syncthreads();
        for (int e = tid; e < L::MR * 16 * 32; e += 64 * NW) {
            const int r = e >> 5, d = 4 * (e & 31);
            const int rho = (chunk * NR + r0) * 16 + r;
            if (rho >= a.rows) break;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w)
                if (w < act) {                                     // uniform
                    const float4 v = *reinterpret_cast<const float4 *>(slab + (w * L::MR * 16 + r) * kPartRow + d);
                    o.x += v.x;
                    o.y += v.y;
                    o.z += v.z;
                    o.w += v.w;
                }
            const float m = m_l[r0 * 16 + r], l = l_l[r0 * 16 + r];
            const int t = BLOCKS ? li.t : (int)pg_div((uint32_t)rho, a.g_magic);
            if (a.splits == 1) {
                const int hq = hk * a.G + (BLOCKS ? rho : rho - t * a.G);
                const float s = cdiv / l;
                float v[4] = {o.x * s, o.y * s, o.z * s, o.w * s};
                uint16_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!BLOCKS && !li.bad && t >= li.nd) v[i] = 0.0f;
                    h[i] = HL ? f32_to_f16_rne(v[i]) : f32_to_bf16_rne(v[i]);
                }
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + ((li.b * a.Hq + hq) * a.T + t) * 128 + d) =
                    make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
            } else {
                float *p = a.ws + (((int64_t)unit * a.splits + split) * a.rows + rho) * kPartRow;
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
// loads in flight (2 x 8 lists of 256 rows in four splits 5.7 us, 64 lists of
// four rows in four 4.6: a launch and two round trips).
template <bool F16, bool BLOCKS>
__global__ __launch_bounds__(256) void page_merge_kernel(PageAttnArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d = 4 * (threadIdx.x & 31);
    if (row >= a.units * a.rows) return;
    const int64_t unit = row / a.rows;
    const int rho = (int)(row - unit * a.rows);
    PgList li = pg_list<BLOCKS>(a, (uint32_t)unit);
    pg_length<BLOCKS>(a, li);
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
    const int t = BLOCKS ? li.t : (int)pg_div((uint32_t)rho, a.g_magic);
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
    bool wide;                   // one row group: twelve waves, one block a CU
    bool pair;                   // two row groups: two blocks a CU
    size_t ws;
};

// Row groups per block and splits of a call, the cheapest by this estimate:
// `units` lists of at most `tiles` tiles, `rows` query rows each.  More rows a
// block share its table and the looked-up operands; fewer leave less of the
// last block empty and fill more CUs.  Measured, lists of 8192 tokens: 64 rows
// in fp16 187 us as one block each, 295 as four; lists of 20,011 tokens with
// 264 rows 179 us as six blocks of 48, 205 as five of 64.  One row group: twelve
// waves where every block has a CU to itself and a long list (256 lists of
// 8192 tokens 51 us, eight waves 59), else eight, two blocks a CU, so that one's
// prologue runs beside the other's tiles (768 lists of 75 to 2917 tokens in
// fp16 55 us, twelve waves 59; 312 selections of 768 tokens 17, 21 with one
// block a CU; 256 lists of 1024 tokens 13 either way, twelve waves 14).  Two
// row groups spill at two blocks a CU (57 registers of a bf16 call with signs, 22
// without): that pays up to four tiles a list (512 lists in tables of 80, 112,
// 144 and 176 tokens 15.8, 17.5, 19.5 and 22.0 us, with one block a CU 17.9,
// 18.3, 18.4 and 19.7).
static PagePlan page_plan(int64_t units, int rows, int64_t tiles, bool hl) {
    // us: a block's fixed part, and per tile by its row groups
    constexpr double kFixed = 8.0, kTile[5] = {0.0, 0.18, 0.27, 0.36, 0.46}, kTileHl[5] = {0.0, 0.24, 0.36, 0.53, 0.70};
    const int64_t cus = device_cus();
    PagePlan p{1, 1, 1, false, false, 0};
    double best = 1e30;
    for (int nr = 1; nr <= 4; ++nr) {
        const int chunks = (rows + 16 * nr - 1) / (16 * nr);
        const int64_t blocks = units * chunks;
        auto consider = [&](int64_t s) {
            if (s < 1 || s > 256 || (s > 1 && tiles / s < 8)) return;
            const int64_t all = blocks * s, n = (tiles + s - 1) / s;
            const bool spills = nr == 2 && !hl && all > cus && n <= 4;
            const int64_t at_once = (nr == 1 && all > cus) || spills ? 2 : 1;
            const double tile = spills ? 1.0 : (hl ? kTileHl : kTile)[nr] * (at_once == 2 ? 2.1 : 1.0);
            const double t = (double)((all + at_once * cus - 1) / (at_once * cus)) * ((spills ? 12.0 : kFixed) + tile * (double)n) +
                             (s > 1 ? 3.0 + 0.03 * (double)s + (double)units * (double)s * rows * kPartRow * 4e-6 * 2 / 3.5 : 0.0);
            if (t < best) {
                best = t;
                p.nr = nr;
                p.chunks = chunks;
                p.splits = (int)s;
                p.pair = spills;
            }
        };
        consider(1);
        for (int r = 1; r <= 4; ++r)
            for (int k = 0; k < 3; ++k) consider(r * cus / (blocks << k));
    }
    p.wide = p.nr == 1 && units * p.chunks * p.splits <= cus && tiles / p.splits >= 64;
    p.ws = p.splits > 1 ? (size_t)units * p.splits * rows * kPartRow * 4 : 0;
    return p;
}

template <int NR, bool HL, bool BLOCKS, int NW, bool PAIR>
static void page_launch(const PageAttnArgs &a, bool qjl, hipStream_t s) {
    const dim3 grid(8u * (unsigned)a.chunks, (unsigned)a.splits, (unsigned)((a.units + 7) / 8));
    if (qjl) hipLaunchKernelGGL((page_attn_kernel<NR, true, HL, BLOCKS, NW, PAIR>), grid, dim3(64 * NW), 0, s, a);
    else hipLaunchKernelGGL((page_attn_kernel<NR, false, HL, BLOCKS, NW, PAIR>), grid, dim3(64 * NW), 0, s, a);
}

template <bool HL, bool BLOCKS>
static void page_launch(const PageAttnArgs &a, bool qjl, const PagePlan &p, hipStream_t s) {
    if constexpr (!HL) {
        if (p.pair) return page_launch<2, false, BLOCKS, 8, true>(a, qjl, s);
    }
    if (p.wide) page_launch<1, HL, BLOCKS, 12, false>(a, qjl, s);
    else if (p.nr == 1) page_launch<1, HL, BLOCKS, 8, true>(a, qjl, s);
    else if (p.nr == 2) page_launch<2, HL, BLOCKS, 8, false>(a, qjl, s);
    else if (p.nr == 3) page_launch<3, HL, BLOCKS, 8, false>(a, qjl, s);
    else page_launch<4, HL, BLOCKS, 8, false>(a, qjl, s);
}

template <bool BLOCKS>
static int page_run(PageAttnArgs &a, int q_dtype, bool qjl, const PagePlan &p, hipStream_t s) {
    const bool hl = q_dtype == OMNI_F16;
    if (hl) page_launch<true, BLOCKS>(a, qjl, p, s);
    else page_launch<false, BLOCKS>(a, qjl, p, s);
    OMNI_CHECK_LAUNCH("page_attn_kernel");
    if (a.splits > 1) {
        const unsigned blocks = (unsigned)((a.units * a.rows + 7) / 8);
        if (hl) hipLaunchKernelGGL((page_merge_kernel<true, BLOCKS>), dim3(blocks), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((page_merge_kernel<false, BLOCKS>), dim3(blocks), dim3(256), 0, s, a);
        OMNI_CHECK_LAUNCH("page_merge_kernel");
    }
    return OMNI_OK;
}

// (b, t, kv head): eight times the 65535 groups that a grid's z holds; times
// 4096 kv heads or 64 tokens below 2^32, for pg_div
constexpr int64_t kMostUnits = 524280;

// What a workspace size may be asked of; a call checks the rest.
static bool page_sizes(int64_t B, int Hq, int Hkv, int64_t T, int64_t pages, int page_size) {
    return B > 0 && Hkv > 0 && Hkv <= 4096 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 1024 && T > 0 && T <= 64 &&
           B <= kMostUnits / Hkv / T && page_size >= 16 && pages > 0 && pages <= (int64_t(1) << 30) / page_size;
}

static uint64_t magic(int64_t d) { return (uint64_t(1) << 32) / (uint64_t)d + 1; }

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
    OMNI_CHECK_ARG(Hkv <= 4096 && B <= kMostUnits / Hkv / T, "%s: at most 4096 kv heads and B * T * n_kv_heads at most %lld", who,
                   (long long)kMostUnits);
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
    if (!page_sizes(B, Hq, Hkv, T, max_pages, page_size)) return 0;
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
                   per_head_codebook, Hq, Hkv, G, (int)T, (int)T * G, p.chunks, p.splits, 0, rotate_q, magic(Hkv), magic(T), magic(G),
                   (float)((double)scale * 1.4426950408889634), (float)(sqrt(2.0 / M_PI) / 128.0), inv_sqrt_dim_f32(128)};
    return page_run<false>(a, q_dtype, with_qjl != 0, p, as_stream(stream));
}

extern "C" size_t omni_attn_blocks_workspace_size(int64_t B, int Hq, int Hkv, int64_t T, int top, int page_size, int q_dtype) {
    if (!page_sizes(B, Hq, Hkv, T, top, page_size)) return 0;
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
                   per_head_codebook, Hq, Hkv, G, (int)T, G, p.chunks, p.splits, top, rotate_q, magic(Hkv), magic(T), magic(G),
                   (float)((double)scale * 1.4426950408889634), (float)(sqrt(2.0 / M_PI) / 128.0), inv_sqrt_dim_f32(128)};
    return page_run<true>(a, q_dtype, with_qjl != 0, p, as_stream(stream));
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
