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
// are left out), in whole numbers: Q and the head's centroids are each
// multiplied by the power of two that brings their largest into [64, 128) and
// rounded to int8.  A sum of 256 products of int8 lies below 2^22, so it does
// not depend on its order; equal scores are equal, and the lower block wins.
// Q+ and Q- are summed in fp64, where sums of 16-bit values are exact (the
// rotation's too: its factor 1/sqrt(128) does not change the order).
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
    int Hkv, page_shift;
};

// One block per (sequence, page that holds a token of [start, end)): a wave
// per head; lane (c, k) reads code bytes 4 c .. + 3 of tokens k, k + 4, ...
// and keeps nibble minima and maxima in 16-bit lanes.  The page's first tokens
// up to `end` count, whatever start is, so what a page says does not depend on
// how it was filled.  Bound by latency where a decode step touches a page per
// sequence, else by the read of the codes.
__global__ __launch_bounds__(256) void block_bounds_kernel(BoundsArgs a) {
    typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
    const int64_t b = blockIdx.y;
    const int64_t cap = a.max_pages << a.page_shift;
    int64_t s = a.start[b], e = a.end ? (int64_t)a.end[b] : s + a.count;
    if (a.kept) {
        // up to the last kept token; the page of the token before them, which
        // the dropped ones may have widened, also where none is kept
        e = s;
        for (int j = 0; j < a.count; ++j) e = a.kept[b * a.count + j] >= 0 ? s + j + 1 : e;
        --s;
    }
    s = s < 0 ? 0 : s;                           // rows outside the table are not written by an append either
    e = e > cap ? cap : e;
    if (s >= e) return;
    const int64_t pi = (s >> a.page_shift) + blockIdx.x;
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
    int32_t *scores;             // [(b T + t) Hkv + hk][max_pages]
    int32_t *blocks;             // (B, Hkv, T, top)
    int64_t max_pages, n_pages;
    int page_shift, per_head, Hq, Hkv, G, T, top, first, recent, rotate, f16;
    int per_block;               // blocks scored by one thread block
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

// Four codes (one a byte) to four int8 centroids from the 16-byte table t.
__device__ __forceinline__ uint32_t four_centroids(uint32_t codes, const uint32_t (&t)[4]) {
    const uint32_t sel = codes & 0x07070707u;
    const uint32_t low = __builtin_amdgcn_perm(t[1], t[0], sel), high = __builtin_amdgcn_perm(t[3], t[2], sel);
    // selectors 12 and 13 give the bytes 0x00 and 0xff
    const uint32_t up = __builtin_amdgcn_perm(0u, 0u, ((codes >> 3) & 0x01010101u) | 0x0C0C0C0Cu);
    return (low & ~up) | (high & up);
}

struct ScoreLds {
    double part[4][256];
    double most[4];
    int8_t q[256];               // Q+, then -Q-
    int8_t cent[16];
};

// Q+ and -Q- of query (b, t)'s heads hk G .. + G - 1 and the centroids, as
// int8, by the block's 256 threads.
__device__ __forceinline__ void whole_query(const SelectArgs &a, ScoreLds &sm, int64_t b, int t, int hk) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double qp[2] = {0.0, 0.0}, qn[2] = {0.0, 0.0};
    for (int h = wave; h < a.G; h += 4) {
        const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q) + ((b * a.Hq + hk * a.G + h) * a.T + t) * 128;
        const uint16_t u0 = src[lane], u1 = src[lane + 64];
        double x = a.f16 ? f16_to_f32(u0) : bf16_to_f32(u0), y = a.f16 ? f16_to_f32(u1) : bf16_to_f32(u1);
        if (a.rotate) {
            if (a.sign_flip) {
                x = a.sign_flip[lane] < 0 ? -x : x;
                y = a.sign_flip[lane + 64] < 0 ? -y : y;
            }
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const double px = __shfl_xor(x, m), py = __shfl_xor(y, m);
                x = lane & m ? px - x : x + px;
                y = lane & m ? py - y : y + py;
            }
            const double u = x, v = y;
            x = u + v;
            y = u - v;
        }
        qp[0] += fmax(x, 0.0);
        qn[0] += fmin(x, 0.0);
        qp[1] += fmax(y, 0.0);
        qn[1] += fmin(y, 0.0);
    }
    sm.part[wave][lane] = qp[0];
    sm.part[wave][lane + 64] = qp[1];
    sm.part[wave][128 + lane] = qn[0];
    sm.part[wave][192 + lane] = qn[1];
    __syncthreads();
    const double v = (sm.part[0][tid] + sm.part[1][tid]) + (sm.part[2][tid] + sm.part[3][tid]);
    double m = fabs(v);
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) m = fmax(m, __shfl_xor(m, k));
    if (lane == 0) sm.most[wave] = m;
    if (tid < 16) {
        const float *c = a.codebooks + (a.per_head ? hk * 16 : 0);
        double cm = 0.0;
        for (int k = 0; k < 16; ++k) cm = fmax(cm, fabs((double)c[k]));
        sm.cent[tid] = (int8_t)whole((double)c[tid] * whole_scale(cm));
    }
    __syncthreads();
    m = fmax(fmax(sm.most[0], sm.most[1]), fmax(sm.most[2], sm.most[3]));
    sm.q[tid] = (int8_t)whole(v * whole_scale(m));
    __syncthreads();
}

// Scores of the blocks between the first and the recent ones: eight lanes a
// block, 16 dims each.  Bound by the read of the bounds (128 B a block and
// head) where there are many, else by launch and the query's preparation.
__global__ __launch_bounds__(256) void block_score_kernel(SelectArgs a) {
    __shared__ ScoreLds sm;
    const int hk = blockIdx.y;
    const int64_t bt = blockIdx.z, b = bt / a.T;
    const int t = (int)(bt - b * a.T);
    const int64_t nb = seen_blocks(a, b, t);
    const int64_t from = a.first + (int64_t)blockIdx.x * a.per_block, to = nb - a.recent;
    if (nb <= a.top || from >= to) return;                       // block-uniform, before any barrier
    whole_query(a, sm, b, t, hk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 7;
    uint32_t qp[4], qn[4], tab[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        qp[j] = reinterpret_cast<const uint32_t *>(sm.q)[4 * c + j];
        qn[j] = reinterpret_cast<const uint32_t *>(sm.q)[32 + 4 * c + j];
        tab[j] = reinterpret_cast<const uint32_t *>(sm.cent)[j];
    }
    const int64_t end = from + a.per_block < to ? from + a.per_block : to;
    const int32_t *pt = a.page_table + b * a.max_pages;
    int32_t *out = a.scores + (bt * a.Hkv + hk) * a.max_pages;
    for (int64_t p0 = from + 8 * wave; p0 < end; p0 += 32) {
        const int64_t p = p0 + (lane >> 3);
        const int32_t id = p < end ? pt[p] : 0;
        const bool ok = id >= 0 && id < a.n_pages;
        const uint4 w4 = *reinterpret_cast<const uint4 *>(a.bounds + ((int64_t)(ok ? id : 0) * a.Hkv + hk) * 128 + 16 * c);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        int s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s = __builtin_amdgcn_sdot4((int)four_centroids((w[j] >> 4) & 0x0F0F0F0Fu, tab), (int)qp[j], s, false);
            s = __builtin_amdgcn_sdot4((int)four_centroids(w[j] & 0x0F0F0F0Fu, tab), (int)qn[j], s, false);
        }
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        s += __shfl_xor(s, 4);
        // a page outside the pool is selected first, so that its rows come out NaN
        if (c == 0 && p < end) out[p] = ok ? s : 0x7fffffff;
    }
}

// ── selection ───────────────────────────────────────────────────────────
//
// One block per (b, t, hk): the score that the last of `need` blocks has, by
// digits of eight bits from the top of the scores' range (a histogram in LDS
// per digit), then the blocks above it and the first ones equal to it in
// ascending order (a scan over the threads' consecutive shares).
constexpr int kPickThreads = 512;
constexpr int kPickLds = 12288;          // scores held in LDS; more are read again for every digit

__global__ __launch_bounds__(kPickThreads) void block_pick_kernel(SelectArgs a) {
    __shared__ uint32_t keys[kPickLds];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t wred[2][kPickThreads / 64];
    __shared__ uint32_t sh[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;                              // (b T + t) Hkv + hk
    const int64_t bt = row / a.Hkv, b = bt / a.T;
    const int hk = (int)(row - bt * a.Hkv), t = (int)(bt - b * a.T);
    const int64_t nb = seen_blocks(a, b, t);
    int32_t *out = a.blocks + ((b * a.Hkv + hk) * a.T + t) * a.top;
    if (nb <= a.top) {
        for (int i = tid; i < a.top; i += kPickThreads) out[i] = i < nb ? i : -1;
        return;
    }
    for (int i = tid; i < a.first + a.recent; i += kPickThreads)
        out[i < a.first ? i : a.top - a.recent + (i - a.first)] = (int32_t)(i < a.first ? i : nb - a.recent + (i - a.first));
    uint32_t need = (uint32_t)(a.top - a.first - a.recent);
    if (need == 0) return;                                       // uniform
    const int n = (int)(nb - a.first - a.recent);                // > need
    const int32_t *src = a.scores + row * a.max_pages + a.first;
    const bool held = n <= kPickLds;
    uint32_t kmin = 0xffffffffu, kmax = 0u;
    for (int i = tid; i < n; i += kPickThreads) {
        const uint32_t k = (uint32_t)src[i] ^ 0x80000000u;
        if (held) keys[i] = k;
        kmin = k < kmin ? k : kmin;
        kmax = k > kmax ? k : kmax;
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
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPickThreads / 64; ++w) {
        kmin = wred[0][w] < kmin ? wred[0][w] : kmin;
        kmax = wred[1][w] > kmax ? wred[1][w] : kmax;
    }
    auto key = [&](int i) { return (held ? keys[i] : (uint32_t)src[i] ^ 0x80000000u) - kmin; };
    // `prefix`: the digits found so far, the key's bits from `shift` up
    const uint32_t range = kmax - kmin;
    int shift = range ? 32 - __builtin_clz(range) : 0;
    uint32_t prefix = 0u;
    while (shift > 0) {
        const int low = shift > 8 ? shift - 8 : 0, width = shift - low;
        __syncthreads();                                         // hist and sh of the last digit are read
        if (tid < 256) hist[tid] = 0u;
        __syncthreads();
        for (int i = tid; i < n; i += kPickThreads) {
            const uint32_t x = key(i);
            if (shift >= 32 || x >> shift == prefix) atomicAdd(&hist[(x >> low) & ((1u << width) - 1u)], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
            uint32_t c[4], sum = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = hist[255 - 4 * lane - j];
                sum += c[j];
            }
            uint32_t incl = sum;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t up = __shfl_up(incl, m);
                incl += lane >= m ? up : 0u;
            }
            uint32_t above = incl - sum;
            if (above < need && need <= incl) {                   // one lane
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above < need && need <= above + c[j]) {
                        sh[0] = (prefix << width) | (uint32_t)(255 - 4 * lane - j);
                        sh[1] = need - above;
                        need = 0u;                                // found
                    }
                    above += c[j];
                }
            }
        }
        __syncthreads();
        prefix = sh[0];
        need = sh[1];
        shift = low;
    }
    // ── the blocks above `prefix`, and the first `need` equal to it ──
    const int each = (n + kPickThreads - 1) / kPickThreads, i0 = tid * each, i1 = i0 + each < n ? i0 + each : n;
    uint32_t gt = 0u, eq = 0u;
    for (int i = i0; i < i1; ++i) {
        const uint32_t x = key(i);
        gt += x > prefix ? 1u : 0u;
        eq += x == prefix ? 1u : 0u;
    }
    uint32_t igt = gt, ieq = eq;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t ug = __shfl_up(igt, m), ue = __shfl_up(ieq, m);
        igt += lane >= m ? ug : 0u;
        ieq += lane >= m ? ue : 0u;
    }
    __syncthreads();
    if (lane == 63) {
        wred[0][wave] = igt;
        wred[1][wave] = ieq;
    }
    __syncthreads();
    uint32_t pg = igt - gt, pe = ieq - eq;
    for (int w = 0; w < wave; ++w) {
        pg += wred[0][w];
        pe += wred[1][w];
    }
    for (int i = i0; i < i1; ++i) {
        const uint32_t x = key(i);
        const bool take = x > prefix || (x == prefix && pe < need);
        if (take) out[a.first + pg + (pe < need ? pe : need)] = a.first + i;
        pg += x > prefix ? 1u : 0u;
        pe += x == prefix ? 1u : 0u;
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
// not matter.  Four threads a token, 16 code bytes of K and V each.
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
    // pages that `count` tokens can touch (any number of tokens: the whole table)
    int64_t pages = end ? max_pages : (count + page_size - 2) / page_size + 1;
    if (pages > max_pages) pages = max_pages;
    const BoundsArgs a{k_nib, bounds, page_table, start, end, nullptr, max_pages, n_pages, count, Hkv, shift};
    hipLaunchKernelGGL(block_bounds_kernel, dim3((unsigned)pages, (unsigned)B), dim3(256), 0, as_stream(stream), a);
    OMNI_CHECK_LAUNCH("block_bounds_kernel");
    return OMNI_OK;
}

extern "C" size_t omni_block_select_workspace_size(int64_t B, int Hkv, int64_t T, int64_t max_pages, int top) {
    if (B <= 0 || Hkv <= 0 || T <= 0 || max_pages <= top) return 0;
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
                 q_dtype == OMNI_F16, 0};
    const int64_t rows = B * T * Hkv;
    if (ws) {
        // shares of 64 blocks at least, four thread blocks a CU
        int64_t per = (max_pages * rows + 4 * device_cus() - 1) / (4 * device_cus());
        per = per < 64 ? 64 : per > (1 << 20) ? 1 << 20 : (per + 31) / 32 * 32;
        a.per_block = (int)per;
        hipLaunchKernelGGL(block_score_kernel, dim3((unsigned)((max_pages + per - 1) / per), (unsigned)Hkv, (unsigned)(B * T)),
                           dim3(256), 0, as_stream(stream), a);
        OMNI_CHECK_LAUNCH("block_score_kernel");
    }
    hipLaunchKernelGGL(block_pick_kernel, dim3((unsigned)rows), dim3(kPickThreads), 0, as_stream(stream), a);
    OMNI_CHECK_LAUNCH("block_pick_kernel");
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
        const BoundsArgs ba{k_nib, bounds, page_table, positions, nullptr, kept, max_pages, n_pages, K, Hkv, shift};
        hipLaunchKernelGGL(block_bounds_kernel, dim3((unsigned)pages, (unsigned)B), dim3(256), 0, as_stream(stream), ba);
        OMNI_CHECK_LAUNCH("block_bounds_kernel");
    }
    return OMNI_OK;
}
