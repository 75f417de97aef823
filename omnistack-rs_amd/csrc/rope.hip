// Norm of query and key heads with the rotation by position, one pass (gfx950).
//
// For every token and head, x of D dims (no counterpart in the reference,
// whose queries and keys come rotated; kernels/hadamard.py:196-234 is the
// other rotation of the same tensors):
//   r = 1 / sqrt(mean_d x_d^2 + eps),   z_d = x_d r w_d      (z = x without weights)
//   y_i  = z_i cos t_i - z_i' sin t_i,  y_i' = z_i' cos t_i + z_i sin t_i
// over the R / 2 pairs (i, i') of the first R dims (i' = i + R / 2, or pairs of
// neighbours), y = z behind them; t_i = pos[axis_i] * freq_i.  The gradient is
// the same rotation by -t of dy, dz; with g = dz w
//   dx = r (g - x r^2 mean_d(g x)),   dw_d = sum over tokens and heads of dz_d x_d r.
//
// Angles: a frequency is held as a 64-bit fraction of a turn per position,
// round(freq / 2 pi * 2^64), so that the low 64 bits of the integer product
// with a position are the angle's fraction of a turn, the whole turns gone by
// overflow.  The product is exact; the frequency's rounding costs |position|
// 2^-65 turns, 2e-7 radians at 2^40, about what the fp32 cosine errs by, and 2e-4
// at 2^50 (a table of cosines would be 512 B a position at D = 128 and end at
// some length).  Its top 32 bits give the quadrant and a remainder within pi / 4,
// where Taylor polynomials of degree 9 and 10 err by less than 2e-9.
//
// Bound by memory: 2 x 2 B an element.  A wave takes a token (or some of its
// heads where tokens are few): a lane holds 16 B of a head, the wave's 64 lanes
// compute each of the token's angles once and pass them through LDS, and the
// pair's other half comes from the lane D / 2 away, in the input's own 16 bits
// and before the norm, whose factor both halves share.
//
// 32 + 8 heads of 128 in bf16: 65536 tokens 253 us, 5.3 TB/s, the rate of a copy
// of as many bytes (1.34 GB; HBM moves just those); 4096 tokens 17 us; 64 tokens
// 4.0 us, a chain of position, angles, LDS and one head.  Two heads' loads ahead
// instead of one, or four times the waves for 4096 tokens: no difference.
#include "omni_common.h"

namespace omni {

constexpr int kRpWaves = 4;
constexpr int kRpMaxPairs = 128;
constexpr int kRpBwdBlocks = 1024;      // at most; rows of partial weight gradients

struct RopeTensor {
    char *p;
    int64_t sb, st, sh;                 // strides in bytes (the last dim is contiguous)
};

struct RopeArgs {
    RopeTensor q, k, yq, yk;            // forward: x, y.  backward: x, dx
    RopeTensor gq, gk;                  // backward: dy
    const void *wq, *wk, *pos;
    const uint64_t *turns;
    const uint8_t *axes;
    float *partial;
    int64_t B, T, units;
    int64_t pa, pb, pt;                 // position strides in elements
    int Hq, Hkv, R, chunks, ppc, passes_q, passes;
    int w_dtype, pos64, inverse;
    float eps;
};

// ── lanes ───────────────────────────────────────────────────────────────

template <int CTRL>
__device__ __forceinline__ uint32_t rp_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

// The value of the lane whose number differs in bit M.
template <int M>
__device__ __forceinline__ uint32_t rp_xor(uint32_t x) {
    if constexpr (M == 1) return rp_dpp<0xB1>(x);                    // quad_perm [1, 0, 3, 2]
    else if constexpr (M == 2) return rp_dpp<0x4E>(x);               // quad_perm [2, 3, 0, 1]
    else if constexpr (M == 4) return rp_dpp<0x141>(rp_dpp<0x1B>(x));   // reversed in fours, then in eights
    else if constexpr (M == 8) return rp_dpp<0x128>(x);              // 8 on, in rows of 16
    else if constexpr (M == 16) {
        const auto t = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return (threadIdx.x & 16) ? t[0] : t[1];
    } else {
        const auto t = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return (threadIdx.x & 32) ? t[0] : t[1];
    }
}

// Sum over aligned groups of N lanes, in every lane.
template <int N>
__device__ __forceinline__ float rp_sum(float v) {
    if constexpr (N > 1) v += __uint_as_float(rp_xor<1>(__float_as_uint(v)));
    if constexpr (N > 2) v += __uint_as_float(rp_xor<2>(__float_as_uint(v)));
    if constexpr (N > 4) v += __uint_as_float(rp_dpp<0x141>(__float_as_uint(v)));   // all of a four are alike
    if constexpr (N > 8) v += __uint_as_float(rp_xor<8>(__float_as_uint(v)));
    if constexpr (N > 16) v += __uint_as_float(rp_xor<16>(__float_as_uint(v)));
    if constexpr (N > 32) v += __uint_as_float(rp_xor<32>(__float_as_uint(v)));
    return v;
}

// ── elements ────────────────────────────────────────────────────────────

template <int DT>
struct RpVec {
    static constexpr int E = DT == OMNI_F32 ? 4 : 8;   // elements in 16 bytes
    uint32_t u[4];
    __device__ __forceinline__ void load(const char *p) {
        const uint4 t = *reinterpret_cast<const uint4 *>(p);
        u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w;
    }
    __device__ __forceinline__ void store(char *p) const {
        *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __device__ __forceinline__ void zero() { u[0] = u[1] = u[2] = u[3] = 0; }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == OMNI_F32) return __uint_as_float(u[i]);
        const uint32_t w = u[i / 2];
        if constexpr (DT == OMNI_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
        else return f16_to_f32((uint16_t)(i & 1 ? w >> 16 : w));
    }
    __device__ __forceinline__ void put(const float (&v)[E]) {
        if constexpr (DT == OMNI_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(v[i]);
        } else if constexpr (DT == OMNI_BF16) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f2 t = {v[2 * i], v[2 * i + 1]};
                u[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, b2));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                u[i] = (uint32_t)f32_to_f16_rne(v[2 * i]) | (uint32_t)f32_to_f16_rne(v[2 * i + 1]) << 16;
        }
    }
};

// Weights d .. d + E - 1 (16-byte aligned, d a multiple of E).
template <int E>
__device__ __forceinline__ void rp_weights(const void *p, int dtype, int d, float (&w)[E]) {
    if (dtype == OMNI_F32) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 t = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + d + e);
            w[e] = t.x; w[e + 1] = t.y; w[e + 2] = t.z; w[e + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const uint2 t = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + d + e);
            const uint32_t u[2] = {t.x, t.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t h = (uint16_t)(i & 1 ? u[i / 2] >> 16 : u[i / 2]);
                w[e + i] = dtype == OMNI_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
            }
        }
    }
}

// cos and sin of `t` / 2^64 turns.
__device__ __forceinline__ void rp_angle(uint64_t t, float &c, float &s) {
    const uint32_t h = (uint32_t)(t >> 32);
    const uint32_t quad = (h + 0x20000000u) >> 30;
    const float a = (float)(int32_t)(h - (quad << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
    const float b = a * a;
    float sn = fmaf(b, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(b, sn, 8.3333333e-3f);
    sn = fmaf(b, sn, -1.6666667e-1f);
    sn = fmaf(a * b, sn, a);
    float cs = fmaf(b, -2.7557319e-7f, 2.4801587e-5f);
    cs = fmaf(b, cs, -1.3888889e-3f);
    cs = fmaf(b, cs, 4.1666667e-2f);
    cs = fmaf(b, cs, -0.5f);
    cs = fmaf(b, cs, 1.0f);
    const float x = quad & 1 ? sn : cs, y = quad & 1 ? cs : sn;
    c = (quad + 1) & 2 ? -x : x;
    s = quad & 2 ? -y : y;
}

// One lane's share of a head: its dims d0 .. d0 + E - 1, their weights and
// angles.  PAIR 0: halves of the whole head, 1: halves of its first R dims,
// 2: neighbours.
template <int DT, int D, int PAIR, bool NORM>
struct RpLane {
    static constexpr int E = RpVec<DT>::E, LPH = D / E, HPW = 64 / LPH;
    float c[E], s[E];                    // of each dim; s carries the pair's sign (neighbours: by pair)
    float w[E], wp[E];                   // own and partner's weights
    int sub, grp, d0, partner;
    bool turns;                          // its dims are among the first R

    __device__ __forceinline__ void place(const RopeArgs &a) {
        const int lane = threadIdx.x & 63;
        sub = lane % LPH;
        grp = lane / LPH;
        d0 = sub * E;
        turns = PAIR == 0 || d0 < a.R;
        partner = lane;
        if constexpr (PAIR == 1) {
            const int half = a.R / 2;
            if (d0 < half) partner = lane + half / E;
            else if (d0 < a.R) partner = lane - half / E;
        }
    }
    __device__ __forceinline__ int partner_dim(int half) const {
        return PAIR == 0 ? (d0 ^ (D / 2)) : PAIR == 1 ? (d0 < half ? d0 + half : d0 < 2 * half ? d0 - half : d0) : d0;
    }
    __device__ __forceinline__ void weights(const RopeArgs &a, const void *p) {
        if constexpr (!NORM) return;
        const int dp = partner_dim(a.R / 2);
        rp_weights(p, a.w_dtype, d0, w);
        rp_weights(p, a.w_dtype, dp, wp);
    }
    // The wave's angles of token (b, t), through cs / sn of LDS.
    __device__ __forceinline__ void angles(const RopeArgs &a, int64_t b, int64_t t, float *cs, float *sn) {
        const int lane = threadIdx.x & 63, half = a.R / 2;
        for (int i = lane; i < half; i += 64) {
            const int64_t at = a.axes[i] * a.pa + b * a.pb + t * a.pt;
            const int64_t p = a.pos64 ? static_cast<const int64_t *>(a.pos)[at] : static_cast<const int32_t *>(a.pos)[at];
            float co, si;
            rp_angle((uint64_t)p * a.turns[i], co, si);
            cs[i] = co;
            sn[i] = a.inverse ? -si : si;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (!turns) {                    // no pair: turn() leaves these dims
#pragma unroll
            for (int e = 0; e < E; ++e) { c[e] = 1.0f; s[e] = 0.0f; }   // as zeros they cost 12 bytes of scratch
        } else if constexpr (PAIR == 2) {
#pragma unroll
            for (int e = 0; e < E / 2; ++e) { c[e] = cs[d0 / 2 + e]; s[e] = sn[d0 / 2 + e]; }
        } else {
            const bool low = d0 < half;
            const int i0 = low ? d0 : d0 - half;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                c[e] = cs[i0 + e];
                s[e] = low ? -sn[i0 + e] : sn[i0 + e];
            }
        }
        // the next token's angles must not overtake these reads
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ RpVec<DT> other(const RpVec<DT> &x) const {
        RpVec<DT> o = x;
        if constexpr (PAIR == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.u[i] = rp_xor<LPH / 2>(x.u[i]);
        } else if constexpr (PAIR == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.u[i] = (uint32_t)__shfl((int)x.u[i], partner, 64);
        }
        return o;
    }
    // z rotated, z of the partner dims in zp (unused for neighbours).  Dims behind
    // R are selected, not turned by nothing: an infinity times a sine of 0 is NaN.
    __device__ __forceinline__ void turn(const float (&z)[E], const float (&zp)[E], float (&y)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (PAIR == 2) {
                const int i = e / 2;
                y[e] = e & 1 ? fmaf(z[e], c[i], z[e - 1] * s[i]) : fmaf(z[e], c[i], -z[e + 1] * s[i]);
            } else {
                y[e] = fmaf(z[e], c[e], zp[e] * s[e]);
            }
            if constexpr (PAIR != 0) y[e] = turns ? y[e] : z[e];
        }
    }
};

// ── forward (and the gradient without a norm: the inverse rotation) ─────

template <int DT, int D, int PAIR, bool NORM>
__device__ __forceinline__ void rp_forward_heads(const RopeArgs &a, RpLane<DT, D, PAIR, NORM> &L, const char *x, int64_t xs,
                                                 char *y, int64_t ys, int H, int p0, int p1) {
    using V = RpVec<DT>;
    constexpr int E = V::E, HPW = RpLane<DT, D, PAIR, NORM>::HPW, LPH = RpLane<DT, D, PAIR, NORM>::LPH;
    int h = p0 * HPW + L.grp;
    const int hend = min(H, p1 * HPW);
    // lanes behind the last head read none and store none, but stay for the exchanges
    const int rounds = p1 - p0;
    V nx;
    nx.zero();
    if (h < hend) nx.load(x + h * xs + L.d0 * (16 / E));
    for (int i = 0; i < rounds; ++i, h += HPW) {
        const V v = nx;
        if (h + HPW < hend) nx.load(x + (h + HPW) * xs + L.d0 * (16 / E));
        float z[E], zp[E], o[E];
        const V vp = L.other(v);
        if constexpr (NORM) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss = fmaf(v.get(e), v.get(e), ss);
            const float r = rsqrtf(fmaf(rp_sum<LPH>(ss), 1.0f / D, a.eps));
#pragma unroll
            for (int e = 0; e < E; ++e) {
                z[e] = v.get(e) * r * L.w[e];
                zp[e] = vp.get(e) * r * L.wp[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                z[e] = v.get(e);
                zp[e] = vp.get(e);
            }
        }
        L.turn(z, zp, o);
        V out;
        out.put(o);
        if (h < hend) out.store(y + h * ys + L.d0 * (16 / E));
    }
}

template <int DT, int D, int PAIR, bool NORM>
__global__ __launch_bounds__(64 * kRpWaves) void rope_kernel(RopeArgs a) {
    __shared__ float cs[kRpWaves][kRpMaxPairs], sn[kRpWaves][kRpMaxPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t unit = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kRpWaves + wave;
    if (unit >= a.units) return;
    const int64_t tok = unit / a.chunks;
    const int chunk = (int)(unit - tok * a.chunks);
    const int64_t b = tok / a.T, t = tok - b * a.T;
    const int p0 = chunk * a.ppc, p1 = min(p0 + a.ppc, a.passes);
    RpLane<DT, D, PAIR, NORM> L;
    L.place(a);
    L.angles(a, b, t, cs[wave], sn[wave]);
    if (p0 < a.passes_q) {
        L.weights(a, a.wq);
        rp_forward_heads(a, L, a.q.p + b * a.q.sb + t * a.q.st, a.q.sh, a.yq.p + b * a.yq.sb + t * a.yq.st, a.yq.sh, a.Hq,
                         p0, min(p1, a.passes_q));
    }
    if (p1 > a.passes_q) {
        L.weights(a, a.wk);
        rp_forward_heads(a, L, a.k.p + b * a.k.sb + t * a.k.st, a.k.sh, a.yk.p + b * a.yk.sb + t * a.yk.st, a.yk.sh, a.Hkv,
                         max(p0 - a.passes_q, 0), p1 - a.passes_q);
    }
}

// ── gradient with a norm ────────────────────────────────────────────────

template <int DT, int D, int PAIR>
__device__ __forceinline__ void rp_backward_heads(const RopeArgs &a, RpLane<DT, D, PAIR, true> &L, const char *x, int64_t xs,
                                                  const char *g, int64_t gs, char *y, int64_t ys, int H, int p0, int p1,
                                                  float (&dw)[RpVec<DT>::E]) {
    using V = RpVec<DT>;
    constexpr int E = V::E, HPW = RpLane<DT, D, PAIR, true>::HPW, LPH = RpLane<DT, D, PAIR, true>::LPH;
    int h = p0 * HPW + L.grp;
    const int hend = min(H, p1 * HPW), rounds = p1 - p0;
    V nx, ng;
    nx.zero();
    ng.zero();
    float own[E];                        // of this token: two short rows of additions err less than a long one
#pragma unroll
    for (int e = 0; e < E; ++e) own[e] = 0.0f;
    if (h < hend) {
        nx.load(x + h * xs + L.d0 * (16 / E));
        ng.load(g + h * gs + L.d0 * (16 / E));
    }
    for (int i = 0; i < rounds; ++i, h += HPW) {
        const bool live = h < hend;
        const V v = nx, u = ng;
        if (h + HPW < hend) {
            nx.load(x + (h + HPW) * xs + L.d0 * (16 / E));
            ng.load(g + (h + HPW) * gs + L.d0 * (16 / E));
        }
        const V up = L.other(u);
        float z[E], zp[E], dz[E];
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            z[e] = u.get(e);
            zp[e] = up.get(e);
            ss = fmaf(v.get(e), v.get(e), ss);
        }
        L.turn(z, zp, dz);
        const float r = rsqrtf(fmaf(rp_sum<LPH>(ss), 1.0f / D, a.eps));
        float xh[E], gx = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            xh[e] = v.get(e) * r;
            if (live) own[e] = fmaf(dz[e], xh[e], own[e]);
            dz[e] *= L.w[e];
            gx = fmaf(dz[e], xh[e], gx);
        }
        const float m = rp_sum<LPH>(gx) * (1.0f / D);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = r * fmaf(-m, xh[e], dz[e]);
        V out;
        out.put(o);
        if (live) out.store(y + h * ys + L.d0 * (16 / E));
    }
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] += own[e];
}

// Weight gradients: a lane's sums over its tokens and heads, the wave's lanes
// of one dim, the block's waves; a row of partial sums a block, summed by
// rope_dw_kernel in their order (the same on every run).  8192 tokens of 32 + 8
// heads of 128 in bf16: 48 us, 5.2 TB/s, and 4.0 us for the sums (20 with fewer
// threads a column).
template <int DT, int D, int PAIR>
__global__ __launch_bounds__(64 * kRpWaves) void rope_backward_kernel(RopeArgs a) {
    using V = RpVec<DT>;
    constexpr int E = V::E, LPH = D / E;
    __shared__ float cs[kRpWaves][kRpMaxPairs], sn[kRpWaves][kRpMaxPairs];
    __shared__ float red[kRpWaves][2][D];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    RpLane<DT, D, PAIR, true> L;
    L.place(a);
    float dwq[E], dwk[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dwq[e] = dwk[e] = 0.0f;
    for (int64_t unit = (int64_t)blockIdx.x * kRpWaves + wave; unit < a.units; unit += (int64_t)gridDim.x * kRpWaves) {
        const int64_t tok = unit / a.chunks;
        const int chunk = (int)(unit - tok * a.chunks);
        const int64_t b = tok / a.T, t = tok - b * a.T;
        const int p0 = chunk * a.ppc, p1 = min(p0 + a.ppc, a.passes);
        L.angles(a, b, t, cs[wave], sn[wave]);
        if (p0 < a.passes_q) {
            L.weights(a, a.wq);
            rp_backward_heads(a, L, a.q.p + b * a.q.sb + t * a.q.st, a.q.sh, a.gq.p + b * a.gq.sb + t * a.gq.st, a.gq.sh,
                              a.yq.p + b * a.yq.sb + t * a.yq.st, a.yq.sh, a.Hq, p0, min(p1, a.passes_q), dwq);
        }
        if (p1 > a.passes_q) {
            L.weights(a, a.wk);
            rp_backward_heads(a, L, a.k.p + b * a.k.sb + t * a.k.st, a.k.sh, a.gk.p + b * a.gk.sb + t * a.gk.st, a.gk.sh,
                              a.yk.p + b * a.yk.sb + t * a.yk.st, a.yk.sh, a.Hkv, max(p0 - a.passes_q, 0), p1 - a.passes_q, dwk);
        }
    }
    auto over_heads = [&](float v) {     // sum over the lanes of one dim
        if constexpr (LPH <= 4) v += __uint_as_float(rp_xor<4>(__float_as_uint(v)));
        if constexpr (LPH <= 8) v += __uint_as_float(rp_xor<8>(__float_as_uint(v)));
        if constexpr (LPH <= 16) v += __uint_as_float(rp_xor<16>(__float_as_uint(v)));
        if constexpr (LPH <= 32) v += __uint_as_float(rp_xor<32>(__float_as_uint(v)));
        return v;
    };
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float vq = over_heads(dwq[e]), vk = over_heads(dwk[e]);
        if (L.grp == 0) {
            red[wave][0][L.d0 + e] = vq;
            red[wave][1][L.d0 + e] = vk;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 64 * kRpWaves) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kRpWaves; ++w) v += red[w][i / D][i % D];
        a.partial[(int64_t)blockIdx.x * 2 * D + i] = v;
    }
}

// Columns of the partial sums: 64 threads a column, 16 columns a block, in 64
// bits (in 32 the two rows of additions left weight gradients of fp32 inputs
// with three times the error of their terms).
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float *partial, int rows, int D, int w_dtype, void *dwq, void *dwk) {
    __shared__ double red[64][17];
    const int col = blockIdx.x * 16 + threadIdx.x % 16, part = threadIdx.x / 16;
    double sum = 0.0;
#pragma unroll 8
    for (int r = part; r < rows; r += 64) sum += partial[(int64_t)r * 2 * D + col];
    red[part][threadIdx.x % 16] = sum;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int p = 1; p < 64; ++p) sum += red[p][threadIdx.x];
    const float v = (float)sum;
    void *out = col < D ? dwq : dwk;
    const int d = col < D ? col : col - D;
    if (w_dtype == OMNI_F32) static_cast<float *>(out)[d] = v;
    else static_cast<uint16_t *>(out)[d] = w_dtype == OMNI_BF16 ? f32_to_bf16_rne(v) : f32_to_f16_rne(v);
}

// ── host ────────────────────────────────────────────────────────────────

// A wave a token while there are tokens for two waves a SIMD, else its heads
// in as many parts as that takes (64 tokens of 40 heads, D = 128: 10 parts).
static void rope_split(RopeArgs &a, int D, int elems, int64_t tokens) {
    const int hpw = 64 / (D / elems);
    a.passes_q = (a.Hq + hpw - 1) / hpw;
    a.passes = a.passes_q + (a.Hkv + hpw - 1) / hpw;
    const int64_t want = 8 * (int64_t)device_cus();
    int64_t parts = (want + tokens - 1) / tokens;
    if (parts > a.passes) parts = a.passes;
    a.ppc = (int)((a.passes + parts - 1) / parts);
    a.chunks = (a.passes + a.ppc - 1) / a.ppc;
    a.units = tokens * a.chunks;
}

static int rope_tensor(const char *who, const char *what, const void *p, const int64_t *s, int size, RopeTensor &t) {
    OMNI_CHECK_ARG(p && s, "%s: NULL %s", who, what);
    OMNI_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0 &&
                       s[2] * size % 16 == 0,
                   "%s: %s and its strides must be multiples of 16 bytes", who, what);
    t.p = static_cast<char *>(const_cast<void *>(p));
    t.sb = s[0] * size;
    t.st = s[1] * size;
    t.sh = s[2] * size;
    return OMNI_OK;
}

static int rope_args(const char *who, int dtype, int64_t B, int64_t T, int Hq, int Hkv, int D, const void *positions,
                     int positions64, const int64_t *ps, const uint64_t *turns, const uint8_t *pair_axes, int rotary_dim,
                     const void *wq, const void *wk, int w_dtype, float eps, RopeArgs &a) {
    OMNI_CHECK_ARG(dtype_ok(dtype) && dtype_ok(w_dtype), "%s: bad dtype", who);
    OMNI_CHECK_ARG(D == 32 || D == 64 || D == 128 || D == 256, "%s: head_dim must be 32, 64, 128 or 256, got %d", who, D);
    OMNI_CHECK_ARG(B >= 0 && T >= 0 && Hq > 0 && Hkv > 0, "%s: bad shape", who);
    // far past any memory.  A token is cut into parts only where tokens are fewer than 8 a CU
    // (rope_split), so that units stay near 2^40
    OMNI_CHECK_ARG(Hq <= (1 << 24) && Hkv <= (1 << 24) && (T == 0 || B <= (int64_t(1) << 40) / T), "%s: shape too large", who);
    const int unit = dtype == OMNI_F32 ? 8 : 16;
    OMNI_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % unit == 0,
                   "%s: rotary_dim must be a multiple of %d up to head_dim, got %d", who, unit, rotary_dim);
    OMNI_CHECK_ARG((wq == nullptr) == (wk == nullptr), "%s: q and k weights go together", who);
    OMNI_CHECK_ARG((reinterpret_cast<uintptr_t>(wq) | reinterpret_cast<uintptr_t>(wk)) % 16 == 0,
                   "%s: weights must be 16-byte aligned", who);
    OMNI_CHECK_ARG(wq == nullptr || eps >= 0.0f, "%s: eps must be >= 0", who);
    if (B == 0 || T == 0) return OMNI_OK;
    OMNI_CHECK_ARG(rotary_dim == 0 || (positions && ps && turns && pair_axes), "%s: NULL positions or frequencies", who);
    a.pos = positions; a.pos64 = positions64;
    a.pa = ps ? ps[0] : 0; a.pb = ps ? ps[1] : 0; a.pt = ps ? ps[2] : 0;
    a.turns = turns; a.axes = pair_axes; a.R = rotary_dim;
    a.wq = wq; a.wk = wk; a.w_dtype = w_dtype; a.eps = eps;
    a.B = B; a.T = T; a.Hq = Hq; a.Hkv = Hkv;
    return OMNI_OK;
}

template <int DT, int D, int PAIR>
static void rope_launch_pair(const RopeArgs &a, bool backward, int blocks, hipStream_t st) {
    if (backward) {
        hipLaunchKernelGGL((rope_backward_kernel<DT, D, PAIR>), dim3(blocks), dim3(64 * kRpWaves), 0, st, a);
        return;
    }
    // fewer than 2^32 threads in a dimension
    const int64_t n = (a.units + kRpWaves - 1) / kRpWaves, gx = n < (1 << 22) ? n : (1 << 22);
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));
    if (a.wq) hipLaunchKernelGGL((rope_kernel<DT, D, PAIR, true>), grid, dim3(64 * kRpWaves), 0, st, a);
    else hipLaunchKernelGGL((rope_kernel<DT, D, PAIR, false>), grid, dim3(64 * kRpWaves), 0, st, a);
}

template <int DT, int D>
static void rope_launch_dim(const RopeArgs &a, int pair, bool backward, int blocks, hipStream_t st) {
    if (pair == 0) rope_launch_pair<DT, D, 0>(a, backward, blocks, st);
    else if (pair == 1) rope_launch_pair<DT, D, 1>(a, backward, blocks, st);
    else rope_launch_pair<DT, D, 2>(a, backward, blocks, st);
}

template <int DT>
static void rope_launch_dtype(const RopeArgs &a, int D, int pair, bool backward, int blocks, hipStream_t st) {
    switch (D) {
        case 32: rope_launch_dim<DT, 32>(a, pair, backward, blocks, st); break;
        case 64: rope_launch_dim<DT, 64>(a, pair, backward, blocks, st); break;
        case 128: rope_launch_dim<DT, 128>(a, pair, backward, blocks, st); break;
        default: rope_launch_dim<DT, 256>(a, pair, backward, blocks, st); break;
    }
}

static void rope_launch(const RopeArgs &a, int dtype, int D, int interleaved, bool backward, int blocks, hipStream_t st) {
    // halves of a part of the head, or no rotation: the exchange between any two lanes
    const int pair = interleaved ? 2 : a.R == D ? 0 : 1;
    if (dtype == OMNI_F32) rope_launch_dtype<OMNI_F32>(a, D, pair, backward, blocks, st);
    else if (dtype == OMNI_F16) rope_launch_dtype<OMNI_F16>(a, D, pair, backward, blocks, st);
    else rope_launch_dtype<OMNI_BF16>(a, D, pair, backward, blocks, st);
}

}  // namespace omni

using namespace omni;

extern "C" int omni_qk_norm_rope(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, int dtype,
                                 int64_t B, int64_t T, int Hq, int Hkv, int head_dim, const void *positions, int positions64,
                                 const int64_t *position_strides, const uint64_t *turns, const uint8_t *pair_axes,
                                 int rotary_dim, int interleaved, const void *q_weight, const void *k_weight, int w_dtype,
                                 float eps, void *q_out, const int64_t *q_out_strides, void *k_out,
                                 const int64_t *k_out_strides, void *stream) {
    const char *who = "omni_qk_norm_rope";
    RopeArgs a = {};
    OMNI_TRY(rope_args(who, dtype, B, T, Hq, Hkv, head_dim, positions, positions64, position_strides, turns, pair_axes,
                       rotary_dim, q_weight, k_weight, w_dtype, eps, a));
    if (B == 0 || T == 0) return OMNI_OK;
    const int size = dtype_size(dtype);
    OMNI_TRY(rope_tensor(who, "q", q, q_strides, size, a.q));
    OMNI_TRY(rope_tensor(who, "k", k, k_strides, size, a.k));
    OMNI_TRY(rope_tensor(who, "q_out", q_out, q_out_strides, size, a.yq));
    OMNI_TRY(rope_tensor(who, "k_out", k_out, k_out_strides, size, a.yk));
    rope_split(a, head_dim, 16 / size, B * T);
    rope_launch(a, dtype, head_dim, interleaved, false, 0, as_stream(stream));
    OMNI_CHECK_LAUNCH(who);
    return OMNI_OK;
}

extern "C" size_t omni_qk_norm_rope_backward_workspace_size(int head_dim) {
    return head_dim > 0 ? (size_t)kRpBwdBlocks * 2 * (size_t)head_dim * sizeof(float) : 0;
}

extern "C" int omni_qk_norm_rope_backward(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides,
                                          int dtype, int64_t B, int64_t T, int Hq, int Hkv, int head_dim,
                                          const void *positions, int positions64, const int64_t *position_strides,
                                          const uint64_t *turns, const uint8_t *pair_axes, int rotary_dim, int interleaved,
                                          const void *q_weight, const void *k_weight, int w_dtype, float eps,
                                          const void *dq_out, const int64_t *dq_out_strides, const void *dk_out,
                                          const int64_t *dk_out_strides, void *dq, const int64_t *dq_strides, void *dk,
                                          const int64_t *dk_strides, void *dq_weight, void *dk_weight, void *workspace,
                                          size_t workspace_bytes, void *stream) {
    const char *who = "omni_qk_norm_rope_backward";
    RopeArgs a = {};
    OMNI_TRY(rope_args(who, dtype, B, T, Hq, Hkv, head_dim, positions, positions64, position_strides, turns, pair_axes,
                       rotary_dim, q_weight, k_weight, w_dtype, eps, a));
    const int size = dtype_size(dtype);
    hipStream_t st = as_stream(stream);
    const bool norm = q_weight != nullptr, empty = B == 0 || T == 0;
    int blocks = 0;
    if (norm) {
        OMNI_CHECK_ARG(dq_weight && dk_weight, "%s: NULL weight gradient", who);
        if (!empty && (!workspace || workspace_bytes < omni_qk_norm_rope_backward_workspace_size(head_dim))) {
            set_error("%s: workspace of %zu bytes needed", who, omni_qk_norm_rope_backward_workspace_size(head_dim));
            return OMNI_EWORKSPACE;
        }
    }
    if (!empty) {
        RopeTensor gq, gk;
        OMNI_TRY(rope_tensor(who, "dq_out", dq_out, dq_out_strides, size, gq));
        OMNI_TRY(rope_tensor(who, "dk_out", dk_out, dk_out_strides, size, gk));
        OMNI_TRY(rope_tensor(who, "dq", dq, dq_strides, size, a.yq));
        OMNI_TRY(rope_tensor(who, "dk", dk, dk_strides, size, a.yk));
        rope_split(a, head_dim, 16 / size, B * T);
        a.inverse = 1;
        if (norm) {
            OMNI_TRY(rope_tensor(who, "q", q, q_strides, size, a.q));
            OMNI_TRY(rope_tensor(who, "k", k, k_strides, size, a.k));
            a.gq = gq;
            a.gk = gk;
            a.partial = static_cast<float *>(workspace);
            const int64_t n = (a.units + kRpWaves - 1) / kRpWaves;
            blocks = (int)(n < kRpBwdBlocks ? n : kRpBwdBlocks);
        } else {
            a.q = gq;                    // the inverse rotation of dy alone
            a.k = gk;
        }
        rope_launch(a, dtype, head_dim, interleaved, norm, blocks, st);
        OMNI_CHECK_LAUNCH(who);
    }
    if (norm) {
        hipLaunchKernelGGL(rope_dw_kernel, dim3(2 * head_dim / 16), dim3(1024), 0, st, static_cast<const float *>(workspace),
                           blocks, head_dim, w_dtype, dq_weight, dk_weight);
        OMNI_CHECK_LAUNCH(who);
    }
    return OMNI_OK;
}
