// Linear with an activation and a residual (rnn_linear_act_*).  No counterpart
// in the reference, whose MLP is SwiGLU.
//
// z = x W^T + b, y = act(z) + res, and for the backward the slope s = act'(z),
// which the forward has at hand (erf and exponential shared): dz = dy s is then one
// product in the loads of the two gradient products, dX = dz W and dW = dz^T x,
// and no pass over z or dz is left.  db is summed from dz on its way to LDS.
//
// One kernel for the three products, each operand stored with k along its rows
// (x, W, dz of the first two) or with k along its columns (W of the second, dz
// and x of the third).  Floats go through registers into LDS as two fp16 parts
// (mfma_half.h) in the layout they have in memory; an operand whose k runs along
// columns is handed back transposed by the LDS itself.  Two LDS buffers, the loads
// of the stage after next in flight, one barrier a stage.  Each row of op(A) and
// column of op(B), the elements that one sum takes, has a power of two of its own,
// which follows the largest magnitude so far, and the accumulators with it: a
// feature or channel keeps its bits beside one 2^30 times as large.
#include "mfma_half.h"

#include <algorithm>
#include <cmath>

namespace {

// The logistic function and its derivative, from exp(-|z|), so that neither 1 - s
// nor an overflow enters.
__device__ __forceinline__ float logistic(float z, float *d) {
    const float e = __builtin_amdgcn_exp2f(fabsf(z) * -1.44269504088896340736f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    *d = er * r;
    return z > 0.0f ? r : er;
}

// z's activation and its slope.
template <uint32_t ACT>
__device__ __forceinline__ float act_both(float z, float *slope) {
    constexpr float LOG2E = 1.44269504088896340736f;
    if constexpr (ACT == RNN_ACT_RELU) {
        *slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;
    } else if constexpr (ACT == RNN_ACT_GELU) {
        // Phi(-|z|) = exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.4 |z|): P of degree 9
        // fitted to erfcx on |z| <= 14 with a largest relative error of 1.5e-8
        // (1.5e-7 with its evaluation in 32 bits); beyond, the exponential is 0.
        // erff and expf take three times the instructions.
        const float x = fabsf(z), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, x, 1.0f));
        const float e = __builtin_amdgcn_exp2f(x * x * (-0.5f * LOG2E));
        float p = 0.032098907977342606f;
        p = __builtin_fmaf(p, t, -0.17618142068386078f);
        p = __builtin_fmaf(p, t, 0.38080015778541565f);
        p = __builtin_fmaf(p, t, -0.3719925582408905f);
        p = __builtin_fmaf(p, t, 0.11776228249073029f);
        p = __builtin_fmaf(p, t, -0.02589939534664154f);
        p = __builtin_fmaf(p, t, 0.09100669622421265f);
        p = __builtin_fmaf(p, t, 0.13320977985858917f);
        p = __builtin_fmaf(p, t, 0.15961924195289612f);
        p = __builtin_fmaf(p, t, 0.15957629680633545f);
        const float q = p * t * e, phi = z > 0.0f ? 1.0f - q : q;
        *slope = __builtin_fmaf(z, 0.39894228040143268f * e, phi);
        return z * phi;
    } else if constexpr (ACT == RNN_ACT_GELU_TANH) {
        // (1 + tanh u) / 2 is the logistic function of 2 u; beyond |z| = 30 the
        // slope is 0 or 1 to the last bit, and z^2 stays finite
        const float c = fminf(fmaxf(z, -30.0f), 30.0f), cc = c * c;
        float d;
        const float s = logistic(1.5957691216f * __builtin_fmaf(0.044715f * cc, c, c), &d);
        *slope = __builtin_fmaf(c * 1.5957691216f * __builtin_fmaf(0.134145f, cc, 1.0f), d, s);
        return z * s;
    } else if constexpr (ACT == RNN_ACT_SILU) {
        float d;
        const float s = logistic(z, &d);
        *slope = __builtin_fmaf(z, d, s);
        return z * s;
    } else {
        *slope = 1.0f;
        return z;
    }
}

template <typename F>
__device__ __forceinline__ void by_act(uint32_t act, F &&f) {
    switch (act) {
        case RNN_ACT_RELU: f(std::integral_constant<uint32_t, RNN_ACT_RELU>()); break;
        case RNN_ACT_GELU: f(std::integral_constant<uint32_t, RNN_ACT_GELU>()); break;
        case RNN_ACT_GELU_TANH: f(std::integral_constant<uint32_t, RNN_ACT_GELU_TANH>()); break;
        case RNN_ACT_SILU: f(std::integral_constant<uint32_t, RNN_ACT_SILU>()); break;
        default: f(std::integral_constant<uint32_t, RNN_ACT_NONE>()); break;
    }
}

struct LinArgs {
    const float *a, *a2, *b;  // op(A) is a, times a2 where set
    float *c, *slope;         // the product's result; EPI_SLABS: slab z at c + z M ldc
    const float *bias, *res;
    double *csum;             // EPI_SLABS: sums of op(A) over k, [split][M]
    float *db;                // EPI_ADD with one split: the same, added
    long long lda, ldb, ldc;  // ldc of slabs: N rounded up to 4
    int M, N, K, kchunk, acc;
    uint32_t act;
};

enum { EPI_ACT, EPI_ADD, EPI_SLABS };

// Four floats at any alignment of 4 bytes, the first cnt of them at a row's end.
__device__ __forceinline__ f4 quad_load(const float *p, int cnt) {
    f4 v = {0.f, 0.f, 0.f, 0.f};
    if (cnt == 4)
        v = *(const f4u *)p;
    else
        for (int e = 0; e < 3; e++)
            if (e < cnt) v[e] = p[e];
    return v;
}
__device__ __forceinline__ void quad_store(float *p, f4 v, int cnt) {
    if (cnt == 4)
        *(f4u *)p = v;
    else
        for (int e = 0; e < 3; e++)
            if (e < cnt) p[e] = v[e];
}

// How an operand of R rows (of C) is staged over a depth of KB: KC: k runs along
// its rows in memory (R rows of KB), 16-byte slots of a row exchanged so that the
// b128 reads of 8 rows fall on distinct banks; a row's power of two comes from its
// threads, which are neighbours.  Else k runs across them (KB rows of R, padded, in
// row_pos' order), read transposed; a row of C is spread over the workgroup then, and
// threads that meet a value past what its power is good for leave it in LDS (a
// maximum, so in any order) a barrier before the stage is written.
// Two register sets: stage t's loads go out while stage t - 3 is computed.
// KEEP (k across rows): the thread's powers of two stay in registers, where the kernel
// has them to spare; else they are read back from LDS.
template <int R, int KB, bool KC, bool PRO, bool KEEP, int NT>
struct Operand {
    using Stage = std::conditional_t<KC, StagePlan<R, KB, NT>, StagePlan<KB, R, NT>>;
    static constexpr int STRIDE = KC ? KB : R + 8;
    static constexpr int PART = (KC ? R : KB) * STRIDE, HALVES = 2 * PART;
    static constexpr int CH = Stage::PASSES;
    static_assert(Stage::ALL, "every thread stages");
    float x[2][CH][8], x2[PRO ? 2 : 1][PRO ? CH : 1][8];
    float up[KC ? CH : KEEP ? 8 : 1];  // powers of two of the thread's rows of C
    float good;                        // !KEEP: what all of them are good for
    const float *p, *p2;
    long long ld;
    int rows, kend, sc, sr;  // rows of C from the block's first on

    __device__ __forceinline__ static int slot(int row, int s) {
        return KB == 32 ? s ^ ((row >> 2) & 3) : s ^ (row & 7);
    }
    __device__ __forceinline__ void init(const float *base, const float *base2, long long ld_,
                                         int r0, int total, int kend_) {
        ld = ld_;
        rows = total - r0;
        kend = kend_;
        p = base + (KC ? r0 * ld : r0);
        p2 = PRO ? base2 + (KC ? r0 * ld : r0) : nullptr;
        good = good_for(FIRST_UP);
        sc = (int)threadIdx.x % Stage::C8 * 8;
        sr = (int)threadIdx.x / Stage::C8;
#pragma unroll
        for (int i = 0; i < (KC ? CH : KEEP ? 8 : 1); i++) up[i] = FIRST_UP;
    }
    template <bool TAIL>
    __device__ __forceinline__ void load_from(const float *src, int k0, float (&v)[CH][8]) const {
        const int left = kend - k0;
        const auto rs = KC ? rows_rsrc(src + k0, left > 0 ? min(rows, R) : 0, ld, left)
                           : rows_rsrc(src + k0 * ld, min(left, KB), ld, rows);
#pragma unroll
        for (int i = 0; i < CH; i++)
            load8<!TAIL>(rs, (uint32_t)(sr + i * Stage::RPP) * (uint32_t)ld + sc,
                         TAIL ? left - sc : 8, v[i]);
    }
    // The values at depth k0 (zeros from kend on) into a set.
    template <int SET>
    __device__ __forceinline__ void load(int k0) {
        if (KC && kend - k0 < KB) {
            load_from<true>(p, k0, x[SET]);
            if constexpr (PRO) load_from<true>(p2, k0, x2[SET]);
        } else {
            load_from<false>(p, k0, x[SET]);
            if constexpr (PRO) load_from<false>(p2, k0, x2[SET]);
        }
    }
    template <int SET>
    __device__ __forceinline__ void multiply() {
        if constexpr (PRO) {
#pragma unroll
            for (int i = 0; i < CH; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) x[SET][i][e] *= x2[SET][i][e];
        }
    }
    // !KEEP: the thread's powers of two in LDS (null: before any).
    __device__ __forceinline__ void powers(const float *ups, float (&u)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            f4 v = {FIRST_UP, FIRST_UP, FIRST_UP, FIRST_UP};
            if (ups) v = *(const f4 *)(ups + sc + e);
#pragma unroll
            for (int i = 0; i < 4; i++) u[e + i] = v[i];
        }
    }
    template <int SET>
    __device__ __forceinline__ float largest(int e) const {
        float m = fabsf(x[SET][0][e]);
        if constexpr (CH > 1) m = max3abs(0.f, x[SET][0][e], x[SET][1][e]);
#pragma unroll
        for (int i = 2; i < CH; i += 2) m = max3abs(m, x[SET][i][e], x[SET][i + 1 < CH ? i + 1 : i][e]);
        return m;
    }
    // !KC: the set's magnitudes past what the powers are good for into the stage's
    // maxima, and its number t beside them.  ups: powers a stage old (they only fall);
    // good: what all of the thread's are good for, beyond which each is looked at.
    template <int SET>
    __device__ __forceinline__ void maxima(const float *ups, uint32_t *most, int *over, int t) {
        multiply<SET>();
        float m[8], y[8];
        if constexpr (KEEP) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                m[e] = largest<SET>(e);
                y[e] = m[e] * up[e];
            }
        } else {
            float all = 0.f;
#pragma unroll
            for (int i = 0; i < CH; i++) all = absmax8(x[SET][i], all);
            if (!(all >= good)) return;
            powers(ups, y);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                m[e] = largest<SET>(e);
                y[e] *= m[e];
            }
        }
        if (!(absmax8(y, 0.f) >= 0x1p15f)) return;
        *over = t;
        // (all eight, also those that are not past theirs: it changes nothing)
#pragma unroll
        for (int e = 0; e < 8; e++) atomicMax(most + e * Stage::C8 + sc / 8, __float_as_uint(m[e]));
    }
    // A set into the tile at t, the powers of two into ups; whether one changed.
    // !KC: last, the stage before's powers (null: before any); most, the stage's maxima
    // where some value was past its power, else null.
    template <int SET>
    __device__ __forceinline__ bool store(_Float16 *t, float *ups, const float *last, const uint32_t *most) {
        if (KC) multiply<SET>();
        bool changed = false;
        float u8[KC ? 1 : 8];
        if constexpr (!KC) {
            if constexpr (KEEP) {
#pragma unroll
                for (int e = 0; e < 8; e++) u8[e] = up[e];
            } else {
                powers(last, u8);
            }
            if (most) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float u = sticky_up(__uint_as_float(most[e * Stage::C8 + sc / 8]), u8[e]);
                    changed = changed || u != u8[e];
                    u8[e] = u;
                }
                if constexpr (KEEP) {
#pragma unroll
                    for (int e = 0; e < 8; e++) up[e] = u8[e];
                } else {
                    float top = u8[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) top = max2(top, u8[e]);
                    good = good_for(top);
                }
            }
            if (sr == 0) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) *(f4 *)(ups + sc + e) = f4{u8[e], u8[e + 1], u8[e + 2], u8[e + 3]};
            }
        }
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int r = sr + i * Stage::RPP;
            if constexpr (KC) {
                float m = absmax8(x[SET][i], 0.f);
                m = max2(m, dpp_f<0xB1>(m));
                m = max2(m, dpp_f<0x4E>(m));
                if (Stage::C8 > 4) m = max2(m, dpp_f<0x141>(m));
                if (Stage::C8 > 8) m = max2(m, dpp_f<0x140>(m));
                const float u = sticky_up(m, up[i]);
                changed = changed || u != up[i];
                up[i] = u;
                if (sc == 0) ups[r] = u;
            }
            _Float16 *d = t + (KC ? r : row_pos(r)) * STRIDE + (KC ? 8 * slot(r, sc / 8) : sc);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = x[SET][i][e] * (KC ? up[i] : u8[KC ? 0 : e]);
            const Half2 h = half_split(v);
            *(h8 *)d = h.hi;
            *(h8 *)(d + PART) = h.lo;
        }
        return changed;
    }
    // The lane's 8 k values of step ks (16 deep) in rows r0 .. r0 + 31 of C.
    __device__ __forceinline__ static h8 frag(const _Float16 *t, int r0, int ks) {
        const int l = threadIdx.x & 63;
        if constexpr (KC) {
            const int r = r0 + (l & 31);
            return *(const h8 *)(t + r * STRIDE + 8 * slot(r, 2 * ks + (l >> 5)));
        } else {
            typedef __attribute__((address_space(3))) g4 *lds_g4;
            const _Float16 *q = t + (16 * ks + 2 * (l >> 5) + (l & 12)) * STRIDE + r0 +
                                16 * ((l >> 4) & 1) + 4 * (l & 3);
            const h4 a = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)q));
            const h4 b = __builtin_bit_cast(
                h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)(q + STRIDE)));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// C[M x N] over k: a tile of BM x BN a workgroup, KB of k a stage, WM x WN x WK
// waves (WK shares of a stage's depth, added at the end).  PRO: op(A) = a a2.
// Waves a SIMD: two workgroups a CU for the 128 x 128 tile of y and dX (dX of 8192 x
// 1152 -> 1152 136 us, 165 with one).
template <int BM, int BN, int KB, int WM, int WN, int WK, bool AK, bool BK, bool PRO, int EPI>
__global__ __launch_bounds__(64 * WM * WN * WK)
__attribute__((amdgpu_waves_per_eu(BM == 32 && BN == 128 ? 1 : BM == 128 && KB == 32 ? 4 : 2))) void
linact_kernel(LinArgs g) {
    constexpr int NW = WM * WN * WK, NT = 64 * NW, MT = BM / 32 / WM, NN = BN / 32 / WN;
    constexpr int KS = KB / 16 / WK;
    using OA = Operand<BM, KB, AK, PRO, false, NT>;
    using OB = Operand<BN, KB, BK, false, AK && !BK && BM < 128, NT>;
    constexpr int STAGE = OA::HALVES + OB::HALVES;
    constexpr size_t LDS = std::max<size_t>(4 * STAGE, (size_t)WK * BM * BN * 4);
    __shared__ __align__(16) char lds_raw[LDS];
    // operands whose k runs across rows: the largest magnitudes of even and odd stages
    // so far, where one was past its power (element e of thread column c at e C8 + c),
    // and the last stage that had one
    __shared__ uint32_t most[2][BM + BN];
    __shared__ int over[2][2];
    // the powers of two of three stages (one is read, one may be compared with it,
    // one is written), and whether a stage's differ from the one before
    __shared__ __align__(16) float ups[3][BM + BN];
    __shared__ int changes[3];
    _Float16 *const lds = (_Float16 *)lds_raw;
    const int wave = wave_index(), lane = threadIdx.x & 63, lr = lane & 31, lh = lane >> 5;
    const int wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN);
    const int tn = (g.N + BN - 1) / BN;
    const long long id = xcd_order(blockIdx.x, gridDim.x);
    const int m0 = (int)(id / tn) * BM, n0 = (int)(id % tn) * BN;
    const int kbeg = (int)blockIdx.y * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
    const int nst = kend > kbeg ? (kend - kbeg + KB - 1) / KB : 0;
    OA A;
    OB B;
    A.init(g.a, g.a2, g.lda, m0, g.M, kend);
    B.init(g.b, nullptr, g.ldb, n0, g.N, kend);
    auto load = [&](int t, auto set) {
        if (t >= nst) return;
        A.template load<decltype(set)::value>(kbeg + t * KB);
        B.template load<decltype(set)::value>(kbeg + t * KB);
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    load(0, even);
    load(1, odd);
    f32x16 acc[MT][NN];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NN; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    constexpr bool SUMS = EPI == EPI_SLABS || (EPI == EPI_ADD && !AK);
    const bool sums = SUMS && n0 == 0 && (g.csum || g.db);
    double cs[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    if (threadIdx.x < 3) changes[threadIdx.x] = 0;
    if (!AK || !BK) {
        for (int i = (int)threadIdx.x; i < 2 * (BM + BN); i += NT) most[0][i] = 0;
        if (threadIdx.x < 4) over[0][threadIdx.x] = -1;
        __syncthreads();
    }
    // (stage t's are written between the barriers t - 2 and t - 1 and read before t)
    auto maxima = [&](int t, auto set) {
        constexpr int S = decltype(set)::value;
        if (t >= nst) return;
        const float *u = t >= 2 ? ups[(t - 2) % 3] : nullptr;
        if constexpr (!AK) A.template maxima<S>(u, most[t & 1], &over[t & 1][0], t);
        if constexpr (!BK) B.template maxima<S>(u ? u + BM : u, most[t & 1] + BM, &over[t & 1][1], t);
    };
    // stage t from its set into its buffer, then the loads of stage t + 2
    auto stage = [&](int t, auto set) {
        constexpr int S = decltype(set)::value;
        if (t >= nst) return;
        _Float16 *d = lds + (t & 1) * STAGE;
        float *u = ups[t % 3];
        const uint32_t *ma = !AK && over[t & 1][0] == t ? most[t & 1] : nullptr;
        const uint32_t *mb = !BK && over[t & 1][1] == t ? most[t & 1] + BM : nullptr;
        const float *last = t ? ups[(t + 2) % 3] : nullptr;
        const bool ca = A.template store<S>(d, u, last, ma);
        const bool cb = B.template store<S>(d + OA::HALVES, u + BM, last ? last + BM : last, mb);
        if (t && (ca || cb)) changes[t % 3] = 1;
        if (SUMS && sums) {
#pragma unroll
            for (int i = 0; i < OA::CH; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) cs[e] += (double)A.x[S][i][e];
        }
        load(t + 2, set);
    };
    auto step = [&](int t, auto cur, auto nxt) {
        __syncthreads();
        const float *u = ups[t % 3];
        if (changes[t % 3]) {
            const float *v = ups[(t + 2) % 3];
#pragma unroll
            for (int j = 0; j < NN; j++) {
                const int c = (wn * NN + j) * 32 + lr;
                const float rb = u[BM + c] * down_of(v[BM + c]);
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int m = (wm * MT + i) * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
                        acc[i][j][r] *= u[m] * down_of(v[m]) * rb;
                    }
            }
        }
        if (threadIdx.x == 0) changes[(t + 2) % 3] = 0;
        stage(t + 1, nxt);
        const _Float16 *const ta = lds + (t & 1) * STAGE, *const tb = ta + OA::HALVES;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int ks = wk * KS + s;
            h8 ah[MT], al[MT], bh[NN], bl[NN];
#pragma unroll
            for (int i = 0; i < MT; i++) {
                ah[i] = OA::frag(ta, (wm * MT + i) * 32, ks);
                al[i] = OA::frag(ta + OA::PART, (wm * MT + i) * 32, ks);
            }
#pragma unroll
            for (int j = 0; j < NN; j++) {
                bh[j] = OB::frag(tb, (wn * NN + j) * 32, ks);
                bl[j] = OB::frag(tb + OB::PART, (wn * NN + j) * 32, ks);
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NN; j++) {
                    acc[i][j] = mm(al[i], bh[j], acc[i][j]);
                    acc[i][j] = mm(ah[i], bl[j], acc[i][j]);
                    acc[i][j] = mm(ah[i], bh[j], acc[i][j]);
                }
        }
        maxima(t + 2, cur);
    };
    maxima(0, even);
    if (!AK || !BK) __syncthreads();
    stage(0, even);
    maxima(1, odd);
    for (int t = 0; t < nst; t += 2) {
        step(t, even, odd);
        if (t + 1 < nst) step(t + 1, odd, even);
    }
    // The waves' tiles through LDS, so that rows are written whole.
    float *const ct = (float *)lds_raw;
    __syncthreads();
    const float *const ul = ups[(nst + 2) % 3];  // the last stage's
#pragma unroll
    for (int j = 0; j < NN; j++) {
        const int c = (wn * NN + j) * 32 + lr;
        const float db = nst ? down_of(ul[BM + c]) : 0.f;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int m = (wm * MT + i) * 32 + 2 * r + 4 * lh;
                const f4 ua = *(const f4 *)(ul + m);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    ct[(wk * BM + m + e) * BN + c] = acc[i][j][r + e] * (nst ? down_of(ua[e]) : 0.f) * db;
            }
    }
    __syncthreads();
    for (int u = (int)threadIdx.x; u < BM * BN / 4; u += NT) {
        const int r = u / (BN / 4), c = u % (BN / 4) * 4, row = m0 + r, col = n0 + c;
        if (row >= g.M || col >= g.N) continue;
        f4 v = *(const f4 *)(ct + r * BN + c);
#pragma unroll
        for (int w = 1; w < WK; w++) v += *(const f4 *)(ct + (w * BM + r) * BN + c);
        const int cnt = min(4, g.N - col);
        const long long at = (long long)row * g.ldc + col;
        float *out = g.c + at + (EPI == EPI_SLABS ? (long long)blockIdx.y * g.M * g.ldc : 0);
        if constexpr (EPI == EPI_ACT) {
            const f4 bias = g.bias ? quad_load(g.bias + col, cnt) : f4{0.f, 0.f, 0.f, 0.f};
            f4 add = {0.f, 0.f, 0.f, 0.f}, s;
            if (g.res) add = quad_load(g.res + at, cnt);
            by_act(g.act, [&](auto a) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float sl;
                    const float y = act_both<decltype(a)::value>(v[e] + bias[e], &sl);
                    v[e] = g.res ? y + add[e] : y;
                    s[e] = sl;
                }
            });
            if (g.slope) quad_store(g.slope + at, s, cnt);
        } else if (EPI == EPI_ADD && g.acc) {
            v = quad_load(out, cnt) + v;
        }
        quad_store(out, v, EPI == EPI_SLABS ? 4 : cnt);
    }
    if constexpr (SUMS) {
        if (!sums) return;
        // op(A)'s sums over k: the passes' rows in order
        __syncthreads();
        double *red = (double *)lds_raw;  // [RPP][BM]
        static_assert((size_t)OA::Stage::RPP * BM * 8 <= LDS, "sums fit");
#pragma unroll
        for (int e = 0; e < 8; e++) red[A.sr * BM + A.sc + e] = cs[e];
        __syncthreads();
        for (int c = (int)threadIdx.x; c < BM; c += NT) {
            if (m0 + c >= g.M) continue;
            double s = 0.0;
            for (int i = 0; i < OA::Stage::RPP; i++) s += red[i * BM + c];
            if (EPI == EPI_SLABS)
                g.csum[(long long)blockIdx.y * g.M + m0 + c] = s;
            else
                g.db[m0 + c] += (float)s;
        }
    }
}

// dw += the slabs, db += the sums, each in split order, four loads ahead.  A
// thread owns a quad of a row of dw (rows of the slabs end on a quad).
__global__ __launch_bounds__(256) void linact_reduce_kernel(const float *__restrict__ slab,
                                                            const double *__restrict__ csum,
                                                            int nz, int M, int N, int quads,
                                                            float *__restrict__ dw,
                                                            float *__restrict__ db, unsigned wblocks) {
    if (blockIdx.x >= wblocks) {
        const int m = (int)(blockIdx.x - wblocks) * 256 + (int)threadIdx.x;
        if (m >= M) return;
        double s = 0.0;
        for (int z = 0; z < nz; z++) s += csum[(long long)z * M + m];
        db[m] += (float)s;
        return;
    }
    const long long u = (long long)blockIdx.x * 256 + threadIdx.x, len = (long long)M * quads;
    if (u >= len) return;
    const int row = (int)(u / quads), col = (int)(u - (long long)row * quads) * 4;
    const int cnt = min(4, N - col);
    float *out = dw + (long long)row * N + col;
    const f4 old = quad_load(out, cnt);
    const f4 *q = (const f4 *)slab + u;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    int z = 0;
    for (; z + 4 <= nz; z += 4) {
        f4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = q[(z + i) * len];
#pragma unroll
        for (int i = 0; i < 4; i++) s += v[i];
    }
    for (; z < nz; z++) s += q[z * len];
    quad_store(out, old + s, cnt);
}

// The tile of y and dX by the number of tiles that it leaves: the largest that
// gives the 256 CUs about one each; in the smaller ones waves share a stage's
// depth.  Forward 8192 x 256 -> 1024 with 128 x 128 / 64 x 128 / 32 x 128 tiles:
// 30.2 / 49.0 / 86.9 us; 1813 x 387 -> 1003: 26.8 / 20.1 / 35.5.  dX of these:
// 50.6 / 33.0 / 57.8 and 57.6 / 32.0 / 30.3 us.
enum { TILE_128, TILE_64X128, TILE_32X128, TILE_32 };
int pick_tile(size_t m, size_t n) {
    auto tiles = [&](size_t bm, size_t bn) { return rnn_div_up(m, bm) * rnn_div_up(n, bn); };
    if (tiles(128, 128) >= 256) return TILE_128;
    if (tiles(64, 128) >= 192) return TILE_64X128;
    if (tiles(32, 128) >= 192) return TILE_32X128;
    return TILE_32;
}

template <int BM, int BN, int KB, int WM, int WN, int WK, bool AK, bool BK, bool PRO, int EPI>
void launch_tile(rnn_ctx *ctx, const LinArgs &g, size_t nz) {
    const size_t tiles = rnn_div_up((size_t)g.M, BM) * rnn_div_up((size_t)g.N, BN);
    linact_kernel<BM, BN, KB, WM, WN, WK, AK, BK, PRO, EPI>
        <<<dim3((unsigned)tiles, (unsigned)nz), 64 * WM * WN * WK, 0, ctx->stream>>>(g);
}
template <bool AK, bool BK, bool PRO, int EPI>
void launch(rnn_ctx *ctx, const LinArgs &g) {
    switch (pick_tile((size_t)g.M, (size_t)g.N)) {
        case TILE_128: launch_tile<128, 128, 32, 2, 4, 1, AK, BK, PRO, EPI>(ctx, g, 1); break;
        case TILE_64X128: launch_tile<64, 128, 64, 1, 4, 2, AK, BK, PRO, EPI>(ctx, g, 1); break;
        case TILE_32X128: launch_tile<32, 128, 64, 1, 2, 2, AK, BK, PRO, EPI>(ctx, g, 1); break;
        default: launch_tile<32, 32, 128, 1, 1, 4, AK, BK, PRO, EPI>(ctx, g, 1); break;
    }
}

// dW's tile and the splits of its k (the rows), at least 128 rows each: about one
// workgroup a CU.  8192 x 256 -> 1024 with 128 x 128 / 64 x 64 tiles: 36 + 7 / 59 + 5
// us with the splits' sum; twice the splits 47 + 12.
struct DwPlan {
    bool wide;  // 128 x 128, else 64 x 64
    size_t nz, kchunk;
};
DwPlan plan_dw(size_t rows, size_t fin, size_t fout) {
    DwPlan p;
    p.wide = fout >= 128 && fin >= 128;
    const size_t b = p.wide ? 128 : 64;
    const size_t tiles = rnn_div_up(fout, b) * rnn_div_up(fin, b);
    size_t nz = tiles ? std::max<size_t>(1, std::min(rnn_div_up(256, tiles), rows / 128)) : 1;
    nz = std::min<size_t>(nz, 64);
    p.kchunk = rnn_round_up(rnn_div_up(std::max<size_t>(rows, 1), nz), 64);
    p.nz = rnn_div_up(std::max<size_t>(rows, 1), p.kchunk);
    return p;
}
template <bool PRO, int EPI>
void launch_dw(rnn_ctx *ctx, const LinArgs &g, const DwPlan &p) {
    if (p.wide)
        launch_tile<128, 128, 64, 2, 2, 2, false, false, PRO, EPI>(ctx, g, p.nz);
    else
        launch_tile<64, 64, 64, 1, 1, 4, false, false, PRO, EPI>(ctx, g, p.nz);
}

struct LinWs {
    size_t slab = 0, csum = 0, bytes = 0;
};
LinWs plan_ws(size_t rows, size_t fin, size_t fout) {
    LinWs w;
    const DwPlan p = plan_dw(rows, fin, fout);
    WsCarve cv;
    if (p.nz > 1) {
        w.slab = cv.take(p.nz * rnn_round_up(fin, 4) * fout * sizeof(float));
        w.csum = cv.take(p.nz * fout * sizeof(double));
    }
    w.bytes = cv.off;
    return w;
}

// (2^30 rows would be a grid of 2^32 threads, which is one too many)
int size_check(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout) {
    if (rows > (1u << 30) - 128 || fin > (1u << 20) || fout > (1u << 20))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "linear_act: %zu x %zu -> %zu", rows, fin, fout);
    return RNN_OK;
}

}  // namespace

extern "C" {

int rnn_linear_act_forward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                           const float *w, const float *b, uint32_t act, const float *res,
                           float *slope, float *y) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (act > RNN_ACT_SILU)
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_forward: activation %u", act);
    const int rc = size_check(ctx, rows, fin, fout);
    if (rc) return rc;
    if (rows == 0 || fout == 0) return RNN_OK;
    if ((fin && (!x || !w)) || !y) return rnn_fail(ctx, RNN_E_NULL, "linear_act_forward: null operand");
    if (y == x || y == w || (slope && (slope == x || slope == w || slope == y || slope == res)))
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_forward: aliased operands");
    RNN_ON_DEVICE(ctx);
    LinArgs g{};
    g.a = x;
    g.b = w;
    g.c = y;
    g.slope = slope;
    g.bias = b;
    g.res = res;
    g.lda = g.ldb = (long long)fin;
    g.ldc = (long long)fout;
    g.M = (int)rows;
    g.N = (int)fout;
    g.K = g.kchunk = (int)fin;
    g.act = act;
    launch<true, true, false, EPI_ACT>(ctx, g);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_linear_act_workspace(size_t rows, size_t fin, size_t fout, size_t *bytes) {
    const int rc = size_check(nullptr, rows, fin, fout);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    *bytes = plan_ws(rows, fin, fout).bytes;
    return RNN_OK;
}

int rnn_linear_act_backward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                            const float *x, const float *w, const float *slope, void *ws,
                            size_t ws_bytes, float *dw, float *db, float *dx, uint32_t flags) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (flags & ~RNN_LINEAR_ACC_DX)
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_backward: flags 0x%x", flags);
    const int rc = size_check(ctx, rows, fin, fout);
    if (rc) return rc;
    if ((rows && fout && !dy) || (rows && fin && (!x || !dx)) || (fin && fout && (!w || !dw)))
        return rnn_fail(ctx, RNN_E_NULL, "linear_act_backward: null operand");
    if (dx && (dx == dy || dx == x || dx == w || dx == slope || dx == dw))
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_backward: dx aliases another operand");
    if (!fin && fout && db)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "linear_act_backward: db without inputs");
    const LinWs plan = plan_ws(rows, fin, fout);
    if (plan.bytes) {
        if (!ws) return rnn_fail(ctx, RNN_E_NULL, "linear_act_backward: workspace is null");
        if (ws_bytes < plan.bytes || ((uintptr_t)ws & 255))
            return rnn_fail(ctx, RNN_E_INVALID,
                            "linear_act_backward: workspace of %zu bytes, needs %zu, 256-byte aligned",
                            ws_bytes, plan.bytes);
    }
    if (!rows) return RNN_OK;
    RNN_ON_DEVICE(ctx);
    LinArgs g{};
    g.a = dy;
    g.a2 = slope;
    // dX = dz W
    if (fin) {
        g.b = w;
        g.c = dx;
        g.lda = (long long)fout;
        g.ldb = g.ldc = (long long)fin;
        g.M = (int)rows;
        g.N = (int)fin;
        g.K = g.kchunk = (int)fout;
        g.acc = (flags & RNN_LINEAR_ACC_DX) ? 1 : 0;
        if (slope)
            launch<true, false, true, EPI_ADD>(ctx, g);
        else
            launch<true, false, false, EPI_ADD>(ctx, g);
        RNN_LAUNCHED(ctx);
    }
    if (!fout || !fin) return RNN_OK;
    // dW += dz^T x and db += the sums of dz
    const DwPlan p = plan_dw(rows, fin, fout);
    g.b = x;
    g.lda = (long long)fout;
    g.ldb = (long long)fin;
    g.M = (int)fout;
    g.N = (int)fin;
    g.K = (int)rows;
    g.kchunk = (int)p.kchunk;
    if (p.nz > 1) {
        g.c = (float *)((char *)ws + plan.slab);
        g.ldc = (long long)rnn_round_up(fin, 4);
        g.csum = db ? (double *)((char *)ws + plan.csum) : nullptr;
        if (slope)
            launch_dw<true, EPI_SLABS>(ctx, g, p);
        else
            launch_dw<false, EPI_SLABS>(ctx, g, p);
        RNN_LAUNCHED(ctx);
        const size_t quads = rnn_div_up(fin, 4);
        const unsigned wb = (unsigned)rnn_div_up(fout * quads, 256);
        const unsigned bb = db ? (unsigned)rnn_div_up(fout, 256) : 0u;
        linact_reduce_kernel<<<wb + bb, 256, 0, ctx->stream>>>(g.c, g.csum, (int)p.nz, (int)fout,
                                                               (int)fin, (int)quads, dw, db, wb);
        RNN_LAUNCHED(ctx);
        return RNN_OK;
    }
    g.c = dw;
    g.db = db;
    g.acc = 1;
    if (slope)
        launch_dw<true, EPI_ADD>(ctx, g, p);
    else
        launch_dw<false, EPI_ADD>(ctx, g, p);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

}  // extern "C"
