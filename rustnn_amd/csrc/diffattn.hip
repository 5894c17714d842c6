// Differential attention (rnn_diff_attn_*).  No counterpart in the reference.
//
//   P_m = softmax(scale Q_m K_m^T), O = (P_1 - lambda P_2) V,
//   y = (1 - lam_init) gain O rsqrt(mean O^2 + eps)
// and backward, with T = (1 - lam_init) gain dy, r = rsqrt(mean O^2 + eps),
// Oh = O r:
//   dO = r (T - Oh mean(T Oh)), dgain = (1 - lam_init) sum dy Oh,
//   dA = dO V^T, D_m = dO . (P_m V),
//   dS_1 = P_1 (dA - D_1), dS_2 = -lambda P_2 (dA - D_2),
//   dQ_m = scale dS_m K_m, dK_m = scale dS_m^T Q_m, dV = (P_1 - lambda P_2)^T dO,
//   dlambda = -sum D_2.
#include "rnn_internal.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MAX_DH = 64;
constexpr float LOG2E = 1.44269504088896340736f;

struct DiffArgs {
    const float *q, *kv, *lam, *gain, *dy;
    const uint32_t *qlen, *klen;
    const float *o12c, *statsc;
    float *y, *o12, *stats;
    float *dq, *dkv;
    float *dout;  // dO, [n][tq][h][2 dh]
    float *dd;    // D_1, D_2, [n][tq][h][2]
    float *part32, *pstat;  // splits: outputs [n][tq][h][splits][2][2 dh], (max, sum) beside them
    double *part; // partials of dgain and dlambda, [blocks][2 dh + h]
    long long qstride, kvstride;
    int n, h, hkv, dh, tq, tk, koff, voff, lam_heads, diag, causal, group;
    int acc_q, acc_kv, rpb, split_keys;
    float scale, lam_init, eps;
};

__device__ __forceinline__ int len_of(const uint32_t *len, int b, int t) {
    return len ? (int)min(len[b], (uint32_t)t) : t;
}

// exp(lq1 . lk1) and exp(lq2 . lk2) of a head, on every lane.
__device__ __forceinline__ void lambda_terms(const float *lam, int lam_heads, int dh, int head,
                                             double *e1, double *e2) {
    const int lane = threadIdx.x & 63;
    const float *l = lam + (lam_heads > 1 ? (long long)head * 4 * dh : 0);
    const bool in = lane < dh;
    const double a = in ? (double)l[lane] * (double)l[dh + lane] : 0.0;
    const double b = in ? (double)l[2 * dh + lane] * (double)l[3 * dh + lane] : 0.0;
    *e1 = exp(rnn_wave_sum_d(a));
    *e2 = exp(rnn_wave_sum_d(b));
}

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct Seen {  // the keys that a query sees, and the queries that see a key
    int nq, nk, shift, diag, causal;
    __device__ Seen(const DiffArgs &g, int b)
        : nq(len_of(g.qlen, b, g.tq)), nk(len_of(g.klen, b, g.tk)), shift(nk - nq), diag(g.diag),
          causal(g.causal) {}
    __device__ bool operator()(int i, int j) const {
        return i < nq && j < nk && !(causal && j > i + shift) && !(diag && i == j);
    }
};

// ---------------------------------------------------------------------------
// fp32 products on the fp16 matrix cores.
//
// A float times a power of two is hi + lo, hi its nearest fp16 and lo the
// nearest fp16 of the rest: hi + lo is within half a step of 2^-22, so 2^-23, of
// it, as long as lo is no subnormal, which ends 2^-25 at 2^15.  With the power
// chosen so that the largest magnitude of a row or tile comes to
// [2^14, 2^15), every element down to 2^-16 of the largest keeps 2^-23, and
// below that all keep 2^-39 of the largest.  a b is then hi hi + hi lo + lo hi:
// products of 22 bits, exact in the matrix core, summed in its fp32
// accumulator; lo lo, left out, is below 2^-22 of the product and of no common
// sign.  Three products an element and four bytes in LDS, where three bf16
// parts (mfma_split.h) take six and six; their range of exponents is not needed
// here, since rows and tiles carry their power of two beside them.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __fp16 g4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct Half2 {
    h8 hi, lo;
};

// The two parts of 8 floats times up (a power of two).
__device__ __forceinline__ Half2 half_split(const float (&x)[8], float up) {
    Half2 r;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const f2 v = {x[2 * j] * up, x[2 * j + 1] * up};
        const h2 h = __builtin_convertvector(v, h2);
        const f2 d = {v[0] - (float)h[0], v[1] - (float)h[1]};
        const h2 l = __builtin_convertvector(d, h2);
        r.hi[2 * j] = h[0];
        r.hi[2 * j + 1] = h[1];
        r.lo[2 * j] = l[0];
        r.lo[2 * j + 1] = l[1];
    }
    return r;
}

// The power of two that takes a largest magnitude m to [2^14, 2^15) (m of 0,
// an infinity or a NaN: 1), and its reciprocal.  Magnitudes below 2^-112 stay
// smaller.
__device__ __forceinline__ float up_of(float m) {
    const int e = (int)(__float_as_uint(m) >> 23) & 255;
    const int f = (e == 255 || m == 0.0f) ? 127 : min(268 - e, 253);
    return __uint_as_float((uint32_t)f << 23);
}
__device__ __forceinline__ float down_of(float up) {
    return __uint_as_float((254u << 23) - __float_as_uint(up));
}

__device__ __forceinline__ f32x16 mm(h8 a, h8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// A tile of ROWS rows of W channels in LDS, both parts: row r's hi at
// r * STRIDE, its lo PART further on.  The 16 bytes of padding put the b128
// reads of 8 consecutive rows on distinct banks (an odd number of 16-byte
// slots a row).
template <int ROWS, int W>
struct HalfTile {
    static constexpr int STRIDE = W + 8;  // in halves
    static constexpr int PART = ROWS * STRIDE;
    static constexpr int HALVES = 2 * PART;
    // 8 consecutive channels of a row: an operand with its k along channels
    static __device__ __forceinline__ h8 along(const _Float16 *t, int row, int c) {
        return *(const h8 *)(t + row * STRIDE + c);
    }
    // Rows row0 + {0..3, 8..11} (row0 + 4 for the upper half wave) of channel
    // c0 + lane % 32: an operand with its k along rows, in the order in which
    // a 32 x 32 accumulator's registers 8 s .. 8 s + 7 hold the rows of the
    // block of 16 at row0.  Each 16 lanes read 4 rows of 16 channels, which
    // the LDS hands back transposed.
    static __device__ __forceinline__ h8 across(const _Float16 *t, int row0, int c0) {
        const int l = threadIdx.x & 63;
        const _Float16 *p = t + (row0 + 4 * (l >> 5) + ((l & 15) >> 2)) * STRIDE + c0 +
                            16 * ((l >> 4) & 1) + 4 * (l & 3);
        typedef __attribute__((address_space(3))) g4 *lds_g4;
        const h4 a = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)p));
        const h4 b = __builtin_bit_cast(
            h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)(p + 8 * STRIDE)));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// 8 consecutive channels, `off` floats into a buffer resource, zero from `lim`
// channels on and past the resource's end.
template <bool VEC>
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t rs, uint32_t off, int lim,
                                      float (&x)[8]) {
    if constexpr (VEC) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint32_t at = 4 * q < lim ? (off + 4 * q) * 4 : DMA_OOB;
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * q + e] = __uint_as_float(v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                rs, e < lim ? (off + e) * 4 : DMA_OOB, 0, 0));
    }
}

// The same from a row's address.
template <bool VEC>
__device__ __forceinline__ void load8g(const float *p, int lim, float (&x)[8]) {
    if constexpr (VEC) {
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 a = lim > 0 ? *(const float4 *)p : z;
        const float4 b = lim > 4 ? *(const float4 *)(p + 4) : z;
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = e < lim ? p[e] : 0.f;
    }
}

// How NT threads stage a tile of ROWS rows of W channels: RPP rows a pass, 8
// channels a thread, so that a thread keeps its channels from pass to pass
// (W = 96: the last quarter of the threads idle).
template <int ROWS, int W, int NT>
struct StagePlan {
    static constexpr int C8 = W / 8;
    static constexpr int fit = NT / C8;
    static constexpr int RPP = fit >= 64 ? 64 : fit >= 32 ? 32 : fit >= 16 ? 16 : 8;
    static constexpr int PASSES = ROWS / RPP;
    static constexpr bool ALL = RPP * C8 == NT;
    static_assert(RPP * C8 <= NT && PASSES * RPP == ROWS, "whole passes");
};

__device__ __forceinline__ float absmax8(const float (&x)[8], float m) {
#pragma unroll
    for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(x[e]));
    return m;
}

constexpr float P_UP = 16384.0f, P_EXP = 14.0f;  // softmax values enter the products times 2^14
constexpr float NO_MAX = -1e30f;                 // a running maximum before any score

// The block's number in an order in which each XCD (block id % 8) gets a
// contiguous run: the blocks that share a problem's keys meet in one L2.
__device__ __forceinline__ long long xcd_order(long long id, long long total) {
    const long long per = total >> 3, rem = total & 7, x = id & 7, loc = id >> 3;
    return x < rem ? x * (per + 1) + loc : rem * (per + 1) + (x - rem) * per + loc;
}

// The four lambda vectors' terms of a lane's own head.
__device__ __forceinline__ float lane_lambda(const DiffArgs &g, int head) {
    const float *l = g.lam + (g.lam_heads > 1 ? (long long)head * 4 * g.dh : 0);
    double a = 0.0, b = 0.0;
    for (int c = 0; c < g.dh; c++) {
        a = fma((double)l[c], (double)l[g.dh + c], a);
        b = fma((double)l[2 * g.dh + c], (double)l[3 * g.dh + c], b);
    }
    return (float)(exp(a) - exp(b) + (double)g.lam_init);
}

// Forward.  One workgroup of 2 QG waves per (image, key head, 32 QG rows); a
// row is a query of one of the head group's heads, so that heads that share
// keys share their tiles.  Wave 2 i + m owns rows [32 i, 32 i + 32) and map m:
// its scores are S^T = K Q^T (lane = row), so that a row's maximum and sum stay
// in two lanes, and the exponentials are, register by register, the operand of
// O^T = V^T P^T.  Tiles of 64 keys and values are split into LDS once for all
// waves; the next tile's loads are in flight meanwhile, and its largest
// magnitudes are taken while they are in registers.
// SPLIT: the keys [z TS, (z + 1) TS) alone (z = blockIdx.y), each map's own
// normalised output, maximum and sum left for diff_join_kernel.
template <int DHP, bool VEC, int QG, bool SPLIT>
__global__ __launch_bounds__(128 * QG)
__attribute__((amdgpu_waves_per_eu(QG == 4 || DHP <= 32 ? 2 : 1))) void
diff_fwd_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TK = 64, NT = 128 * QG, KS = DHP / 16, CT = DHP / 16;
    using Tile = HalfTile<TK, W>;
    using Stage = StagePlan<TK, W, NT>;
    constexpr int CH = Stage::PASSES;
    static_assert((int)sizeof(_Float16) * 2 * Tile::HALVES >= QG * CT * 16 * 64 * 4, "exchange");
    __shared__ __align__(16) _Float16 lds[2 * Tile::HALVES];
    __shared__ float tmax[2][2][2 * QG];
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int map = wave & 1, qg = wave >> 1;
    const int R = g.tq * g.group, nrb = (R + 32 * QG - 1) / (32 * QG);
    const long long id = xcd_order(blockIdx.x, gridDim.x);
    const int prob = (int)(id / nrb), rb = nrb - 1 - (int)(id % nrb);  // causal: longest first
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int row = rb * 32 * QG + qg * 32 + lr;
    const int qi = row / g.group, head = kh * g.group + row % g.group;
    const bool live = qi < nq;
    // keys that some row of the block sees
    const int last_q = min(nq - 1, (rb * 32 * QG + 32 * QG - 1) / g.group);
    int kend = g.causal ? min(nk, last_q + shift + 1) : nk;
    if (rb * 32 * QG / g.group >= nq) kend = 0;
    const int kbeg = SPLIT ? (int)blockIdx.y * g.split_keys : 0;
    if (SPLIT) kend = min(kend, kbeg + g.split_keys);
    const int ntile = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;

    const float *kv = g.kv + (long long)b * g.tk * g.kvstride;
    const float *kp = kv + g.koff + 2 * kh * g.dh, *vp = kv + g.voff + 2 * kh * g.dh;
    float xk[CH][8], xv[CH][8];
    // the thread's channels [sc, sc + 8) of rows sr, sr + RPP, ...; keys: two
    // runs of dh padded to DHP, values: one of 2 dh
    const int sc = (int)threadIdx.x % Stage::C8 * 8, sr = (int)threadIdx.x / Stage::C8;
    const bool stager = Stage::ALL || sr < Stage::RPP;
    const int run = sc >= DHP ? 1 : 0;
    const int klim = stager ? g.dh - (sc - run * DHP) : 0, vlim = stager ? 2 * g.dh - sc : 0;
    const uint32_t koff = sr * (uint32_t)g.kvstride + sc - run * (DHP - g.dh);
    const uint32_t voff = sr * (uint32_t)g.kvstride + sc;
    auto load = [&](int k0) {
        // rows from kend on are past the resource's end
        const uint32_t bytes = (uint32_t)min(kend - k0, TK) * (uint32_t)g.kvstride * 4;
        const long long at = k0 * g.kvstride;
        const auto rk = make_rsrc(kp + at, bytes), rv = make_rsrc(vp + at, bytes);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const uint32_t step = i * Stage::RPP * (uint32_t)g.kvstride;
            load8<VEC>(rk, koff + step, klim, xk[i]);
            load8<VEC>(rv, voff + step, vlim, xv[i]);
        }
    };
    auto maxima = [&](int slot) {
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            mk = absmax8(xk[i], mk);
            mv = absmax8(xv[i], mv);
        }
        mk = wave_max(mk);
        mv = wave_max(mv);
        if (lane == 0) {
            tmax[slot][0][wave] = mk;
            tmax[slot][1][wave] = mv;
        }
    };
    if (ntile) load(kbeg);

    // the row's query of this map, times its own power of two
    Half2 q[KS];
    float qdown;
    {
        const float *qp = g.q + ((long long)b * g.tq + min(qi, g.tq - 1)) * g.qstride +
                          (2 * head + map) * g.dh;
        float v[KS][8], mx = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int c = 16 * s + 8 * lh;
            load8g<VEC>(qp + c, live ? g.dh - c : 0, v[s]);
            mx = absmax8(v[s], mx);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float up = up_of(mx);
        qdown = down_of(up) * (g.scale * LOG2E);
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = half_split(v[s], up);
    }
    f32x16 o[CT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[c][r] = 0.f;
    float m = NO_MAX, l = 0.f, vdown = 0.f, odown = 0.f;
    // rows of the wave's queries, for tiles that every one of them sees whole
    const int w_first = (rb * 32 * QG + qg * 32) / g.group;
    const int w_last = min(nq - 1, (rb * 32 * QG + qg * 32 + 31) / g.group);
    if (ntile) maxima(0);
    _Float16 *const kt = lds, *const vt = lds + Tile::HALVES;
    for (int t = 0; t < ntile; t++) {
        const int k0 = kbeg + t * TK;
        __syncthreads();
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * QG; i++) {
            mk = fmaxf(mk, tmax[t & 1][0][i]);
            mv = fmaxf(mv, tmax[t & 1][1][i]);
        }
        const float kup = up_of(mk);
        // the output's unit follows the tile's; at most 2^60 down at once, so
        // that what is there does not overflow
        float vup = up_of(mv);
        if (t) vup = fminf(vup, down_of(vdown) * 0x1p60f);
        vdown = down_of(vup);
        if (stager) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                _Float16 *d = kt + (sr + i * Stage::RPP) * Tile::STRIDE + sc;
                const Half2 hk = half_split(xk[i], kup), hv = half_split(xv[i], vup);
                *(h8 *)d = hk.hi;
                *(h8 *)(d + Tile::PART) = hk.lo;
                *(h8 *)(d + Tile::HALVES) = hv.hi;
                *(h8 *)(d + Tile::HALVES + Tile::PART) = hv.lo;
            }
        }
        if (t + 1 < ntile) load(k0 + TK);
        __syncthreads();
        const bool any = g.causal ? k0 <= w_last + shift : true;
        if (any && w_first < nq) {
            const float f = down_of(kup) * qdown;
            float u[2][16];
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++) {
                f32x16 hh, sm;
#pragma unroll
                for (int r = 0; r < 16; r++) hh[r] = sm[r] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const int c = map * DHP + 16 * s + 8 * lh;
                    const h8 hi = Tile::along(kt, 32 * s2 + lr, c);
                    const h8 lo = Tile::along(kt + Tile::PART, 32 * s2 + lr, c);
                    sm = mm(hi, q[s].lo, sm);
                    hh = mm(hi, q[s].hi, hh);
                    sm = mm(lo, q[s].hi, sm);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) u[s2][r] = (hh[r] + sm[r]) * f;
            }
            const bool whole = k0 + TK <= nk && !(g.causal && k0 + TK - 1 > w_first + shift) &&
                               !(g.diag && k0 <= w_last && w_first < k0 + TK);
            if (!whole) {
#pragma unroll
                for (int s2 = 0; s2 < 2; s2++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int j = k0 + 32 * s2 + 8 * (r >> 2) + 4 * lh + (r & 3);
                        const bool in = j < nk && !(g.causal && j > qi + shift) &&
                                        !(g.diag && j == qi);
                        u[s2][r] = in ? u[s2][r] : -INFINITY;
                    }
            }
            float mn = m;
#pragma unroll
            for (int r = 0; r < 16; r++) mn = fmaxf(mn, fmaxf(u[0][r], u[1][r]));
            mn = fmaxf(mn, __shfl_xor(mn, 32, 64));
            const float al = __builtin_amdgcn_exp2f(m - mn), base = mn - P_EXP;
            m = mn;
            l *= al;
            Half2 p[4];
            float ps = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    e[i] = __builtin_amdgcn_exp2f(u[s >> 1][8 * (s & 1) + i] - base);
                    ps += e[i];
                }
                p[s] = half_split(e, 1.0f);
            }
            l += ps;
            const float keep = al * (odown * vup);
            odown = vdown;
#pragma unroll
            for (int c = 0; c < CT; c++) {
                f32x16 a;
#pragma unroll
                for (int r = 0; r < 16; r++) a[r] = 0.f;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const h8 hi = Tile::across(vt, 16 * s, 32 * c);
                    const h8 lo = Tile::across(vt + Tile::PART, 16 * s, 32 * c);
                    a = mm(lo, p[s].hi, a);
                    a = mm(hi, p[s].lo, a);
                    a = mm(hi, p[s].hi, a);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) o[c][r] = __builtin_fmaf(o[c][r], keep, a[r]);
            }
        }
        if (t + 1 < ntile) maxima((t + 1) & 1);
    }
    l += __shfl_xor(l, 32, 64);
    const bool some = live && l > 0.f;
    const float il = some ? odown / l : 0.f;  // both carry 2^14
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[c][r] = some ? o[c][r] * il : 0.f;
    if (!some) m = 0.f;
    const int dv = 2 * g.dh;
    const long long out = ((long long)b * g.tq + qi) * g.h + head;  // (image, query, head)
    if constexpr (SPLIT) {
        if (row < R) {
            const long long at = (out * gridDim.y + blockIdx.y) * 2 + map;
            if (lh == 0) *(f2 *)(g.pstat + at * 2) = f2{m, some ? l : 0.f};
            float *dst = g.part32 + at * dv;
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int ch = 32 * c + 8 * (r >> 2) + 4 * lh + (r & 3);
                    if (ch < dv) dst[ch] = o[c][r];
                }
        }
        return;
    }
    // map 1's output to its partner wave
    __syncthreads();
    float *ex = (float *)lds + qg * CT * 16 * 64;
    if (map == 1) {
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) ex[(c * 16 + r) * 64 + lane] = o[c][r];
    }
    if (g.stats && row < R && lh == 0)
        *(f2 *)(g.stats + out * 4 + 2 * map) = f2{m, some ? P_UP / l : 0.f};
    float lam = 0.f;
    if (map == 0) lam = lane_lambda(g, min(head, g.h - 1));
    __syncthreads();
    const bool vst = VEC;  // whole float4s: dv % 4 == 0, aligned rows
    auto store = [&](float *dst, auto &&val) {
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int ch = 32 * c + 2 * r + 4 * lh;
                if (vst) {
                    if (ch < dv)
                        *(float4 *)(dst + ch) =
                            make_float4(val(c, r, ch), val(c, r + 1, ch + 1),
                                        val(c, r + 2, ch + 2), val(c, r + 3, ch + 3));
                } else {
                    for (int e = 0; e < 4; e++)
                        if (ch + e < dv) dst[ch + e] = val(c, r + e, ch + e);
                }
            }
    };
    if (row >= R) return;
    if (g.o12)
        store(g.o12 + (out * 2 + map) * dv, [&](int c, int r, int) { return o[c][r]; });
    if (map == 1) return;
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            o[c][r] = o[c][r] - lam * ex[(c * 16 + r) * 64 + lane];
            ss += o[c][r] * o[c][r];
        }
    float rn = 1.0f;
    if (g.gain) {
        ss += __shfl_xor(ss, 32, 64);
        rn = (1.0f / sqrtf(ss / (float)dv + g.eps)) * (1.0f - g.lam_init);
        store(g.y + out * dv, [&](int c, int r, int ch) { return o[c][r] * rn * g.gain[ch]; });
    } else {
        store(g.y + out * dv, [&](int c, int r, int) { return o[c][r]; });
    }
}

// The splits of diff_fwd_kernel joined: one wave per (image, query, head); lane
// c holds channels c and c + 64.  Each map: M = max of the splits' maxima,
// weights l_s 2^(m_s - M), in split order.
__global__ __launch_bounds__(256) void diff_join_kernel(DiffArgs g, int splits) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + wave_index();
    if (w >= (long long)g.n * g.tq * g.h) return;
    const int hd = (int)(w % g.h), dv = 2 * g.dh;
    float o[2][2], st[4];
#pragma unroll
    for (int mp = 0; mp < 2; mp++) {
        float M = NO_MAX;
        for (int s0 = 0; s0 < splits; s0 += 64) {
            const int s = s0 + lane;
            if (s < splits) {
                const f2 v = *(const f2 *)(g.pstat + ((w * splits + s) * 2 + mp) * 2);
                if (v[1] > 0.f) M = fmaxf(M, v[0]);
            }
        }
        M = wave_max(M);
        float tot = 0.f;
        o[mp][0] = o[mp][1] = 0.f;
        for (int s = 0; s < splits; s++) {
            const long long at = (w * splits + s) * 2 + mp;
            const f2 v = *(const f2 *)(g.pstat + at * 2);
            const float wt = v[1] > 0.f ? v[1] * __builtin_amdgcn_exp2f(v[0] - M) : 0.f;
            tot += wt;
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (lane + 64 * u < dv)
                    o[mp][u] = __builtin_fmaf(wt, g.part32[at * dv + lane + 64 * u], o[mp][u]);
        }
        const float il = tot > 0.f ? 1.0f / tot : 0.f;
        o[mp][0] *= il;
        o[mp][1] *= il;
        st[2 * mp] = tot > 0.f ? M : 0.f;
        st[2 * mp + 1] = tot > 0.f ? P_UP / tot : 0.f;
    }
    double e1, e2;
    lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
    const float lam = (float)(e1 - e2 + (double)g.lam_init);
    float out[2], ss = 0.f;
    for (int u = 0; u < 2; u++) {
        out[u] = o[0][u] - lam * o[1][u];
        if (lane + 64 * u < dv) ss += out[u] * out[u];
    }
    const float rn = (1.0f / sqrtf(wave_sum(ss) / (float)dv + g.eps)) * (1.0f - g.lam_init);
    for (int u = 0; u < 2; u++) {
        const int c = lane + 64 * u;
        if (c >= dv) continue;
        g.y[w * dv + c] = g.gain ? out[u] * rn * g.gain[c] : out[u];
        if (g.o12) {
            g.o12[(w * 2) * dv + c] = o[0][u];
            g.o12[(w * 2 + 1) * dv + c] = o[1][u];
        }
    }
    if (g.stats && lane == 0) *(float4 *)(g.stats + w * 4) = make_float4(st[0], st[1], st[2], st[3]);
}

// dO and D_1, D_2 of the rows [blk rpb, (blk + 1) rpb) of tokens, and the
// block's partials of dgain and dlambda.
__global__ __launch_bounds__(256) void diff_bwd_pre_kernel(DiffArgs g) {
    extern __shared__ double sh[];  // [4][2 dh + h]
    const int lane = threadIdx.x & 63, wv = wave_index(), dv = 2 * g.dh, cols = dv + g.h;
    double dg[2] = {0.0, 0.0};
    const int rows = g.n * g.tq, r0 = (int)blockIdx.x * g.rpb, r1 = min(rows, r0 + g.rpb);
    for (int hd = 0; hd < g.h; hd++) {
        double e1, e2;
        lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
        const float lam = (float)(e1 - e2 + (double)g.lam_init);
        double dl = 0.0;
        for (int row = r0 + wv; row < r1; row += 4) {
            const long long w = (long long)row * g.h + hd;
            const int b = row / g.tq, i = row % g.tq;
            const bool live = i < len_of(g.qlen, b, g.tq);
            float o1[2], o2[2], o[2], dy[2], t[2], ss = 0.f;
            for (int u = 0; u < 2; u++) {
                const int c = lane + 64 * u;
                const bool in = live && c < dv;
                o1[u] = in ? g.o12c[(w * 2) * dv + c] : 0.f;
                o2[u] = in ? g.o12c[(w * 2 + 1) * dv + c] : 0.f;
                dy[u] = in ? g.dy[w * dv + c] : 0.f;
                o[u] = o1[u] - lam * o2[u];
                ss += o[u] * o[u];
            }
            float d[2];
            if (g.gain) {
                const float r = 1.0f / sqrtf(wave_sum(ss) / (float)dv + g.eps);
                float s = 0.f;
                for (int u = 0; u < 2; u++) {
                    const int c = lane + 64 * u;
                    o[u] *= r;
                    t[u] = c < dv ? dy[u] * (g.gain[c] * (1.0f - g.lam_init)) : 0.f;
                    s += t[u] * o[u];
                    dg[u] += (double)(dy[u] * o[u]);
                }
                s = wave_sum(s) / (float)dv;
                for (int u = 0; u < 2; u++) d[u] = r * (t[u] - o[u] * s);
            } else {
                for (int u = 0; u < 2; u++) d[u] = dy[u];
            }
            float d1 = 0.f, d2 = 0.f;
            for (int u = 0; u < 2; u++) {
                const int c = lane + 64 * u;
                if (c < dv) g.dout[w * dv + c] = d[u];
                d1 += d[u] * o1[u];
                d2 += d[u] * o2[u];
            }
            d1 = wave_sum(d1);
            d2 = wave_sum(d2);
            if (lane == 0) {
                g.dd[w * 2] = d1;
                g.dd[w * 2 + 1] = d2;
            }
            dl += (double)d2;
        }
        if (lane == 0) sh[wv * cols + dv + hd] = -dl;
    }
    for (int u = 0; u < 2; u++)
        if (lane + 64 * u < dv)
            sh[wv * cols + lane + 64 * u] = dg[u] * (double)(1.0f - g.lam_init);
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 256)
        g.part[(long long)blockIdx.x * cols + c] =
            sh[c] + sh[cols + c] + sh[2 * cols + c] + sh[3 * cols + c];
}

// dgain and dlam from the blocks' partials: the block's 16 groups of rows
// each in order, then the groups in order.  Block 0 takes lambda's columns,
// block 1 + i the gain's columns [16 i, 16 i + 16).
__global__ __launch_bounds__(256) void diff_bwd_params_kernel(const double *__restrict__ part,
                                                              int nblk, const float *lam,
                                                              int lam_heads, int dh, int h,
                                                              float *dlam, float *dgain) {
    __shared__ double red[16][16];
    __shared__ double tot[16];
    const int dv = 2 * dh, cols = dv + h, jl = threadIdx.x % 16, q = threadIdx.x / 16;
    const int lane = threadIdx.x & 63, wv = wave_index();
    const int per = (nblk + 15) / 16, k0 = min(nblk, q * per), k1 = min(nblk, k0 + per);
    const bool gain = blockIdx.x > 0;
    const int first = gain ? 16 * ((int)blockIdx.x - 1) : 0, end = gain ? dv : h;
    // a shared lambda's gradient: the heads' in order
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    double shared_dl = 0.0;
    for (int j0 = first; j0 < (gain ? first + 1 : end); j0 += 16) {
        const int j = j0 + jl;
        double s = 0.0;
        if (j < end)
            for (int k = k0; k < k1; k++) s += part[(long long)k * cols + (gain ? j : dv + j)];
        red[q][jl] = s;
        __syncthreads();
        if (q == 0) {
            double t = 0.0;
            for (int u = 0; u < 16; u++) t += red[u][jl];
            tot[jl] = t;
            if (gain && j < end) dgain[j] += (float)t;
        }
        __syncthreads();
        if (!gain) {
            if (lam_heads == 1) {
                for (int u = 0; u < 16 && j0 + u < h; u++) shared_dl += tot[u];
            } else {
                for (int u = wv; u < 16 && j0 + u < h; u += 4) {
                    double e1, e2;
                    lambda_terms(lam, lam_heads, dh, j0 + u, &e1, &e2);
                    const float *l = lam + (long long)(j0 + u) * 4 * dh;
                    float *d = dlam + (long long)(j0 + u) * 4 * dh;
                    if (lane < dh) {
                        d[lane] += (float)(tot[u] * e1 * l[dh + lane]);
                        d[dh + lane] += (float)(tot[u] * e1 * l[lane]);
                        d[2 * dh + lane] -= (float)(tot[u] * e2 * l[3 * dh + lane]);
                        d[3 * dh + lane] -= (float)(tot[u] * e2 * l[2 * dh + lane]);
                    }
                }
            }
        }
        __syncthreads();
    }
    (void)acc;
    if (!gain && lam_heads == 1 && wv == 0) {
        double e1, e2;
        lambda_terms(lam, 1, dh, 0, &e1, &e2);
        if (lane < dh) {
            const double t = shared_dl;
            dlam[lane] += (float)(t * e1 * lam[dh + lane]);
            dlam[dh + lane] += (float)(t * e1 * lam[lane]);
            dlam[2 * dh + lane] -= (float)(t * e2 * lam[3 * dh + lane]);
            dlam[3 * dh + lane] -= (float)(t * e2 * lam[2 * dh + lane]);
        }
    }
}

// dQ of one (image, query, head) a wave.
__global__ __launch_bounds__(256) void diff_dq_row_kernel(DiffArgs g) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + wave_index();
    if (w >= (long long)g.n * g.tq * g.h) return;
    const int hd = (int)(w % g.h);
    const long long row = w / g.h;
    const int i = (int)(row % g.tq), b = (int)(row / g.tq);
    const Seen see(g, b);
    const float *q = g.q + row * g.qstride + 2 * hd * g.dh;
    const float *kv = g.kv + (long long)b * g.tk * g.kvstride;
    const int kh = hd / g.group, dv = 2 * g.dh;
    const float *k0 = kv + g.koff + 2 * kh * g.dh, *v0 = kv + g.voff + kh * dv;
    const float4 st = *(const float4 *)(g.statsc + w * 4);
    double e1, e2;
    lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
    const float lam = (float)(e1 - e2 + (double)g.lam_init);
    const float d1 = g.dd[w * 2], d2 = g.dd[w * 2 + 1];
    const float *dout = g.dout + w * dv;
    float acc[2][1] = {{0.f}, {0.f}};
    const int last = i < see.nq ? (g.causal ? min(see.nk, i + see.shift + 1) : see.nk) : 0;
    for (int j0 = 0; j0 < last; j0 += 64) {
        const int j = j0 + lane;
        const bool in = see(i, j);
        const long long off = (long long)min(j, see.nk - 1) * g.kvstride;
        float s1 = 0.f, s2 = 0.f, da = 0.f;
        for (int c = 0; c < g.dh; c++) {
            s1 = __builtin_fmaf(q[c], k0[off + c], s1);
            s2 = __builtin_fmaf(q[g.dh + c], k0[off + g.dh + c], s2);
        }
        for (int c = 0; c < dv; c++) da = __builtin_fmaf(dout[c], v0[off + c], da);
        const float p1 = in ? exp2f(s1 * (g.scale * LOG2E) - st.x) * st.y : 0.f;
        const float p2 = in ? exp2f(s2 * (g.scale * LOG2E) - st.z) * st.w : 0.f;
        const float ds1 = in ? p1 * (da - d1) * g.scale : 0.f;
        const float ds2 = in ? -lam * p2 * (da - d2) * g.scale : 0.f;
        const int cnt = min(64, last - j0);
        for (int t = 0; t < cnt; t++) {
            const float a = __shfl(ds1, t, 64), c2 = __shfl(ds2, t, 64);
            const float *kr = k0 + (long long)(j0 + t) * g.kvstride;
            if (lane < g.dh && see(i, j0 + t)) {
                acc[0][0] = __builtin_fmaf(a, kr[lane], acc[0][0]);
                acc[1][0] = __builtin_fmaf(c2, kr[g.dh + lane], acc[1][0]);
            }
        }
    }
    float *dq = g.dq + row * g.qstride + 2 * hd * g.dh;
    if (lane < g.dh)
        for (int m = 0; m < 2; m++) {
            float *p = dq + m * g.dh + lane;
            *p = g.acc_q ? *p + acc[m][0] : acc[m][0];
        }
}

// dK and dV of one (image, key, key head) a wave.
__global__ __launch_bounds__(256) void diff_dkv_row_kernel(DiffArgs g) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + wave_index();
    if (w >= (long long)g.n * g.tk * g.hkv) return;
    const int kh = (int)(w % g.hkv);
    const long long row = w / g.hkv;
    const int j = (int)(row % g.tk), b = (int)(row / g.tk);
    const Seen see(g, b);
    const int dv = 2 * g.dh;
    const float *k = g.kv + row * g.kvstride + g.koff + 2 * kh * g.dh;
    const float *v = g.kv + row * g.kvstride + g.voff + kh * dv;
    float dk[2] = {0.f, 0.f}, dvv[2] = {0.f, 0.f};
    const int from = g.causal ? max(0, j - see.shift) : 0, last = j < see.nk ? see.nq : 0;
    for (int hd = kh * g.group; hd < (kh + 1) * g.group; hd++) {
        double e1, e2;
        lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
        const float lam = (float)(e1 - e2 + (double)g.lam_init);
        for (int i0 = from; i0 < last; i0 += 64) {
            const int i = i0 + lane, ic = min(i, see.nq - 1);
            const bool in = see(i, j);
            const long long qr = (long long)b * g.tq + ic, wr = qr * g.h + hd;
            const float *q = g.q + qr * g.qstride + 2 * hd * g.dh;
            const float4 st = *(const float4 *)(g.statsc + wr * 4);
            const float *dout = g.dout + wr * dv;
            float s1 = 0.f, s2 = 0.f, da = 0.f;
            for (int c = 0; c < g.dh; c++) {
                s1 = __builtin_fmaf(q[c], k[c], s1);
                s2 = __builtin_fmaf(q[g.dh + c], k[g.dh + c], s2);
            }
            for (int c = 0; c < dv; c++) da = __builtin_fmaf(dout[c], v[c], da);
            const float p1 = in ? exp2f(s1 * (g.scale * LOG2E) - st.x) * st.y : 0.f;
            const float p2 = in ? exp2f(s2 * (g.scale * LOG2E) - st.z) * st.w : 0.f;
            const float a = p1 - lam * p2;
            const float ds1 = in ? p1 * (da - g.dd[wr * 2]) * g.scale : 0.f;
            const float ds2 = in ? -lam * p2 * (da - g.dd[wr * 2 + 1]) * g.scale : 0.f;
            const int cnt = min(64, last - i0);
            for (int t = 0; t < cnt; t++) {
                const float at = __shfl(a, t, 64), x1 = __shfl(ds1, t, 64), x2 = __shfl(ds2, t, 64);
                const long long qt = (long long)b * g.tq + i0 + t;
                const float *qq = g.q + qt * g.qstride + 2 * hd * g.dh;
                const float *dd = g.dout + (qt * g.h + hd) * dv;
                if (lane < g.dh) {
                    dk[0] = __builtin_fmaf(x1, qq[lane], dk[0]);
                    dk[1] = __builtin_fmaf(x2, qq[g.dh + lane], dk[1]);
                }
                for (int u = 0; u < 2; u++)
                    if (lane + 64 * u < dv) dvv[u] = __builtin_fmaf(at, dd[lane + 64 * u], dvv[u]);
            }
        }
    }
    float *dkp = g.dkv + row * g.kvstride + g.koff + 2 * kh * g.dh;
    float *dvp = g.dkv + row * g.kvstride + g.voff + kh * dv;
    for (int u = 0; u < 2; u++) {
        if (lane < g.dh) {
            float *p = dkp + u * g.dh + lane;
            *p = g.acc_kv ? *p + dk[u] : dk[u];
        }
        if (lane + 64 * u < dv) {
            float *p = dvp + lane + 64 * u;
            *p = g.acc_kv ? *p + dvv[u] : dvv[u];
        }
    }
}

// Token rows of a block of the backward's first pass, and its blocks: at most
// 1024, four rows or more each.
int pre_rows(size_t rows) { return (int)std::max<size_t>(4, rnn_div_up(rows, 1024)); }

// Row groups of 32 a workgroup of the forward, and the splits of the keys: a
// power of two of groups up to four, keys split where the rows leave CUs idle.
struct FwdPlan {
    int qg, splits, split_keys;
    size_t blocks;
};
FwdPlan plan_fwd(const rnn_diff_attn_desc *d, size_t n, bool vec) {
    FwdPlan p;
    const size_t R = (size_t)d->tq * (d->h / d->hkv), probs = n * d->hkv;
    p.qg = !vec ? 4 : R <= 32 ? 1 : R <= 64 ? 2 : 4;
    p.blocks = probs * rnn_div_up(R, (size_t)32 * p.qg);
    const size_t tiles = rnn_div_up(d->tk, (size_t)64);
    size_t s = p.blocks ? std::min(tiles / 4, 512 / p.blocks) : 1;
    s = std::max<size_t>(1, std::min<size_t>(s, 256));
    const size_t per = rnn_div_up(std::max<size_t>(tiles, 1), s);
    p.split_keys = (int)per * 64;
    p.splits = (int)rnn_div_up(std::max<size_t>(tiles, 1), per);
    return p;
}

struct DiffWs {
    size_t part32 = 0, pstat = 0, dout = 0, dd = 0, part = 0, bytes = 0;
};

DiffWs plan_ws(const rnn_diff_attn_desc *d, size_t n, bool backward) {
    DiffWs w;
    WsCarve cv;
    const size_t rows = n * d->tq, heads = rows * d->h;
    if (backward) {
        w.dout = cv.take(heads * 2 * d->dh * sizeof(float));
        w.dd = cv.take(heads * 2 * sizeof(float));
        const size_t nblk = rows ? rnn_div_up(rows, (size_t)pre_rows(rows)) : 0;
        w.part = cv.take(nblk * (2 * d->dh + d->h) * sizeof(double));
    } else {
        // whichever alignment the operands turn out to have
        const int splits = std::max(plan_fwd(d, n, true).splits, plan_fwd(d, n, false).splits);
        if (splits > 1) {
            w.part32 = cv.take(heads * splits * 4 * d->dh * sizeof(float));
            w.pstat = cv.take(heads * splits * 4 * sizeof(float));
        }
    }
    w.bytes = cv.off;
    return w;
}

int diff_check(rnn_ctx *ctx, const rnn_diff_attn_desc *d, size_t n) {
    if (!d) return rnn_fail(ctx, RNN_E_NULL, "diff_attn: desc is null");
    if (!d->h || !d->hkv || !d->dh) return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: zero heads or channels");
    if (d->h % d->hkv)
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: %u heads over %u key heads", d->h, d->hkv);
    if (d->lam_heads != 1 && d->lam_heads != d->h)
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: lam_heads %u (1 or %u)", d->lam_heads, d->h);
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale))
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: scale %g", (double)d->scale);
    if (!(d->lam_init >= 0.0f) || !(d->lam_init < 1.0f) || !(d->eps > 0.0f) || !std::isfinite(d->eps))
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: lam_init %g, eps %g", (double)d->lam_init,
                        (double)d->eps);
    if (d->dh > MAX_DH) return rnn_fail(ctx, RNN_E_UNSUPPORTED, "diff_attn: dh %u above 64", d->dh);
    if (d->h > 1024) return rnn_fail(ctx, RNN_E_UNSUPPORTED, "diff_attn: %u heads above 1024", d->h);
    const size_t qw = (size_t)2 * d->h * d->dh, kw = (size_t)2 * d->hkv * d->dh;
    if (d->qoff > d->qstride || d->qstride - d->qoff < qw || d->koff > d->kvstride ||
        d->kvstride - d->koff < kw || d->voff > d->kvstride || d->kvstride - d->voff < kw)
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: heads do not fit a row");
    if (d->koff < d->voff + kw && d->voff < d->koff + kw)
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: keys and values overlap");
    const size_t lim = 0x7fffffffu;
    if (n > lim || d->tq > (1u << 26) || d->tk > (1u << 26) || d->kvstride > (1u << 22) || d->qstride > (1u << 22) ||
        (d->tq && n > lim / d->tq) || (d->tk && n > lim / d->tk) ||
        n * std::max(d->tq, d->tk) > lim / d->h)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "diff_attn: too many rows");
    return RNN_OK;
}

void fill_args(DiffArgs &g, const rnn_diff_attn_desc *d, size_t n, const float *q, const float *kv,
               const float *lam, const float *gain, const uint32_t *qlen, const uint32_t *klen) {
    g = DiffArgs{};
    g.q = q ? q + d->qoff : nullptr;
    g.kv = kv;
    g.lam = lam;
    g.gain = gain;
    g.qlen = qlen;
    g.klen = klen;
    g.qstride = (long long)d->qstride;
    g.kvstride = (long long)d->kvstride;
    g.n = (int)n;
    g.h = (int)d->h;
    g.hkv = (int)d->hkv;
    g.dh = (int)d->dh;
    g.tq = (int)d->tq;
    g.tk = (int)d->tk;
    g.koff = (int)d->koff;
    g.voff = (int)d->voff;
    g.lam_heads = (int)d->lam_heads;
    g.diag = d->mask_diag ? 1 : 0;
    g.causal = d->causal ? 1 : 0;
    g.group = (int)(d->h / d->hkv);
    g.scale = d->scale;
    g.lam_init = d->lam_init;
    g.eps = d->eps;
}

// float4 accesses: every head of queries, keys, values and outputs starts on 16
// bytes and is whole float4s long.
bool rows_vec(const DiffArgs &g) {
    auto al = [](const void *p) { return ((uintptr_t)p & 15) == 0; };
    return g.dh % 4 == 0 && g.qstride % 4 == 0 && g.kvstride % 4 == 0 && g.koff % 4 == 0 &&
           g.voff % 4 == 0 && al(g.q) && al(g.kv) && al(g.y) && al(g.o12) && al(g.o12c) &&
           al(g.dy) && al(g.dq) && al(g.dkv);
}

template <int DHP, bool VEC, int QG>
void launch_fwd_qg(rnn_ctx *ctx, const DiffArgs &g, const FwdPlan &p) {
    const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
    if (p.splits > 1)
        diff_fwd_kernel<DHP, VEC, QG, true><<<grid, 128 * QG, 0, ctx->stream>>>(g);
    else
        diff_fwd_kernel<DHP, VEC, QG, false><<<grid, 128 * QG, 0, ctx->stream>>>(g);
}
template <int DHP>
void launch_fwd(rnn_ctx *ctx, const DiffArgs &g, const FwdPlan &p, bool vec) {
    if (!vec)
        launch_fwd_qg<DHP, false, 4>(ctx, g, p);
    else if (p.qg == 1)
        launch_fwd_qg<DHP, true, 1>(ctx, g, p);
    else if (p.qg == 2)
        launch_fwd_qg<DHP, true, 2>(ctx, g, p);
    else
        launch_fwd_qg<DHP, true, 4>(ctx, g, p);
}

int check_ws(rnn_ctx *ctx, const DiffWs &w, const void *ws, size_t ws_bytes) {
    if (!w.bytes) return RNN_OK;
    if (!ws) return rnn_fail(ctx, RNN_E_NULL, "diff_attn: workspace is null");
    if (ws_bytes < w.bytes)
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: workspace of %zu bytes, needs %zu", ws_bytes,
                        w.bytes);
    if ((uintptr_t)ws & 255) return rnn_fail(ctx, RNN_E_INVALID, "diff_attn: workspace not 256-byte aligned");
    return RNN_OK;
}

}  // namespace

extern "C" {

int rnn_diff_attn_workspace(const rnn_diff_attn_desc *d, size_t n, int backward, size_t *bytes) {
    const int rc = diff_check(nullptr, d, n);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    *bytes = plan_ws(d, n, backward != 0).bytes;
    return RNN_OK;
}

int rnn_diff_attn_forward(rnn_ctx *ctx, const rnn_diff_attn_desc *d, size_t n, const float *q,
                          const float *kv, const float *lam, const float *gain,
                          const uint32_t *qlen, const uint32_t *klen, void *ws, size_t ws_bytes,
                          float *y, float *o12, float *stats) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = diff_check(ctx, d, n);
    if (rc) return rc;
    if (!n || !d->tq) return RNN_OK;
    if (!q || (d->tk && !kv) || !lam || !y)
        return rnn_fail(ctx, RNN_E_NULL, "diff_attn_forward: null operand");
    if (!o12 != !stats)
        return rnn_fail(ctx, RNN_E_NULL, "diff_attn_forward: o12 and stats are kept together");
    const DiffWs w = plan_ws(d, n, false);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    if ((uintptr_t)stats & 15) return rnn_fail(ctx, RNN_E_INVALID, "diff_attn_forward: stats not 16-byte aligned");
    RNN_ON_DEVICE(ctx);
    DiffArgs g;
    fill_args(g, d, n, q, kv, lam, gain, qlen, klen);
    g.y = y;
    g.o12 = o12;
    g.stats = stats;
    const bool vec = rows_vec(g);
    const FwdPlan p = plan_fwd(d, n, vec);
    g.split_keys = p.split_keys;
    if (p.splits > 1) {
        g.part32 = (float *)((char *)ws + w.part32);
        g.pstat = (float *)((char *)ws + w.pstat);
    }
    switch ((g.dh + 15) / 16) {
        case 1: launch_fwd<16>(ctx, g, p, vec); break;
        case 2: launch_fwd<32>(ctx, g, p, vec); break;
        case 3: launch_fwd<48>(ctx, g, p, vec); break;
        default: launch_fwd<64>(ctx, g, p, vec); break;
    }
    RNN_LAUNCHED(ctx);
    if (p.splits > 1) {
        diff_join_kernel<<<(unsigned)rnn_div_up(n * d->tq * d->h, 4), 256, 0, ctx->stream>>>(
            g, p.splits);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

int rnn_diff_attn_backward(rnn_ctx *ctx, const rnn_diff_attn_desc *d, size_t n, const float *q,
                           const float *kv, const float *lam, const float *gain,
                           const uint32_t *qlen, const uint32_t *klen, const float *o12,
                           const float *stats, const float *dy, void *ws, size_t ws_bytes,
                           float *dq, float *dkv, float *dlam, float *dgain, uint32_t flags) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = diff_check(ctx, d, n);
    if (rc) return rc;
    if (flags & ~(uint32_t)(RNN_ATTN_SET_DQ | RNN_ATTN_SET_DKV))
        return rnn_fail(ctx, RNN_E_INVALID, "diff_attn_backward: unknown flags 0x%x", flags);
    if (!n || (!d->tq && !d->tk)) return RNN_OK;
    if ((d->tq && (!q || !o12 || !stats || !dy || !dq)) || (d->tk && (!kv || !dkv)) || !lam || !dlam)
        return rnn_fail(ctx, RNN_E_NULL, "diff_attn_backward: null operand");
    if (!gain != !dgain)
        return rnn_fail(ctx, RNN_E_NULL, "diff_attn_backward: gain and dgain go together");
    if ((uintptr_t)stats & 15) return rnn_fail(ctx, RNN_E_INVALID, "diff_attn_backward: stats not 16-byte aligned");
    const DiffWs w = plan_ws(d, n, true);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    DiffArgs g;
    fill_args(g, d, n, q, kv, lam, gain, qlen, klen);
    g.dy = dy;
    g.o12c = o12;
    g.statsc = stats;
    g.dq = dq ? dq + d->qoff : nullptr;
    g.dkv = dkv;
    g.dout = (float *)((char *)ws + w.dout);
    g.dd = (float *)((char *)ws + w.dd);
    g.part = (double *)((char *)ws + w.part);
    g.acc_q = (flags & RNN_ATTN_SET_DQ) ? 0 : 1;
    g.acc_kv = (flags & RNN_ATTN_SET_DKV) ? 0 : 1;
    const size_t rows = n * d->tq;
    if (rows) {
        g.rpb = pre_rows(rows);
        const unsigned nblk = (unsigned)rnn_div_up(rows, (size_t)g.rpb);
        const int cols = 2 * g.dh + g.h;
        diff_bwd_pre_kernel<<<nblk, 256, 4 * cols * sizeof(double), ctx->stream>>>(g);
        RNN_LAUNCHED(ctx);
        diff_bwd_params_kernel<<<1 + (gain ? (unsigned)rnn_div_up(2 * g.dh, 16) : 0u), 256, 0,
                                 ctx->stream>>>(g.part, (int)nblk, lam, g.lam_heads, g.dh, g.h,
                                                dlam, dgain);
        RNN_LAUNCHED(ctx);
        diff_dq_row_kernel<<<(unsigned)rnn_div_up(rows * d->h, 4), 256, 0, ctx->stream>>>(g);
        RNN_LAUNCHED(ctx);
    }
    if (d->tk) {
        diff_dkv_row_kernel<<<(unsigned)rnn_div_up(n * d->tk * d->hkv, 4), 256, 0, ctx->stream>>>(g);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

}  // extern "C"
