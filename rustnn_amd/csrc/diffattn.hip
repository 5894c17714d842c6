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
    float *rec;   // [n][tq][h][8]: the forward's stats, D_1, D_2, |dO|, lambda
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
    static constexpr int most = fit >= 64 ? 64 : fit >= 32 ? 32 : fit >= 16 ? 16 : fit >= 8 ? 8 : 4;
    static constexpr int RPP = most < ROWS ? most : ROWS;
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

// Tiles of TK keys and values on their way to LDS: a thread's share in registers
// from its loads on.
template <int DHP, int TK, int NT, bool VEC>
struct KvStage {
    static constexpr int W = 2 * DHP;
    using Tile = HalfTile<TK, W>;
    using Stage = StagePlan<TK, W, NT>;
    static constexpr int CH = Stage::PASSES;
    float xk[CH][8], xv[CH][8];
    const float *kp, *vp;
    long long stride;
    uint32_t koff, voff, step;
    int kend, klim, vlim, sc, sr;
    // The thread's channels [sc, sc + 8) of rows sr, sr + RPP, ...; keys: two
    // runs of dh padded to DHP, values: one of 2 dh.
    __device__ __forceinline__ KvStage(const DiffArgs &g, int b, int kh, int kend_) : kend(kend_) {
        const float *kv = g.kv + (long long)b * g.tk * g.kvstride;
        kp = kv + g.koff + 2 * kh * g.dh;
        vp = kv + g.voff + 2 * kh * g.dh;
        stride = g.kvstride;
        sc = (int)threadIdx.x % Stage::C8 * 8;
        sr = (int)threadIdx.x / Stage::C8;
        const int run = sc >= DHP ? 1 : 0;
        klim = stager() ? g.dh - (sc - run * DHP) : 0;
        vlim = stager() ? 2 * g.dh - sc : 0;
        koff = sr * (uint32_t)stride + sc - run * (DHP - g.dh);
        voff = sr * (uint32_t)stride + sc;
        step = Stage::RPP * (uint32_t)stride;
    }
    __device__ __forceinline__ bool stager() const { return Stage::ALL || sr < Stage::RPP; }
    __device__ __forceinline__ void load(int k0) {
        // rows from kend on are past the resource's end
        const uint32_t bytes = (uint32_t)min(kend - k0, TK) * (uint32_t)stride * 4;
        const auto rk = make_rsrc(kp + k0 * stride, bytes), rv = make_rsrc(vp + k0 * stride, bytes);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            load8<VEC>(rk, koff + i * step, klim, xk[i]);
            load8<VEC>(rv, voff + i * step, vlim, xv[i]);
        }
    }
    __device__ __forceinline__ void maxima(float *mk, float *mv) const {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            a = absmax8(xk[i], a);
            b = absmax8(xv[i], b);
        }
        a = wave_max(a);
        b = wave_max(b);
        if ((threadIdx.x & 63) == 0) {
            mk[wave_index()] = a;
            mv[wave_index()] = b;
        }
    }
    // K's tile at lds, V's behind it.
    __device__ __forceinline__ void store(_Float16 *lds, float kup, float vup) const {
        if (!stager()) return;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            _Float16 *d = lds + (sr + i * Stage::RPP) * Tile::STRIDE + sc;
            const Half2 hk = half_split(xk[i], kup), hv = half_split(xv[i], vup);
            *(h8 *)d = hk.hi;
            *(h8 *)(d + Tile::PART) = hk.lo;
            *(h8 *)(d + Tile::HALVES) = hv.hi;
            *(h8 *)(d + Tile::HALVES + Tile::PART) = hv.lo;
        }
    }
};

// Channels c0 + {0..3} + 4 lh + 8 j of a row (an accumulator of 32 channels, lane
// = row), below lim, times f (live) or 0, stored or added.
template <bool VEC>
__device__ __forceinline__ void put_channels(float *dst, int lim, int c0, const f32x16 &a, float f,
                                             bool live, int add) {
    const int lh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const int ch = c0 + 2 * r + 4 * lh;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = live ? a[r + e] * f : 0.f;
        if (VEC) {
            if (ch >= lim) continue;
            float4 *d = (float4 *)(dst + ch);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (add) o = *d;
            *d = make_float4(o.x + v[0], o.y + v[1], o.z + v[2], o.w + v[3]);
        } else {
            for (int e = 0; e < 4; e++)
                if (ch + e < lim) dst[ch + e] = add ? dst[ch + e] + v[e] : v[e];
        }
    }
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

    KvStage<DHP, TK, NT, VEC> st(g, b, kh, kend);
    if (ntile) st.load(kbeg);

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
    if (ntile) st.maxima(tmax[0][0], tmax[0][1]);
    const _Float16 *const kt = lds, *const vt = lds + Tile::HALVES;
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
        st.store(lds, kup, vup);
        if (t + 1 < ntile) st.load(k0 + TK);
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
        if (t + 1 < ntile) st.maxima(tmax[(t + 1) & 1][0], tmax[(t + 1) & 1][1]);
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

// Backward's first pass: dO, D_1 and D_2 of the rows [blk rpb, (blk + 1) rpb) of
// tokens, and the block's partials of dgain and dlambda.  One wave per (row,
// head), lane c on channels c and c + 64.  The dots are 64-bit sums: dO is
// perpendicular to O, so that D_2, whose sum dlambda is, is small beside its
// terms.
__global__ __launch_bounds__(256) void diff_bwd_pre_kernel(DiffArgs g) {
    extern __shared__ double sh[];  // [4][2 dh + h]
    const int lane = threadIdx.x & 63, wv = wave_index(), dv = 2 * g.dh, cols = dv + g.h;
    double dg[2] = {0.0, 0.0};
    const int rows = g.n * g.tq, r0 = (int)blockIdx.x * g.rpb, r1 = min(rows, r0 + g.rpb);
    float gain[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; u++)
        if (g.gain && lane + 64 * u < dv) gain[u] = g.gain[lane + 64 * u] * (1.0f - g.lam_init);
    for (int hd = 0; hd < g.h; hd++) {
        double e1, e2;
        lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
        const float lam = (float)(e1 - e2 + (double)g.lam_init);
        double dl = 0.0;
        for (int row = r0 + wv; row < r1; row += 4) {
            const long long w = (long long)row * g.h + hd;
            const int b = row / g.tq, i = row % g.tq;
            const bool live = i < len_of(g.qlen, b, g.tq);
            float o1[2], o2[2], o[2], dy[2], d[2], ss = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int c = lane + 64 * u;
                const bool in = live && c < dv;
                o1[u] = in ? g.o12c[(w * 2) * dv + c] : 0.f;
                o2[u] = in ? g.o12c[(w * 2 + 1) * dv + c] : 0.f;
                dy[u] = in ? g.dy[w * dv + c] : 0.f;
                o[u] = o1[u] - lam * o2[u];
                ss += o[u] * o[u];
                d[u] = dy[u];
            }
            if (g.gain) {
                const float r = 1.0f / sqrtf(wave_sum(ss) / (float)dv + g.eps);
                float s = 0.f;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    o[u] *= r;
                    s += dy[u] * gain[u] * o[u];
                    dg[u] += (double)(dy[u] * o[u]);
                }
                s = wave_sum(s) / (float)dv;
#pragma unroll
                for (int u = 0; u < 2; u++) d[u] = r * (dy[u] * gain[u] - o[u] * s);
            }
            double d1 = 0.0, d2 = 0.0;
            float nd = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int c = lane + 64 * u;
                if (c < dv) g.dout[w * dv + c] = d[u];
                d1 += (double)d[u] * (double)o1[u];
                d2 += (double)d[u] * (double)o2[u];
                nd += d[u] * d[u];
            }
            d1 = rnn_wave_sum_d(d1);
            d2 = rnn_wave_sum_d(d2);
            nd = sqrtf(wave_sum(nd));
            if (lane == 0) {
                const float4 st = live ? *(const float4 *)(g.statsc + w * 4)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
                float4 *rec = (float4 *)(g.rec + w * 8);
                rec[0] = st;
                rec[1] = make_float4((float)d1, (float)d2, nd, lam);
            }
            dl += d2;
        }
        if (lane == 0) sh[wv * cols + dv + hd] = -dl;
    }
#pragma unroll
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

// A bound for 2 |dA| of rows with |dO| <= nd and values of magnitude <= vmax, and
// the power of two that keeps dS below 2^15 under it.
template <int W>
__device__ __forceinline__ float ds_up(float nd, float vmax) {
    constexpr float root = W == 32 ? 5.6568543f : W == 64 ? 8.0f : W == 96 ? 9.7979590f : 11.313709f;
    return up_of(nd * (2.0f * root * vmax));
}

// dQ.  Rows and tiles as in the forward, a wave on both maps of its 32 rows:
// S_m^T = K_m Q_m^T and dA^T = V dO^T (lane = row), dS_m in registers is the
// operand of dQ_m^T = K_m^T dS_m^T.  Each tile's products are summed apart and
// added to the gradient in fp32, which carries the tile's powers of two and
// rounds to nearest (the matrix core's own sum cuts off).
template <int DHP, bool VEC, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DHP <= 32 ? 2 : 1))) void
diff_dq_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TK = 32, NT = 64 * NW, KS = DHP / 16, VS = W / 16;
    constexpr int CT = (DHP + 31) / 32;
    using Tile = HalfTile<TK, W>;
    // (a map's last 32-channel tile may run past the row: into the padding)
    __shared__ __align__(16) _Float16 lds[2 * Tile::HALVES + 32];
    __shared__ float tmax[2][2][NW];
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int R = g.tq * g.group, nrb = (R + 32 * NW - 1) / (32 * NW);
    const long long id = xcd_order(blockIdx.x, gridDim.x);
    const int prob = (int)(id / nrb), rb = nrb - 1 - (int)(id % nrb);
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int row = rb * 32 * NW + wave * 32 + lr;
    const int qi = row / g.group, head = kh * g.group + row % g.group;
    const bool live = qi < nq;
    const int last_q = min(nq - 1, (rb * 32 * NW + 32 * NW - 1) / g.group);
    int kend = g.causal ? min(nk, last_q + shift + 1) : nk;
    if (rb * 32 * NW / g.group >= nq) kend = 0;
    const int ntile = kend > 0 ? (kend + TK - 1) / TK : 0;
    KvStage<DHP, TK, NT, VEC> st(g, b, kh, kend);
    if (ntile) st.load(0);

    // the row's queries, its dO and what the first pass left of it
    Half2 q[2][KS], d[VS];
    float qdown[2], ddown, nd;
    const long long qr = (long long)b * g.tq + min(qi, g.tq - 1);
    const long long at = qr * g.h + head;
    {
        const float *qp = g.q + qr * g.qstride + 2 * head * g.dh;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            float v[KS][8], mx = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int c = 16 * s + 8 * lh;
                load8g<VEC>(qp + m * g.dh + c, live ? g.dh - c : 0, v[s]);
                mx = absmax8(v[s], mx);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float up = up_of(mx);
            qdown[m] = down_of(up) * (g.scale * LOG2E);
#pragma unroll
            for (int s = 0; s < KS; s++) q[m][s] = half_split(v[s], up);
        }
        float v[VS][8], mx = 0.f;
#pragma unroll
        for (int s = 0; s < VS; s++) {
            const int c = 16 * s + 8 * lh;
            load8g<VEC>(g.dout + at * 2 * g.dh + c, live ? 2 * g.dh - c : 0, v[s]);
            mx = absmax8(v[s], mx);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float up = up_of(mx);
        ddown = down_of(up);
#pragma unroll
        for (int s = 0; s < VS; s++) d[s] = half_split(v[s], up);
    }
    float4 sm4 = make_float4(0.f, 0.f, 0.f, 0.f), dd4 = sm4;
    if (live) {
        sm4 = *(const float4 *)(g.rec + at * 8);
        dd4 = *(const float4 *)(g.rec + at * 8 + 4);
    }
    nd = dd4.z;
    f32x16 acc[2][CT];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[m][c][r] = 0.f;
    const int w_first = (rb * 32 * NW + wave * 32) / g.group;
    const int w_last = min(nq - 1, (rb * 32 * NW + wave * 32 + 31) / g.group);
    if (ntile) st.maxima(tmax[0][0], tmax[0][1]);
    const _Float16 *const kt = lds, *const vt = lds + Tile::HALVES;
    for (int t = 0; t < ntile; t++) {
        const int k0 = t * TK;
        __syncthreads();
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            mk = fmaxf(mk, tmax[t & 1][0][i]);
            mv = fmaxf(mv, tmax[t & 1][1][i]);
        }
        const float kup = up_of(mk), vup = up_of(mv);
        st.store(lds, kup, vup);
        if (t + 1 < ntile) st.load(k0 + TK);
        __syncthreads();
        if (w_first < nq && !(g.causal && k0 > w_last + shift)) {
            const bool whole = k0 + TK <= nk && !(g.causal && k0 + TK - 1 > w_first + shift) &&
                               !(g.diag && k0 <= w_last && w_first < k0 + TK);
            const float kdown = down_of(kup);
            const float dup = ds_up<W>(nd, mv), fd = down_of(vup) * ddown * dup;
            f32x16 da;
            {
                f32x16 hh, sm;
#pragma unroll
                for (int r = 0; r < 16; r++) hh[r] = sm[r] = 0.f;
#pragma unroll
                for (int s = 0; s < VS; s++) {
                    const h8 hi = Tile::along(vt, lr, 16 * s + 8 * lh);
                    const h8 lo = Tile::along(vt + Tile::PART, lr, 16 * s + 8 * lh);
                    sm = mm(hi, d[s].lo, sm);
                    hh = mm(hi, d[s].hi, hh);
                    sm = mm(lo, d[s].hi, sm);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) da[r] = (hh[r] + sm[r]) * fd;
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                f32x16 hh, sm;
#pragma unroll
                for (int r = 0; r < 16; r++) hh[r] = sm[r] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const int c = m * DHP + 16 * s + 8 * lh;
                    const h8 hi = Tile::along(kt, lr, c);
                    const h8 lo = Tile::along(kt + Tile::PART, lr, c);
                    sm = mm(hi, q[m][s].lo, sm);
                    hh = mm(hi, q[m][s].hi, hh);
                    sm = mm(lo, q[m][s].hi, sm);
                }
                const float f = kdown * qdown[m], mx = m ? sm4.z : sm4.x, il = m ? sm4.w : sm4.y;
                const float D = (m ? dd4.y : dd4.x) * dup;
                Half2 ds[2];
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int r = 8 * s + i;
                        float p = __builtin_amdgcn_exp2f((hh[r] + sm[r]) * f - mx) * il;
                        if (!whole) {
                            const int j = k0 + 8 * (r >> 2) + 4 * lh + (r & 3);
                            const bool in = j < nk && !(g.causal && j > qi + shift) &&
                                            !(g.diag && j == qi);
                            p = in ? p : 0.f;
                        }
                        e[i] = p * (da[r] - D);
                    }
                    ds[s] = half_split(e, 1.0f);
                }
                const float back = kdown * down_of(dup);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    f32x16 a;
#pragma unroll
                    for (int r = 0; r < 16; r++) a[r] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const h8 hi = Tile::across(kt, 16 * s, m * DHP + 32 * c);
                        const h8 lo = Tile::across(kt + Tile::PART, 16 * s, m * DHP + 32 * c);
                        a = mm(lo, ds[s].hi, a);
                        a = mm(hi, ds[s].lo, a);
                        a = mm(hi, ds[s].hi, a);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        acc[m][c][r] = __builtin_fmaf(a[r], back, acc[m][c][r]);
                }
            }
        }
        if (t + 1 < ntile) st.maxima(tmax[(t + 1) & 1][0], tmax[(t + 1) & 1][1]);
    }
    if (row >= R) return;
    float *dst = g.dq + qr * g.qstride + 2 * head * g.dh;
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const float f = m ? -dd4.w * g.scale : g.scale;
#pragma unroll
        for (int c = 0; c < CT; c++)
            put_channels<VEC>(dst + m * g.dh, g.dh, 32 * c, acc[m][c], f, live, g.acc_q);
    }
}

// dK and dV.  One workgroup of NW waves per (image, key head, 32 NW keys), wave
// w on 32 of them: its keys' and values' parts stay in registers.  Tiles of 32
// rows (queries of the head group) are split into LDS with their records:
// S_m = Q_m K_m^T and dA = dO V^T (lane = key), and P and dS in registers are
// the operands of dV^T = dO^T (P_1 - lambda P_2) and dK_m^T = Q_m^T dS_m.
template <int DHP, bool VEC, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DHP <= 16 ? 2 : 1))) void
diff_dkv_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TR = 32, NT = 64 * NW, KS = DHP / 16, VS = W / 16;
    constexpr int CT = (DHP + 31) / 32, VT = DHP / 16;
    using Tile = HalfTile<TR, W>;
    using Stage = StagePlan<TR, W, NT>;
    constexpr int CH = Stage::PASSES;
    __shared__ __align__(16) _Float16 lds[2 * Tile::HALVES + 32];
    __shared__ __align__(16) float rec[7][TR];  // m1, il1, m2, il2, D1, D2, lambda
    __shared__ float tmax[2][4][NW];  // largest |q|, |dO|, |dO|_2, |lambda|
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int nkb = (g.tk + 32 * NW - 1) / (32 * NW);
    const long long id = xcd_order(blockIdx.x, gridDim.x);
    const int prob = (int)(id / nkb), kb = (int)(id % nkb);
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int w_first = kb * 32 * NW + wave * 32, key = w_first + lr;
    const bool live = key < nk;
    // rows that see some key of the block
    const int first_q = g.causal ? max(0, kb * 32 * NW - shift) : 0;
    const int row_end = kb * 32 * NW < nk ? nq * g.group : 0;
    const int row_beg = min(first_q, nq) * g.group;
    const int ntile = row_end > row_beg ? (row_end - row_beg + TR - 1) / TR : 0;
    const float ginv = 1.0f / (float)g.group;

    float xq[CH][8], xd[CH][8];
    float4 r0 = make_float4(0.f, 0.f, 0.f, 0.f), r1 = r0;
    const int sc = (int)threadIdx.x % Stage::C8 * 8, sr = (int)threadIdx.x / Stage::C8;
    const bool stager = Stage::ALL || sr < Stage::RPP;
    const int run = sc >= DHP ? 1 : 0;
    const float *qimg = g.q + (long long)b * g.tq * g.qstride + 2 * kh * g.group * g.dh;
    const float *dimg = g.dout + ((long long)b * g.tq * g.h + kh * g.group) * 2 * g.dh;
    auto load = [&](int row0) {
        // rows of a tile lie in queries [q0, q0 + 32]; row x of the tile is
        // query q0 + (x0 + x) / group (x0 + x < 32 + group, exact in floats)
        const int q0 = row0 / g.group, x0 = row0 - q0 * g.group;
        const float *qb = qimg + q0 * g.qstride;
        const float *db = dimg + (long long)q0 * g.h * 2 * g.dh;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int x = sr + i * Stage::RPP;
            const int dq = (int)(((float)(x0 + x) + 0.5f) * ginv), hd = x0 + x - dq * g.group;
            const bool in = stager && row0 + x < row_end;
            load8g<VEC>(qb + dq * g.qstride + (2 * hd + run) * g.dh + sc - run * DHP,
                        in ? g.dh - (sc - run * DHP) : 0, xq[i]);
            load8g<VEC>(db + ((long long)dq * g.h + hd) * 2 * g.dh + sc, in ? 2 * g.dh - sc : 0,
                        xd[i]);
        }
        if (threadIdx.x < TR) {
            const int x = (int)threadIdx.x;
            const int dq = (int)(((float)(x0 + x) + 0.5f) * ginv), hd = x0 + x - dq * g.group;
            r0 = r1 = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row0 + x < row_end) {
                const float *rp = g.rec + (((long long)b * g.tq + q0 + dq) * g.h + kh * g.group + hd) * 8;
                r0 = *(const float4 *)rp;
                r1 = *(const float4 *)(rp + 4);
            }
        }
    };
    auto maxima = [&](int slot) {
        float mq = 0.f, md = 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            mq = absmax8(xq[i], mq);
            md = absmax8(xd[i], md);
        }
        mq = wave_max(mq);
        md = wave_max(md);
        const float mn = wave_max(r1.z), ml = wave_max(fabsf(r1.w));
        if (lane == 0) {
            tmax[slot][0][wave] = mq;
            tmax[slot][1][wave] = md;
            tmax[slot][2][wave] = mn;
            tmax[slot][3][wave] = ml;
        }
    };
    if (ntile) load(row_beg);

    // the lane's key and value
    Half2 k[2][KS], v[VS];
    float kdown[2], vdown, vmax;
    const long long krow = (long long)b * g.tk + min(key, g.tk - 1);
    {
        const float *kp = g.kv + krow * g.kvstride + g.koff + 2 * kh * g.dh;
        const float *vp = g.kv + krow * g.kvstride + g.voff + 2 * kh * g.dh;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            float x[KS][8], mx = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int c = 16 * s + 8 * lh;
                load8g<VEC>(kp + m * g.dh + c, live ? g.dh - c : 0, x[s]);
                mx = absmax8(x[s], mx);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float up = up_of(mx);
            kdown[m] = down_of(up) * (g.scale * LOG2E);
#pragma unroll
            for (int s = 0; s < KS; s++) k[m][s] = half_split(x[s], up);
        }
        float x[VS][8];
        vmax = 0.f;
#pragma unroll
        for (int s = 0; s < VS; s++) {
            const int c = 16 * s + 8 * lh;
            load8g<VEC>(vp + c, live ? 2 * g.dh - c : 0, x[s]);
            vmax = absmax8(x[s], vmax);
        }
        vmax = fmaxf(vmax, __shfl_xor(vmax, 32, 64));
        const float up = up_of(vmax);
        vdown = down_of(up);
#pragma unroll
        for (int s = 0; s < VS; s++) v[s] = half_split(x[s], up);
    }
    f32x16 dk[2][CT], dv[VT];
#pragma unroll
    for (int r = 0; r < 16; r++) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int c = 0; c < CT; c++) dk[m][c][r] = 0.f;
#pragma unroll
        for (int c = 0; c < VT; c++) dv[c][r] = 0.f;
    }
    if (ntile) maxima(0);
    const _Float16 *const qt = lds, *const dt = lds + Tile::HALVES;
    for (int t = 0; t < ntile; t++) {
        const int row0 = row_beg + t * TR;
        __syncthreads();
        float mq = 0.f, md = 0.f, mn = 0.f, ml = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            mq = fmaxf(mq, tmax[t & 1][0][i]);
            md = fmaxf(md, tmax[t & 1][1][i]);
            mn = fmaxf(mn, tmax[t & 1][2][i]);
            ml = fmaxf(ml, tmax[t & 1][3][i]);
        }
        const float qup = up_of(mq), dup = up_of(md);
        if (stager) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                _Float16 *p = lds + (sr + i * Stage::RPP) * Tile::STRIDE + sc;
                const Half2 hq = half_split(xq[i], qup), hd = half_split(xd[i], dup);
                *(h8 *)p = hq.hi;
                *(h8 *)(p + Tile::PART) = hq.lo;
                *(h8 *)(p + Tile::HALVES) = hd.hi;
                *(h8 *)(p + Tile::HALVES + Tile::PART) = hd.lo;
            }
        }
        if (threadIdx.x < TR) {
            rec[0][threadIdx.x] = r0.x;
            rec[1][threadIdx.x] = r0.y;
            rec[2][threadIdx.x] = r0.z;
            rec[3][threadIdx.x] = r0.w;
            rec[4][threadIdx.x] = r1.x;
            rec[5][threadIdx.x] = r1.y;
            rec[6][threadIdx.x] = r1.w;
        }
        if (t + 1 < ntile) load(row0 + TR);
        __syncthreads();
        const int tq0 = row0 / g.group, tq1 = min(nq - 1, (row0 + TR - 1) / g.group);
        if (w_first < nk && !(g.causal && w_first > tq1 + shift)) {
            // rows past the last carry il = 0, keys past the last are not stored
            const bool whole = !(g.causal && w_first + 31 > tq0 + shift) &&
                               !(g.diag && w_first <= tq1 && tq0 <= w_first + 31);
            const int x0 = row0 - tq0 * g.group;
            const float qd = down_of(qup), dd = down_of(dup);
            const float up = ds_up<W>(mn, vmax), fd = vdown * dd * up;
            const float lup = up_of(ml) * 0x1p-15f;  // takes lambda below 1
            float p1[16], p2[16], da[16];
            {
                f32x16 hh, sm;
#pragma unroll
                for (int r = 0; r < 16; r++) hh[r] = sm[r] = 0.f;
#pragma unroll
                for (int s = 0; s < VS; s++) {
                    const h8 hi = Tile::along(dt, lr, 16 * s + 8 * lh);
                    const h8 lo = Tile::along(dt + Tile::PART, lr, 16 * s + 8 * lh);
                    sm = mm(hi, v[s].lo, sm);
                    hh = mm(hi, v[s].hi, hh);
                    sm = mm(lo, v[s].hi, sm);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) da[r] = (hh[r] + sm[r]) * fd;
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                f32x16 hh, sm;
#pragma unroll
                for (int r = 0; r < 16; r++) hh[r] = sm[r] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const int c = m * DHP + 16 * s + 8 * lh;
                    const h8 hi = Tile::along(qt, lr, c);
                    const h8 lo = Tile::along(qt + Tile::PART, lr, c);
                    sm = mm(hi, k[m][s].lo, sm);
                    hh = mm(hi, k[m][s].hi, hh);
                    sm = mm(lo, k[m][s].hi, sm);
                }
                const float f = qd * kdown[m];
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const float4 mx = *(const float4 *)&rec[2 * m][2 * r + 4 * lh];
                    const float4 il = *(const float4 *)&rec[2 * m + 1][2 * r + 4 * lh];
                    const float mxv[4] = {mx.x, mx.y, mx.z, mx.w}, ilv[4] = {il.x, il.y, il.z, il.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float p = __builtin_amdgcn_exp2f((hh[r + e] + sm[r + e]) * f - mxv[e]) * ilv[e];
                        if (!whole) {
                            const int i = tq0 + (int)(((float)(x0 + 2 * r + 4 * lh + e) + 0.5f) * ginv);
                            const bool in = !(g.causal && key > i + shift) && !(g.diag && key == i);
                            p = in ? p : 0.f;
                        }
                        (m ? p2 : p1)[r + e] = p;
                    }
                }
            }
            // dV: (P_1 - lambda P_2) times a power of two that no lambda passes
            const float aup = up_of(1.0f + ml), adown = down_of(aup) * dd;
            {
                Half2 a[2];
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 lv = *(const float4 *)&rec[6][2 * (8 * s + i) + 4 * lh];
                        const float l4[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            e[i + j] = p1[8 * s + i + j] - l4[j] * p2[8 * s + i + j];
                    }
                    a[s] = half_split(e, aup);
                }
#pragma unroll
                for (int c = 0; c < VT; c++) {
                    f32x16 x;
#pragma unroll
                    for (int r = 0; r < 16; r++) x[r] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const h8 hi = Tile::across(dt, 16 * s, 32 * c);
                        const h8 lo = Tile::across(dt + Tile::PART, 16 * s, 32 * c);
                        x = mm(lo, a[s].hi, x);
                        x = mm(hi, a[s].lo, x);
                        x = mm(hi, a[s].hi, x);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) dv[c][r] = __builtin_fmaf(x[r], adown, dv[c][r]);
                }
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                Half2 ds[2];
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 Dv = *(const float4 *)&rec[4 + m][2 * (8 * s + i) + 4 * lh];
                        const float4 lv = *(const float4 *)&rec[6][2 * (8 * s + i) + 4 * lh];
                        const float D4[4] = {Dv.x, Dv.y, Dv.z, Dv.w}, l4[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int r = 8 * s + i + j;
                            const float x = (m ? p2 : p1)[r] * (da[r] - D4[j] * up);
                            e[i + j] = m ? x * l4[j] : x;
                        }
                    }
                    ds[s] = half_split(e, m ? lup : 1.0f);
                }
                const float back = (m ? down_of(lup) : 1.0f) * qd * down_of(up);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    f32x16 a;
#pragma unroll
                    for (int r = 0; r < 16; r++) a[r] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const h8 hi = Tile::across(qt, 16 * s, m * DHP + 32 * c);
                        const h8 lo = Tile::across(qt + Tile::PART, 16 * s, m * DHP + 32 * c);
                        a = mm(lo, ds[s].hi, a);
                        a = mm(hi, ds[s].lo, a);
                        a = mm(hi, ds[s].hi, a);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        dk[m][c][r] = __builtin_fmaf(a[r], back, dk[m][c][r]);
                }
            }
        }
        if (t + 1 < ntile) maxima((t + 1) & 1);
    }
    if (key >= g.tk) return;
    float *kd = g.dkv + krow * g.kvstride + g.koff + 2 * kh * g.dh;
    float *vd = g.dkv + krow * g.kvstride + g.voff + 2 * kh * g.dh;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int c = 0; c < CT; c++)
            put_channels<VEC>(kd + m * g.dh, g.dh, 32 * c, dk[m][c], m ? -g.scale : g.scale, live,
                              g.acc_kv);
#pragma unroll
    for (int c = 0; c < VT; c++)
        put_channels<VEC>(vd, 2 * g.dh, 32 * c, dv[c], 1.0f, live, g.acc_kv);
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
    size_t part32 = 0, pstat = 0, dout = 0, rec = 0, part = 0, bytes = 0;
};

DiffWs plan_ws(const rnn_diff_attn_desc *d, size_t n, bool backward) {
    DiffWs w;
    WsCarve cv;
    const size_t rows = n * d->tq, heads = rows * d->h;
    if (backward) {
        w.dout = cv.take(heads * 2 * d->dh * sizeof(float));
        w.rec = cv.take(heads * 8 * sizeof(float));
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

// Waves of a workgroup by the rows (or keys) that there are: 32 each, up to four.
int waves_of(size_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

template <int DHP, bool VEC, int NW>
void launch_dq(rnn_ctx *ctx, const DiffArgs &g) {
    const size_t R = (size_t)g.tq * g.group;
    const unsigned grid = (unsigned)((size_t)g.n * g.hkv * rnn_div_up(R, 32 * NW));
    diff_dq_kernel<DHP, VEC, NW><<<grid, 64 * NW, 0, ctx->stream>>>(g);
}
template <int DHP, bool VEC, int NW>
void launch_dkv(rnn_ctx *ctx, const DiffArgs &g) {
    const unsigned grid = (unsigned)((size_t)g.n * g.hkv * rnn_div_up((size_t)g.tk, 32 * NW));
    diff_dkv_kernel<DHP, VEC, NW><<<grid, 64 * NW, 0, ctx->stream>>>(g);
}
template <int DHP>
void launch_bwd(rnn_ctx *ctx, const DiffArgs &g, bool vec) {
    if (g.tq) {
        const int nw = waves_of((size_t)g.tq * g.group);
        if (!vec)
            launch_dq<DHP, false, 4>(ctx, g);
        else if (nw == 1)
            launch_dq<DHP, true, 1>(ctx, g);
        else if (nw == 2)
            launch_dq<DHP, true, 2>(ctx, g);
        else
            launch_dq<DHP, true, 4>(ctx, g);
    }
    if (g.tk) {
        const int nw = waves_of((size_t)g.tk);
        if (!vec)
            launch_dkv<DHP, false, 4>(ctx, g);
        else if (nw == 1)
            launch_dkv<DHP, true, 1>(ctx, g);
        else if (nw == 2)
            launch_dkv<DHP, true, 2>(ctx, g);
        else
            launch_dkv<DHP, true, 4>(ctx, g);
    }
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
    g.rec = (float *)((char *)ws + w.rec);
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
    }
    const bool vec = rows_vec(g);
    switch ((g.dh + 15) / 16) {
        case 1: launch_bwd<16>(ctx, g, vec); break;
        case 2: launch_bwd<32>(ctx, g, vec); break;
        case 3: launch_bwd<48>(ctx, g, vec); break;
        default: launch_bwd<64>(ctx, g, vec); break;
    }
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

}  // extern "C"
