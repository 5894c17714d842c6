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
#include "mfma_half.h"

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
    double *part; // partials of dgain and dlambda, [blocks][2 dh + groups of a block]
    long long qstride, kvstride;
    int n, h, hkv, dh, tq, tk, koff, voff, lam_heads, diag, causal, group;
    int acc_q, acc_kv, split_keys;
    long long first;       // the launch's first block of rows, keys or problems
    int nblk, gpb;         // blocks of the backward's first pass, their groups of lanes
    float *dlam, *dgain;
    float scale, lam_init, eps;
};

__device__ __forceinline__ int len_of(const uint32_t *len, int b, int t) {
    return len ? (int)min(len[b], (uint32_t)t) : t;
}

// lq1 . lk1 and lq2 . lk2 of a head, on every lane, summed in 64 bits.
__device__ __forceinline__ void lambda_dots(const float *lam, int lam_heads, int dh, int head,
                                            double *a, double *b) {
    const int lane = threadIdx.x & 63, c = min(lane, dh - 1);
    const float *l = lam + (lam_heads > 1 ? (long long)head * 4 * dh : 0);
    const float x = l[c], y = l[dh + c], z = l[2 * dh + c], w = l[3 * dh + c];
    *a = rnn_wave_sum_d(lane < dh ? (double)x * (double)y : 0.0);
    *b = rnn_wave_sum_d(lane < dh ? (double)z * (double)w : 0.0);
}

// acc += the rows of a tile times a register operand over channels c0 ..
// c0 + 16 N - 1: accumulator rows are the tile's, columns the operand's lanes.
template <class Tile, int N>
__device__ __forceinline__ void dot_along(const _Float16 *t, int c0, const Half2 (&x)[N], f32x16 &acc) {
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int s = 0; s < N; s++) {
        const h8 hi = Tile::along(t, l & 31, c0 + 16 * s + 8 * (l >> 5));
        const h8 lo = Tile::along(t + Tile::PART, l & 31, c0 + 16 * s + 8 * (l >> 5));
        acc = mm(lo, x[s].hi, acc);
        acc = mm(hi, x[s].lo, acc);
        acc = mm(hi, x[s].hi, acc);
    }
}
// acc += channels c0 .. c0 + 31 of a tile (accumulator rows) times a register
// operand over the tile's first 16 N rows.
template <class Tile, int N>
__device__ __forceinline__ void dot_across(const _Float16 *t, int c0, const Half2 (&x)[N], f32x16 &acc) {
#pragma unroll
    for (int s = 0; s < N; s++) {
        const h8 hi = Tile::across(t, 16 * s, c0), lo = Tile::across(t + Tile::PART, 16 * s, c0);
        acc = mm(lo, x[s].hi, acc);
        acc = mm(hi, x[s].lo, acc);
        acc = mm(hi, x[s].hi, acc);
    }
}

// Tells the scheduler to keep LDS reads AHEAD steps before the products that
// take them, in a block of STEPS steps of READS reads and three products each:
// with one or two waves a SIMD nothing else hides their latency.
template <int STEPS, int READS, int AHEAD>
__device__ __forceinline__ void read_ahead() {
    constexpr int A = AHEAD < STEPS ? AHEAD : STEPS;
    __builtin_amdgcn_sched_group_barrier(0x100, READS * A, 0);
#pragma unroll
    for (int i = 0; i < STEPS - A; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 3, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 3 * A, 0);
}

// A lane's row of 16 N channels (of `lim` channels, zeros past them); the lanes l
// and l + 32 hold it together.  split() makes it an operand, times the power of two
// that its largest magnitude (mx) calls for, whose reciprocal is returned.
template <int N>
struct RowFrag {
    float v[N][8], mx;
    template <bool VEC>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t off, int lim) {
        const int lh = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int s = 0; s < N; s++)
            load8<VEC>(rs, off + 16 * s + 8 * lh, lim - (16 * s + 8 * lh), v[s]);
    }
    __device__ __forceinline__ float split(Half2 (&x)[N]) {
        mx = 0.f;
#pragma unroll
        for (int s = 0; s < N; s++) mx = absmax8(v[s], mx);
        mx = pair32(mx, max2);
        const float up = up_of(mx);
#pragma unroll
        for (int s = 0; s < N; s++) x[s] = half_split(v[s], up);
        return down_of(up);
    }
};
// Softmax values enter the products times 2^6, relative to a reference that a row's
// largest score may pass by 2^8 before it moves: at most 2^14.
constexpr float P_UP = 64.0f, P_EXP = 6.0f, SLACK = 8.0f;
constexpr float NO_MAX = -0x1.fffffep127f;       // a running maximum before any score
constexpr float SQUARES_MAX = 0x1p120f;          // a norm's sum of squares that has not overflowed
constexpr float FAR_SCORE = 0x1p17f;             // a maximum whose own rounding shows in 2^x

// Lambda of a lane's own head: the wave's one head together, else each lane its
// own.
__device__ __forceinline__ float lane_lambda(const DiffArgs &g, int head) {
    double a = 0.0, b = 0.0;
    if (g.lam_heads == 1 || g.group == 1) {
        lambda_dots(g.lam, g.lam_heads, g.dh, __builtin_amdgcn_readfirstlane(head), &a, &b);
    } else {
        const float *l = g.lam + (long long)head * 4 * g.dh;
        for (int c = 0; c < g.dh; c++) {
            a = fma((double)l[c], (double)l[g.dh + c], a);
            b = fma((double)l[2 * g.dh + c], (double)l[3 * g.dh + c], b);
        }
    }
    return expf((float)a) - expf((float)b) + g.lam_init;
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
    int kend, klim, vlim, sc, sr, width;
    // The thread's channels [sc, sc + 8) of rows sr, sr + RPP, ...; keys: two
    // runs of dh padded to DHP, values: one of 2 dh.
    __device__ __forceinline__ KvStage(const DiffArgs &g, int b, int kh, int kend_) : kend(kend_) {
        const float *kv = g.kv + (long long)b * g.tk * g.kvstride;
        kp = kv + g.koff + 2 * kh * g.dh;
        vp = kv + g.voff + 2 * kh * g.dh;
        stride = g.kvstride;
        width = 2 * g.dh;
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
        const int rows = min(kend - k0, TK);
        const auto rk = rows_rsrc(kp + k0 * stride, rows, stride, width);
        const auto rv = rows_rsrc(vp + k0 * stride, rows, stride, width);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            load8<VEC>(rk, koff + i * step, klim, xk[i]);
            load8<VEC>(rv, voff + i * step, vlim, xv[i]);
        }
    }
    // Each wave's largest magnitudes, where one passes what its power of two is good
    // for (else 0: the reductions are rarely taken).
    __device__ __forceinline__ void maxima(f2 *mx, float kgood, float vgood) const {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            a = absmax8(xk[i], a);
            b = absmax8(xv[i], b);
        }
        f2 m = {0.f, 0.f};
        if (__any(a > kgood || b > vgood)) m = f2{wave_max(a), wave_max(b)};
        if ((threadIdx.x & 63) == 0) mx[wave_index()] = m;
    }
    // K's tile at lds, V's `behind` halves further on.
    __device__ __forceinline__ void store(_Float16 *lds, float kup, float vup,
                                          int behind = Tile::HALVES) const {
        if (!stager()) return;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            _Float16 *d = lds + row_pos(sr + i * Stage::RPP) * Tile::STRIDE + sc;
            const Half2 hk = half_split(xk[i], kup), hv = half_split(xv[i], vup);
            *(h8 *)d = hk.hi;
            *(h8 *)(d + Tile::PART) = hk.lo;
            *(h8 *)(d + behind) = hv.hi;
            *(h8 *)(d + behind + Tile::PART) = hv.lo;
        }
    }
};

// Channels c0 + {0..3} + 4 lh + 8 j of a row (an accumulator of 32 channels, lane
// = row), below lim, times f f2 (live) or 0, stored or added.
template <bool VEC>
__device__ __forceinline__ void put_channels(float *dst, int lim, int c0, const f32x16 &a, float f,
                                             float f2, bool live, int add) {
    const int lh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const int ch = c0 + 2 * r + 4 * lh;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = live ? a[r + e] * f * f2 : 0.f;
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
// waves, in two buffers: while one is read the next is written, and the loads of
// the one after it are in flight.  KH: two waves take half of each tile's keys and
// join their sums at the end (wave 2 (QG h + i) + m).
// A tile's chain bounds it (barrier, S, maximum, exponentials, split, P V) with two
// waves a SIMD: 8 heads of 4096 rows and keys over 2 key heads, dh 64, 308 us, 223
// TFLOP/s of fp32 work, the matrix cores busy half of the time (rnn_matmul 168);
// small problems by memory: 128 x 4 heads of 64, dh 32, 19 us (50 MB), 64 rows on 256
// keys 28 us (101 MB).  One query over 4 images of up to 16384 keys, split, 31 us for
// the 100 MB of three quarters of them: 3.2 TB/s, since splits are cut from tk, and
// those past an image's length end at once while the others walk their tiles.
// SPLIT: the keys [z TS, (z + 1) TS) alone (z = blockIdx.y), each map's own
// normalised output, maximum and sum left for diff_join_kernel.
template <int DHP, bool VEC, int QG, int KH, bool SPLIT>
__global__ __launch_bounds__(128 * QG * KH)
__attribute__((amdgpu_waves_per_eu(QG * KH == 4 || (QG == 2 && DHP <= 32) ? 2 : 1))) void
diff_fwd_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TK = QG * KH < 4 && DHP > 32 ? 32 : 64, NT = 128 * QG * KH, KS = DHP / 16;
    constexpr int CT = DHP / 16, S2 = TK / 32 / KH, HALF = (CT * 16 + 3) * 64;
    using Tile = HalfTile<TK, W>;
    static_assert(8 * Tile::HALVES >= 4 * ((KH - 1) * 2 * QG * HALF + QG * CT * 16 * 64) && (KH == 1 || !SPLIT), "exchange");
    __shared__ __align__(16) _Float16 lds[2][2 * Tile::HALVES];
    __shared__ f2 tmax[2][2 * QG * KH];
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int map = wave & 1, qg = (wave >> 1) % QG, half = (wave >> 1) / QG;
    const int R = g.tq * g.group, nrb = (R + 32 * QG - 1) / (32 * QG);
    const long long id = g.first + xcd_order(blockIdx.x, gridDim.x);
    const int prob = (int)(id / nrb), rb = nrb - 1 - (int)(id % nrb);  // causal: longest first
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int row0 = rb * 32 * QG + qg * 32, row = row0 + lr;
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
    // the row's query of this map; the wave's queries
    const int w_first = row0 / g.group, w_last = min(nq - 1, (row0 + 31) / g.group);
    const int q0 = min(w_first, g.tq - 1);
    Half2 q[KS];
    RowFrag<KS> qf;
    qf.template load<VEC>(rows_rsrc(g.q + ((long long)b * g.tq + q0) * g.qstride,
                                    min(g.tq - q0, 32), g.qstride, 2 * g.h * g.dh),
                          (uint32_t)(qi - q0) * (uint32_t)g.qstride + (2 * head + map) * g.dh,
                          live ? g.dh : 0);
    float lam = 0.f;
    if (!SPLIT && map == 0) lam = lane_lambda(g, min(head, g.h - 1));
    const float qdown = qf.split(q) * (g.scale * LOG2E);
    f32x16 o[CT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[c][r] = 0.f;
    // the softmax reference, the sum, and the largest score itself
    float m = NO_MAX, l = 0.f, mtop = NO_MAX;
    // the largest key so far, and powers of two of the tile that is staged; the
    // output is in the values' unit
    float kmax = 0.f, kup1 = 1.f, vup1 = FIRST_UP, vup = FIRST_UP;
    auto maxima = [&](int slot) { st.maxima(tmax[slot], kmax, good_for(vup1)); };
    auto stage = [&](int t) {
        float mv = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * QG * KH; i++) {
            const f2 m = tmax[t & 1][i];
            kmax = max2(kmax, m[0]);
            mv = max2(mv, m[1]);
        }
        kup1 = up_of(kmax);
        vup1 = sticky_up(mv, vup1);
        st.store(lds[t & 1], kup1, vup1);
    };
    if (ntile) {
        maxima(0);
        __syncthreads();
        stage(0);
        if (ntile > 1) {
            st.load(kbeg + TK);
            maxima(1);
        }
    }
    for (int t = 0; t < ntile; t++) {
        const int k0 = kbeg + t * TK, k1 = k0 + 32 * S2 * half;
        __syncthreads();
        const _Float16 *const kt = lds[t & 1] + 32 * S2 * half * Tile::STRIDE, *const vt = kt + Tile::HALVES;
        // (f stays above 0, so that a hidden score, -infinity, stays hidden: where it
        // would be smaller, all scores are 0 to the last bit of an exponential)
        const float f = fmaxf(down_of(kup1) * qdown, 0x1p-120f), turn = down_of(vup) * vup1;
        vup = vup1;
        if (t + 1 < ntile) stage(t + 1);
        if (t + 2 < ntile) st.load(k0 + 2 * TK);
        f32x16 u[S2];
#pragma unroll
        for (int s2 = 0; s2 < S2; s2++) {
#pragma unroll
            for (int r = 0; r < 16; r++) u[s2][r] = 0.f;
            dot_along<Tile>(kt + 32 * s2 * Tile::STRIDE, map * DHP, q, u[s2]);
        }
        const bool whole = k1 + 32 * S2 <= nk && !(g.causal && k1 + 32 * S2 - 1 > w_first + shift) &&
                           !(g.diag && k1 <= w_last && w_first < k1 + 32 * S2);
        if (!whole) {
#pragma unroll
            for (int s2 = 0; s2 < S2; s2++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int j = k1 + 32 * s2 + 8 * (r >> 2) + 4 * lh + (r & 3);
                    const bool in = j < nk && !(g.causal && j > qi + shift) && !(g.diag && j == qi);
                    u[s2][r] = in ? u[s2][r] : -INFINITY;
                }
        }
        float top = u[0][0];
#pragma unroll
        for (int s2 = 0; s2 < S2; s2++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) top = max3(top, u[s2][r], u[s2][r + 1]);
        // (a score times f: f > 0 keeps the order)
        top = pair32(top, max2) * f;
        mtop = max2(mtop, top);
        // the reference moves where a score passes it by the slack, the output's
        // unit where the tile's does; both rarely after the first tile
        const bool moves = top > m + SLACK;
        if (__any(moves || turn != 1.0f)) {
            const float mn = moves ? top : m, al = __builtin_amdgcn_exp2f(m - mn), keep = al * turn;
            m = mn;
            l *= al;
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[c][r] *= keep;
        }
        float fe = f, base = P_EXP - m;
        // far from 0 the reference is taken off the rounded score: off the exact one, as
        // a fused multiply-add does it, what its rounding left would be an exponent
        const bool far = fabsf(m) > FAR_SCORE && m != NO_MAX;
        if (__any(far)) {
#pragma unroll
            for (int s = 0; s < S2; s++)
#pragma unroll
                for (int r = 0; r < 16; r++) u[s][r] = far ? u[s][r] * f - m : u[s][r];
            fe = far ? 1.0f : f;
            base = far ? P_EXP : base;
        }
        Half2 p[2 * S2];
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S2; s++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                u[s][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(u[s][r], fe, base));
                ps[r & 3] += u[s][r];
            }
            split16(u[s], *(Half2(*)[2]) & p[2 * s]);
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
        for (int c = 0; c < CT; c++) dot_across<Tile>(vt, 32 * c, p, o[c]);
        if (t + 2 < ntile) maxima(t & 1);
    }
    l = pair32(l, add2);
    if constexpr (KH > 1) {  // the second half's sums to the first
        static_assert(KH == 2);
        __syncthreads();
        float *const e = (float *)lds[0] + (2 * qg + map) * HALF + lane;
        if (half) {
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++) e[(c * 16 + r) * 64] = o[c][r];
            e[CT * 16 * 64] = m;
            e[CT * 16 * 64 + 64] = l;
            e[CT * 16 * 64 + 128] = mtop;
        }
        __syncthreads();
        if (!half) {
            const float m2 = e[CT * 16 * 64], top = max2(m, m2);
            const float x = __builtin_amdgcn_exp2f(m - top), y = __builtin_amdgcn_exp2f(m2 - top);
            l = l * x + e[CT * 16 * 64 + 64] * y;
            m = top;
            mtop = max2(mtop, e[CT * 16 * 64 + 128]);
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    o[c][r] = __builtin_fmaf(o[c][r], x, e[(c * 16 + r) * 64] * y);
        }
    }
    // whether the row sees a key (of the split): its sum is then above 0, or no number
    // for want of one
    const int seen = min(kend, g.causal ? qi + shift + 1 : nk) - kbeg;
    const bool some = live && seen > (g.diag && qi >= kbeg && qi < kbeg + seen ? 1 : 0);
    const float il = some ? down_of(vup) / l : 0.f;  // both carry 2^6
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[c][r] = some ? o[c][r] * il : 0.f;
    // the statistics kept are relative to the largest score itself, so that the
    // backward's exponentials are at most 1
    l *= __builtin_amdgcn_exp2f(m - mtop);
    m = some ? mtop : 0.f;
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
    if (KH == 1) __syncthreads();
    float *ex = (float *)lds[0] + (KH - 1) * 2 * QG * HALF + qg * CT * 16 * 64;
    if (map == 1 && !half) {
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) ex[(c * 16 + r) * 64 + lane] = o[c][r];
    }
    if (g.stats && row < R && lh == 0 && !half)
        *(f2 *)(g.stats + out * 4 + 2 * map) = f2{m, some ? P_UP / l : 0.f};
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
    if (row >= R || half) return;
    if (g.o12)
        store(g.o12 + (out * 2 + map) * dv, [&](int c, int r, int) { return o[c][r]; });
    if (map == 1) return;
    // (the gain in registers before the stores, which its loads would wait for)
    f32x16 gv[CT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int r = 0; r < 16; r++)
            gv[c][r] = g.gain ? g.gain[min(32 * c + 8 * (r >> 2) + 4 * lh + (r & 3), dv - 1)] : 1.f;
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
        ss = pair32(ss, add2);
        rn = 1.0f / sqrtf(ss / (float)dv + g.eps);
        if (__any(ss > SQUARES_MAX)) {  // again from values 2^-64 their size
            float sm = 0.f;
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float x = o[c][r] * 0x1p-64f;
                    sm += x * x;
                }
            sm = pair32(sm, add2);
            if (ss > SQUARES_MAX) rn = 0x1p-64f / sqrtf(sm / (float)dv + g.eps * 0x1p-128f);
        }
        rn *= 1.0f - g.lam_init;
        store(g.y + out * dv, [&](int c, int r, int) { return o[c][r] * rn * gv[c][r]; });
    } else {
        store(g.y + out * dv, [&](int c, int r, int) { return o[c][r]; });
    }
}

// The splits of diff_fwd_kernel joined, WPR waves per (image, query, head): each
// map's M = max of the splits' maxima, weights l_s 2^(m_s - M).  Lane s holds
// split s's statistics (at most 64 splits); wave w adds the splits w, w + WPR, ...
// in order, eight loads ahead, then the waves' sums are added in order.  Lane c
// holds channels 2 c and 2 c + 1.
template <int WPR>
__global__ __launch_bounds__(256) void diff_join_kernel(DiffArgs g, int splits) {
    __shared__ f2 sums[4][2][64];
    const int lane = threadIdx.x & 63, wave = wave_index(), part = wave % WPR;
    const long long w = (long long)blockIdx.x * (4 / WPR) + wave / WPR;
    const long long total = (long long)g.n * g.tq * g.h;
    if (WPR == 1 && w >= total) return;
    const int hd = (int)(w % g.h), dv = 2 * g.dh;
    const f4 st = lane < splits ? *(const f4 *)(g.pstat + (w * splits + lane) * 4)
                                : f4{NO_MAX, 0.f, NO_MAX, 0.f};
    // (not "above 0": a NaN stays one)
    const bool has0 = !(st[1] <= 0.f), has1 = !(st[3] <= 0.f);
    const float M0 = wave_max(has0 ? st[0] : NO_MAX), M1 = wave_max(has1 ? st[2] : NO_MAX);
    const float w0 = has0 ? st[1] * __builtin_amdgcn_exp2f(st[0] - M0) : 0.f;
    const float w1 = has1 ? st[3] * __builtin_amdgcn_exp2f(st[2] - M1) : 0.f;
    const float t0 = wave_sum(w0), t1 = wave_sum(w1);
    const bool some0 = !(t0 <= 0.f), some1 = !(t1 <= 0.f);
    f2 o0 = {0.f, 0.f}, o1 = o0;
    const int c = 2 * lane;
    // (every lane goes along, since it hands its split's weights to the others; those
    // past the row read its last channels)
    const float *src = g.part32 + w * splits * 2 * dv + min(c, dv - 2);
    for (int s0 = part; s0 < splits; s0 += 8 * WPR) {
        f2 a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long at = (long long)min(s0 + i * WPR, splits - 1) * 2 * dv;
            a[i] = *(const f2 *)(src + at);
            b[i] = *(const f2 *)(src + at + dv);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int s = s0 + i * WPR;
            if (s >= splits) break;
            const float x = __shfl(w0, s, 64), y = __shfl(w1, s, 64);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                o0[e] = __builtin_fmaf(x, a[i][e], o0[e]);
                o1[e] = __builtin_fmaf(y, b[i][e], o1[e]);
            }
        }
    }
    if constexpr (WPR > 1) {
        sums[wave][0][lane] = o0;
        sums[wave][1][lane] = o1;
        __syncthreads();
        if (part) return;
        for (int i = 1; i < WPR; i++) {
            o0 += sums[wave + i][0][lane];
            o1 += sums[wave + i][1][lane];
        }
    }
    o0 *= some0 ? 1.0f / t0 : 0.f;
    o1 *= some1 ? 1.0f / t1 : 0.f;
    const float lam = lane_lambda(g, hd);
    f2 out = o0 - lam * o1;
    float rn = 1.0f;
    f2 gn = {1.f, 1.f};
    if (g.gain) {
        const float ss = wave_sum(c < dv ? out[0] * out[0] + out[1] * out[1] : 0.f);
        rn = 1.0f / sqrtf(ss / (float)dv + g.eps);
        if (ss > SQUARES_MAX) {
            const f2 x = out * 0x1p-64f;
            const float sm = wave_sum(c < dv ? x[0] * x[0] + x[1] * x[1] : 0.f);
            rn = 0x1p-64f / sqrtf(sm / (float)dv + g.eps * 0x1p-128f);
        }
        rn *= 1.0f - g.lam_init;
        if (c < dv) gn = f2{g.gain[c], g.gain[c + 1]};
    }
    if (c < dv) {
        out *= rn;
        *(f2u *)(g.y + w * dv + c) = out * gn;
        if (g.o12) {
            *(f2u *)(g.o12 + (w * 2) * dv + c) = o0;
            *(f2u *)(g.o12 + (w * 2 + 1) * dv + c) = o1;
        }
    }
    if (g.stats && lane == 0)
        *(f4 *)(g.stats + w * 4) = f4{some0 ? M0 : 0.f, some0 ? P_UP / t0 : 0.f,
                                      some1 ? M1 : 0.f, some1 ? P_UP / t1 : 0.f};
}

// Backward's first pass: dO, D_1 and D_2 of every (row, head), and the block's
// partials of dgain and dlambda.  LPU lanes a unit, four channels each (VEC), or a
// wave (LPU 64), two each; a group of lanes keeps one head, the groups in the
// grid being a multiple of the heads.  In 64 bits up to dO's own rounding: dO is
// perpendicular to O, so that D_2, whose sum dlambda is, is small beside its
// terms.  128 x 4 heads of 64, dh 32, 13 us: 7 for its 35 MB at a copy's rate, the
// rest first loads, drain and the 64-bit reductions.
template <int LPU>
__device__ __forceinline__ double group_sum(double v) {
    v += rnn_dpp_d<0xB1>(v);
    v += rnn_dpp_d<0x4E>(v);
    v += rnn_dpp_d<0x141>(v);
    if (LPU > 8) v += rnn_dpp_d<0x140>(v);
    if (LPU > 16) v += __shfl_xor(v, 16, 64);
    if (LPU > 32) v += __shfl_xor(v, 32, 64);
    return v;
}
template <int LPU>
__global__ __launch_bounds__(256) void diff_bwd_pre_kernel(DiffArgs g) {
    constexpr bool VEC = LPU < 64;
    constexpr int E = VEC ? 4 : 2, GPB = 256 / LPU;  // channels a lane, groups a block
    __shared__ double sh[GPB][128];
    const int c0 = ((int)threadIdx.x % LPU) * E, grp = (int)threadIdx.x / LPU, dv = 2 * g.dh;
    const bool in = c0 < dv;
    const int stride = (int)gridDim.x * GPB;  // a multiple of h
    const int unit0 = (int)blockIdx.x * GPB + grp, hd = unit0 % g.h;
    const float *lp = g.lam + (g.lam_heads > 1 ? (long long)hd * 4 * g.dh : 0);
    double e1 = 0.0, e2 = 0.0;
    for (int c = (int)threadIdx.x % LPU; c < g.dh; c += LPU) {
        e1 += (double)lp[c] * (double)lp[g.dh + c];
        e2 += (double)lp[2 * g.dh + c] * (double)lp[3 * g.dh + c];
    }
    const float lam = expf((float)group_sum<LPU>(e1)) - expf((float)group_sum<LPU>(e2)) + g.lam_init;
    float gain[E];
    double dg[E], dl = 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        gain[e] = g.gain && c0 + e < dv ? g.gain[c0 + e] * (1.0f - g.lam_init) : 0.f;
        dg[e] = 0.0;
    }
    const int units = g.n * g.tq * g.h;
    for (int u = unit0; u < units; u += stride) {
        const int row = u / g.h, b = row / g.tq;
        const bool live = row - b * g.tq < len_of(g.qlen, b, g.tq);
        float o1[E], o2[E], dy[E];
        double o[E], d[E], ss = 0.0;
        const float *p1 = g.o12c + (long long)u * 2 * dv + c0, *py = g.dy + (long long)u * dv + c0;
        if constexpr (VEC) {
            const f4 z = {0.f, 0.f, 0.f, 0.f};
            const f4 a = live && in ? *(const f4 *)p1 : z, c = live && in ? *(const f4 *)(p1 + dv) : z;
            const f4 y = live && in ? *(const f4 *)py : z;
#pragma unroll
            for (int e = 0; e < E; e++) o1[e] = a[e], o2[e] = c[e], dy[e] = y[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool ok = live && c0 + e < dv;
                o1[e] = ok ? p1[e] : 0.f;
                o2[e] = ok ? p1[dv + e] : 0.f;
                dy[e] = ok ? py[e] : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            o[e] = (double)o1[e] - (double)lam * (double)o2[e];
            ss += o[e] * o[e];
            d[e] = (double)dy[e];
        }
        if (g.gain) {
            const double r = 1.0 / sqrt(group_sum<LPU>(ss) / (double)dv + (double)g.eps);
            double t = 0.0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                o[e] *= r;
                t += (double)dy[e] * (double)gain[e] * o[e];
                dg[e] += (double)dy[e] * o[e];
            }
            t = group_sum<LPU>(t) / (double)dv;
#pragma unroll
            for (int e = 0; e < E; e++) d[e] = r * ((double)dy[e] * (double)gain[e] - o[e] * t);
        }
        double d1 = 0.0, d2 = 0.0, nd = 0.0;  // (a float's square underflows below 1e-19)
#pragma unroll
        for (int e = 0; e < E; e++) {
            d1 += d[e] * (double)o1[e];
            d2 += d[e] * (double)o2[e];
            nd += d[e] * d[e];
        }
        d1 = group_sum<LPU>(d1);
        d2 = group_sum<LPU>(d2);
        nd = sqrt(group_sum<LPU>(nd));
        float *pd = g.dout + (long long)u * dv + c0;
        if constexpr (VEC) {
            if (in) *(f4 *)pd = f4{(float)d[0], (float)d[1], (float)d[2], (float)d[3]};
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (c0 + e < dv) pd[e] = (float)d[e];
        }
        if (c0 == 0) {
            const f4 z = {0.f, 0.f, 0.f, 0.f};
            f4 *rec = (f4 *)(g.rec + (long long)u * 8);
            rec[0] = live ? *(const f4 *)(g.statsc + (long long)u * 4) : z;
            rec[1] = f4{(float)d1, (float)d2, (float)nd, lam};
        }
        dl += d2;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        if (c0 + e < dv) sh[grp][c0 + e] = dg[e] * (double)(1.0f - g.lam_init);
    double *part = g.part + (long long)blockIdx.x * (dv + GPB);
    if (c0 == 0) part[dv + grp] = -dl;
    __syncthreads();
    for (int c = threadIdx.x; c < dv; c += 256) {
        double t = 0.0;
        for (int i = 0; i < GPB; i++) t += sh[i][c];
        part[c] = t;
    }
}

// dgain and dlam from the first pass's partials, in the first blocks of dQ's launch
// (on their own they took 5 to 6 us), NT threads each.  Block i < ceil(dv / 16): the
// gain's columns [16 i, 16 i + 16), NT / 16 groups of partials each in order, then
// the groups in order.  The others: one set of lambda vectors each, the partials of
// its heads (every group of every block for a shared set, else group index % h =
// head) in NT strided sums, added in a fixed tree.
__device__ __forceinline__ int params_blocks(const DiffArgs &g) {
    return g.first ? 0 : (g.dgain ? (2 * g.dh + 15) / 16 : 0) + g.lam_heads;
}
template <int NT>
__device__ __forceinline__ void bwd_params(const DiffArgs &g, int blk, double *red) {
    const int dv = 2 * g.dh, cols = dv + g.gpb, ngain = g.dgain ? (dv + 15) / 16 : 0;
    const int lane = threadIdx.x & 63, wv = wave_index();
    if (blk < ngain) {
        constexpr int Q = NT / 16;
        const int jl = threadIdx.x % 16, q = threadIdx.x / 16, j = 16 * blk + jl;
        const int per = (g.nblk + Q - 1) / Q, k0 = min(g.nblk, q * per), k1 = min(g.nblk, k0 + per);
        const double *src = g.part + min(j, dv - 1);
        double s = 0.0;
        for (int k = k0; k < k1; k += 16) {
            double v[16];
#pragma unroll
            for (int u = 0; u < 16; u++) v[u] = src[(long long)min(k + u, k1 - 1) * cols];
#pragma unroll
            for (int u = 0; u < 16; u++)
                if (k + u < k1) s += v[u];
        }
        red[q * 16 + jl] = s;
        __syncthreads();
        if (q == 0 && j < dv) {
            double t = 0.0;
            for (int u = 0; u < Q; u++) t += red[u * 16 + jl];
            g.dgain[j] += (float)t;
        }
        return;
    }
    const int set = blk - ngain, step = g.lam_heads > 1 ? g.h : 1;
    const int groups = g.nblk * g.gpb;
    double s = 0.0;
    for (int k0 = set + step * (int)threadIdx.x; k0 < groups; k0 += step * NT * 8) {
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int k = min(k0 + u * step * NT, groups - 1);
            v[u] = g.part[(long long)(k / g.gpb) * cols + dv + k % g.gpb];
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (k0 + u * step * NT < groups) s += v[u];
    }
    s = rnn_wave_sum_d(s);
    if (lane == 0) red[wv] = s;
    __syncthreads();
    if (wv) return;
    double t = 0.0;
    for (int i = 0; i < NT / 64; i++) t += red[i];
    double e1, e2;
    lambda_dots(g.lam, g.lam_heads, g.dh, set, &e1, &e2);
    e1 = exp(e1);
    e2 = exp(e2);
    const int dh = g.dh;
    const float *l = g.lam + (long long)set * 4 * dh;
    float *d = g.dlam + (long long)set * 4 * dh;
    if (lane < dh) {
        d[lane] += (float)(t * e1 * l[dh + lane]);
        d[dh + lane] += (float)(t * e1 * l[lane]);
        d[2 * dh + lane] -= (float)(t * e2 * l[3 * dh + lane]);
        d[3 * dh + lane] -= (float)(t * e2 * l[2 * dh + lane]);
    }
}

// The power of two of dA - D for rows with |dO| <= nd and values of magnitude <=
// vmax, from m = ds_bound >= |dA| + |D| (|dA| <= nd sqrt(W) vmax; D, a mean of dA over
// all of the row's keys, may be far above it where vmax is of some of them alone): it
// takes m to [1, 2), and stays as it was (up) until m times it passes 2.  It keeps dS
// within a float's range and no more: ds_fit has the bits of its two parts.
template <int W>
__device__ __forceinline__ constexpr float ds_root() {
    return W == 32 ? 11.313709f : W == 64 ? 16.0f : W == 96 ? 19.595918f : 22.627417f;
}
// dmax: the larger |D_m|.  (At most 2^126, whose power is the smallest with a
// reciprocal: ds_fit makes up for what is past it.)
template <int W>
__device__ __forceinline__ float ds_bound(float nd, float vmax, float dmax) {
    return fminf(max2(nd * (ds_root<W>() * vmax), 2.0f * dmax), 0x1p126f);
}
__device__ __forceinline__ float ds_up(float m, float up) {
    return m * up < 2.0f ? up : up_of(m) * 0x1p-14f;
}
// From a product of V's and dO's operands to dA times its power of two.  dO of zeros
// alone leaves the powers where they started, whose product may be infinite: cut off,
// so that it stays 0 times a number.
__device__ __forceinline__ float da_unit(float vdown, float ddown, float up) {
    return fminf(vdown * (ddown * up), 0x1.fffffep127f);
}
// A softmax value before its row's reciprocal sum, from a score less the largest: at
// most 1, also where a score's error passes an exponent (v_exp_f32 cuts it off itself).
__device__ __forceinline__ float exp_below(float x) {
    return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(x), 0.0f, 1.0f);
}
// The power of two that softmax values, and lambda times them, enter the backward's
// products with, from the largest of them in the rows: they come to at most 2^14, so
// that P_1 - lambda P_2 stays below 2^15.
__device__ __forceinline__ float p_up(float pmax) { return up_of(pmax) * 0.5f; }

// The power of two of a lane's dS, its row's in dQ or its key's in dK, on top of what
// bounds say: it follows the largest magnitude so far as sticky_up does, and the
// lane's accumulators with it.  Bounds alone left dS an error in proportion to the
// keys (P falls with them, and |dA| is a hundredth of its bound), 9e-6 of dQ and dK
// at 65536 keys, and with any outlier of V; now dK is 3e-7 off there, and dQ 2e-6, by
// the length of its sums.  It costs eight instructions a map and tile, sixteen more
// in dK, and a branch that is rarely taken: 2 x 8 causal heads of 1568, dh 64, dQ 107
// us and dK, dV 179 against 105 and 171 without; 4 x 8 of 2048 490 and 559 against
// 453 and 558.
constexpr float DS_START = 0x1p108f;  // (dS is at most 2^15 before it)
// The largest magnitude, which ds_fit is called for from 2^15 on.
__device__ __forceinline__ float absmax16(const f32x16 &s) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) m = max3abs(m, s[r], s[r + 1]);
    return m;
}
// Takes m, the lane's largest |dS|, to [2^10, 2^11) where it is past 2^15; the factor.
__device__ __forceinline__ float ds_fit(f32x16 &s, float &m, float &up) {
    m = pair32(m, max2);
    const float f = m >= 0x1p15f ? up_of(m) * 0x1p-4f : 1.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] *= f;
    up *= f;
    m *= f;
    return f;
}
template <int C>
__device__ __forceinline__ void scale_all(f32x16 (&acc)[C], float f) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[c][r] *= f;
}

// The matrix core's sum is cut off towards -inf, which leaves every element of
// a long sum a little low.  Two thirds of the way (where a sum that grows with
// the square root of its length has collected half of it) the accumulators
// change sign, and the operand from registers with them.
__device__ __forceinline__ int flip_at(int ntile) { return (2 * ntile + 2) / 3; }

// dQ.  Rows as in the forward, RG groups of 32 a workgroup, a wave on NM maps of its
// rows (both, or a pair of waves one each, dA in both) and on one of the KG 32 keys
// of a tile; tiles in two LDS buffers: S_m^T = K_m Q_m^T and dA^T = V dO^T (lane =
// row), and P (dA - D) in registers is the operand of dQ_m^T = K_m^T dS_m^T, which
// is summed over all tiles in the accumulators.  Their units are powers of two that
// hardly change (sticky_up, ds_up, ds_fit); where one does they are rescaled.  The
// waves that share rows add theirs at the end.  Bound as the forward: 4 x 8 heads of
// 2048, dh 64, 498 us (207 TFLOP/s of fp32 work; the parts' powers by row cost a tenth
// here); 2 x 8 causal heads of 1568 107 us (141, the longest rows' chain); 8 x 6
// ragged of up to 577, dh 32, 42 us.
template <int DHP, bool VEC, int RG, int KG, int NM>
__global__ __launch_bounds__(128 / NM * RG * KG)
__attribute__((amdgpu_waves_per_eu((DHP <= 32 && RG > 1) || NM == 1 ? 2 : 1))) void
diff_dq_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TK = 32 * KG, NW = 2 / NM * RG * KG, NT = 64 * NW, KS = DHP / 16, VS = W / 16;
    constexpr int CT = (DHP + 31) / 32, BR = 32 * RG;
    using Tile = HalfTile<TK, W>;
    // (a map's last 32-channel tile may run past the row: into the padding)
    __shared__ __align__(16) _Float16 lds[2][2 * Tile::HALVES + 32];
    static_assert(KG == 1 || sizeof(lds) >= (size_t)(KG - 1) * RG * 2 * CT * 16 * 64 * 4, "exchange");
    __shared__ f2 tmax[2][NW];
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int map = NM == 2 ? 0 : wave & 1;  // the first of the wave's
    const int rg = wave / (2 / NM) % RG, kg = wave / (2 / NM) / RG;
    const int R = g.tq * g.group, nrb = (R + BR - 1) / BR;
    const int np = params_blocks(g);
    if ((int)blockIdx.x < np) {
        bwd_params<NT>(g, (int)blockIdx.x, (double *)lds);
        return;
    }
    const long long id = g.first + xcd_order(blockIdx.x - np, gridDim.x - np);
    const int prob = (int)(id / nrb), rb = nrb - 1 - (int)(id % nrb);
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int row = rb * BR + rg * 32 + lr;
    const int qi = row / g.group, head = kh * g.group + row % g.group;
    const bool live = qi < nq;
    const int last_q = min(nq - 1, (rb * BR + BR - 1) / g.group);
    int kend = g.causal ? min(nk, last_q + shift + 1) : nk;
    if (rb * BR / g.group >= nq) kend = 0;
    const int ntile = kend > 0 ? (kend + TK - 1) / TK : 0;
    KvStage<DHP, TK, NT, VEC> st(g, b, kh, kend);
    if (ntile) st.load(0);

    // the row's queries, its dO and what the first pass left of it
    const int w_first = (rb * BR + rg * 32) / g.group;
    const int w_last = min(nq - 1, (rb * BR + rg * 32 + 31) / g.group);
    const int q0 = min(w_first, g.tq - 1), qx = qi - q0, dv = 2 * g.dh;
    const long long img = (long long)b * g.tq + q0;
    const int left = min(g.tq - q0, 32);
    const auto rq = rows_rsrc(g.q + img * g.qstride, left, g.qstride, 2 * g.h * g.dh);
    const auto rd = rows_rsrc(g.dout + img * g.h * dv, left, (long long)g.h * dv, g.h * dv);
    const auto rr = rows_rsrc(g.rec + img * g.h * 8, left, (long long)g.h * 8, g.h * 8);
    f32x4 sm, dd;
    {
        const uint32_t at = live ? (uint32_t)(qx * g.h + head) * 32u : DMA_OOB;
        sm = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, at, 0, 0));
        dd = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, at + 16u, 0, 0));
    }
    Half2 q[NM][KS], d[VS];
    float qdown[NM], ddown;
    {
        RowFrag<KS> qf[NM];
        RowFrag<VS> df;
#pragma unroll
        for (int m = 0; m < NM; m++)
            qf[m].template load<VEC>(rq, (uint32_t)qx * (uint32_t)g.qstride + (2 * head + map + m) * g.dh,
                                     live ? g.dh : 0);
        df.template load<VEC>(rd, (uint32_t)(qx * g.h + head) * dv, live ? dv : 0);
#pragma unroll
        for (int m = 0; m < NM; m++) qdown[m] = qf[m].split(q[m]) * (g.scale * LOG2E);
        ddown = df.split(d);
    }
    const float pup = p_up(max2(sm[1], fabsf(sm[3] * dd[3])));
    const float dmax = max2(fabsf(dd[0]), fabsf(dd[1]));
    float nm[NM], il[NM], D[NM], own[NM];  // own: dS's power of two, on top of P's
#pragma unroll
    for (int m = 0; m < NM; m++) {
        const bool second = map + m;
        nm[m] = second ? -sm[2] : -sm[0];
        own[m] = DS_START;
        il[m] = (second ? sm[3] * dd[3] : sm[1]) * pup * DS_START;
        D[m] = second ? -dd[1] : -dd[0];
    }
    f32x16 acc[NM][CT];
#pragma unroll
    for (int m = 0; m < NM; m++)
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[m][c][r] = 0.f;
    // the largest value so far, and powers of two: of the tile that is staged (.1)
    // and of the one that is computed
    float vmax = 0.f, kup1 = FIRST_UP, vup1 = 1.f, kup = FIRST_UP, dsup = FIRST_UP, sgn = 1.f;
    const int flip = flip_at(ntile);
    auto maxima = [&](int slot) { st.maxima(tmax[slot], good_for(kup1), vmax); };
    auto stage = [&](int t) {  // tile t, whose maxima are there, into its buffer
        float mk = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const f2 m = tmax[t & 1][i];
            mk = max2(mk, m[0]);
            vmax = max2(vmax, m[1]);
        }
        kup1 = sticky_up(mk, kup1);
        vup1 = up_of(vmax);
        st.store(lds[t & 1], kup1, vup1);
    };
    if (ntile) {
        maxima(0);
        __syncthreads();
        stage(0);
        if (ntile > 1) {
            st.load(TK);
            maxima(1);
        }
    }
    for (int t = 0; t < ntile; t++) {
        const int k0 = t * TK;
        __syncthreads();
        // dS's power of two, and the accumulators in the tile's unit
        const float vup = vup1, dsup1 = ds_up(ds_bound<W>(dd[2], vmax, dmax), dsup);
        float ratio = down_of(kup) * kup1 * (down_of(dsup) * dsup1);
        kup = kup1;
        dsup = dsup1;
        if (t == flip) {
            sgn = -1.0f;
#pragma unroll
            for (int m = 0; m < NM; m++) il[m] = -il[m];
            ratio = -ratio;
        }
        if (NM == 1 && __any(ratio != 1.0f)) {  // (with one map, registers are short below)
            scale_all(acc[0], ratio);
            ratio = 1.0f;
        }
        if (t + 1 < ntile) stage(t + 1);
        if (t + 2 < ntile) st.load(k0 + 2 * TK);
        {
            const _Float16 *const kt = lds[t & 1] + 32 * kg * Tile::STRIDE, *const vt = kt + Tile::HALVES;
            const int k1 = k0 + 32 * kg;
            const float kdown = down_of(kup);
            f32x16 s[NM], da;
#pragma unroll
            for (int r = 0; r < 16; r++) da[r] = 0.f;
#pragma unroll
            for (int m = 0; m < NM; m++) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[m][r] = 0.f;
                dot_along<Tile>(kt, (map + m) * DHP, q[m], s[m]);
            }
            dot_along<Tile>(vt, 0, d, da);
            read_ahead<NM * KS + VS, 2, 3>();
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const float f = kdown * qdown[m];
#pragma unroll
                for (int r = 0; r < 16; r++)
                    s[m][r] = exp_below(__builtin_fmaf(s[m][r], f, nm[m])) * il[m];
            }
            const bool whole = k1 + 32 <= nk && !(g.causal && k1 + 31 > w_first + shift) &&
                               !(g.diag && k1 <= w_last && w_first < k1 + 32);
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int j = k1 + 8 * (r >> 2) + 4 * lh + (r & 3);
                    const bool in = j < nk && !(g.causal && j > qi + shift) && !(g.diag && j == qi);
#pragma unroll
                    for (int m = 0; m < NM; m++) s[m][r] = in ? s[m][r] : 0.f;
                }
            }
            const float fd = da_unit(down_of(vup), ddown, dsup);
            float mx[NM];
            bool past = NM > 1 && ratio != 1.0f;
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const float dm = D[m] * dsup;
#pragma unroll
                for (int r = 0; r < 16; r++) s[m][r] *= __builtin_fmaf(da[r], fd, dm);
                mx[m] = absmax16(s[m]);
                past = past || mx[m] >= 0x1p15f;
            }
            if (__builtin_expect(__any(past), 0)) {
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    const float f = ds_fit(s[m], mx[m], own[m]);
                    il[m] *= f;
                    scale_all(acc[m], NM > 1 ? f * ratio : f);
                }
            }
#pragma unroll
            for (int m = 0; m < NM; m++) {
                Half2 ds[2];
                split16(s[m], ds);
#pragma unroll
                for (int c = 0; c < CT; c++)
                    dot_across<Tile>(kt, (map + m) * DHP + 32 * c, ds, acc[m][c]);
            }
            read_ahead<2 * NM * CT, 4, 3>();
        }
        if (t + 2 < ntile) maxima(t & 1);
    }
    // (dS's own powers of two come off first: waves that share rows have different ones)
#pragma unroll
    for (int m = 0; m < NM; m++) scale_all(acc[m], down_of(own[m]));
    if constexpr (KG > 1) {
        __syncthreads();
        float *const ex = (float *)lds + (rg * 2 + map) * CT * 16 * 64 + lane;
        auto each = [&](int i, auto &&f) {
            float *e = ex + (i - 1) * RG * 2 * CT * 16 * 64;
#pragma unroll
            for (int m = 0; m < NM; m++)
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int r = 0; r < 16; r++) f(e[((m * CT + c) * 16 + r) * 64], acc[m][c], r);
        };
        if (kg) each(kg, [](float &e, f32x16 &v, int r) { e = v[r]; });
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int i = 1; i < KG; i++) each(i, [](float &e, f32x16 &v, int r) { v[r] += e; });
    }
    if (row >= R) return;
    float *dst = g.dq + ((long long)b * g.tq + qi) * g.qstride + 2 * head * g.dh;
    const float f = down_of(kup) * (g.scale * sgn), f2 = down_of(dsup) * down_of(pup);
#pragma unroll
    for (int m = 0; m < NM; m++)
#pragma unroll
        for (int c = 0; c < CT; c++)
            put_channels<VEC>(dst + (map + m) * g.dh, g.dh, 32 * c, acc[m][c], map + m ? -f : f, f2, live,
                              g.acc_q);
}

// dK and dV.  One workgroup of 2 KG waves per (image, key head, 32 KG keys); a pair
// of waves takes 32 keys, wave 2 i + m map m of them: its half of a row's channels
// of Q K^T (a map) and of dO V^T stays in registers.  Tiles of 32 rows (queries of
// the head group) and their records in two LDS buffers: S_m = Q_m K_m^T and the
// wave's half of dA = dO V^T (lane = key); P_m and that half go to the partner
// through LDS, and then P and dS in registers are the operands of the wave's half
// of dV^T = dO^T (P_1 - lambda P_2) and of dK_m^T = Q_m^T dS_m, summed over all tiles
// in the accumulators as in diff_dq_kernel.
// A tile's chain bounds it here too: 4 x 8 heads of 2048, dh 64, 567 us (243 TFLOP/s
// of fp32 work); 2 x 8 causal heads of 1568 180 us (111); 8 x 6 ragged of up to 577,
// dh 32, 60 us.
template <int DHP, bool VEC, int KG>
__global__ __launch_bounds__(128 * KG) __attribute__((amdgpu_waves_per_eu(DHP <= 32 && KG > 1 ? 2 : 1))) void
diff_dkv_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, TR = 32, NW = 2 * KG, NT = 64 * NW, KS = DHP / 16;
    constexpr int CT = (DHP + 31) / 32, VT = (DHP / 16 + 1) / 2, BK = 32 * KG;
    using Tile = HalfTile<TR, W>;
    using Stage = StagePlan<TR, W, NT>;
    constexpr int CH = Stage::PASSES;
    __shared__ __align__(16) _Float16 lds[2][2 * Tile::HALVES + 32];
    // -m1, il1, -m2, -lambda il2, -D1, -D2, with their powers of two
    __shared__ __align__(16) float rec[2][6][TR];
    // largest |q|, |dO|, |dO|_2 and P (or lambda times it) of a tile past what is known
    // of them; with |dO|_2's, the largest |D_m|
    __shared__ f4 tmax[2][NW];
    __shared__ float tdmax[2];
    __shared__ float vmaxs[NW];
    __shared__ float vkey[NW][32];
    __shared__ __align__(16) f32x4 ex[NW][8][64];  // P_m and a half of dA, each wave's
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int kg = wave >> 1, map = wave & 1;
    const int nkb = (g.tk + BK - 1) / BK;
    const long long id = g.first + xcd_order(blockIdx.x, gridDim.x);
    const int prob = (int)(id / nkb), kb = (int)(id % nkb);
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int w_first = kb * BK + kg * 32, key = w_first + lr;
    const bool live = key < nk;
    // rows that see some key of the block
    const int first_q = g.causal ? max(0, kb * BK - shift) : 0;
    const int row_end = kb * BK < nk ? nq * g.group : 0;
    const int row_beg = min(first_q, nq) * g.group;
    const int ntile = row_end > row_beg ? (row_end - row_beg + TR - 1) / TR : 0;
    const float ginv = 1.0f / (float)g.group;

    float xq[CH][8], xd[CH][8];
    f32x4 r0 = {0.f, 0.f, 0.f, 0.f}, r1 = r0;
    const int sc = (int)threadIdx.x % Stage::C8 * 8, sr = (int)threadIdx.x / Stage::C8;
    const bool stager = Stage::ALL || sr < Stage::RPP;
    const int run = sc >= DHP ? 1 : 0, dw = 2 * g.dh;
    const int qlim = stager ? g.dh - (sc - run * DHP) : 0, dlim = stager ? dw - sc : 0;
    const long long img = (long long)b * g.tq;
    const int qc = run * g.dh + sc - run * DHP;
    // row x of a tile is query q0 + (x0 + x) / group, head (x0 + x) % group of the
    // group (x0 + x < TR + group, exact in floats).  lq0, lx0: of the tile that is
    // loaded next, whose offsets are those of every tile where the group divides TR.
    int lq0 = row_beg / g.group, lx0 = 0, cq0 = lq0, cx0 = 0;
    const bool steady = TR % g.group == 0;
    auto next = [&](int &q0, int &x0) {
        q0 += TR / g.group;
        x0 += TR % g.group;
        if (x0 >= g.group) {
            x0 -= g.group;
            q0++;
        }
    };
    uint32_t qo[CH], od[CH], ro;
    auto offsets = [&] {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int x = lx0 + sr + i * Stage::RPP;
            const int dq = (int)(((float)x + 0.5f) * ginv), hd = x - dq * g.group;
            qo[i] = (uint32_t)dq * (uint32_t)g.qstride + 2 * hd * g.dh + qc;
            od[i] = (uint32_t)(dq * g.h + hd) * dw + sc;
        }
        const int x = lx0 + lr, dq = (int)(((float)x + 0.5f) * ginv);
        ro = (uint32_t)(dq * g.h + x - dq * g.group) * 32u;
    };
    offsets();
    auto load = [&] {
        if (!steady) offsets();
        // queries from nq on are past the resources' end
        const int rows = min(nq - lq0, TR + 1);
        const auto rq = rows_rsrc(g.q + (img + lq0) * g.qstride + 2 * kh * g.group * g.dh, rows,
                                  g.qstride, 2 * g.group * g.dh);
        const auto rd = rows_rsrc(g.dout + ((img + lq0) * g.h + kh * g.group) * dw, rows,
                                  (long long)g.h * dw, g.group * dw);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            load8<VEC>(rq, qo[i], qlim, xq[i]);
            load8<VEC>(rd, od[i], dlim, xd[i]);
        }
        if (wave == 0) {
            const auto rr = rows_rsrc(g.rec + ((img + lq0) * g.h + kh * g.group) * 8, rows,
                                      (long long)g.h * 8, g.group * 8);
            r0 = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, ro, 0, 0));
            r1 = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, ro + 16u, 0, 0));
        }
        next(lq0, lx0);
    };
    // the largest value and P so far, the powers of two of the tile that is staged (.1)
    // and of the one that is computed; the lane's own of dS
    float sown = DS_START;
    float vmax = INFINITY, ml = 0.f, qup1 = FIRST_UP, dup1 = FIRST_UP, pup1 = 1.f, sup1 = FIRST_UP;
    float qup = FIRST_UP, dup = FIRST_UP, pup = 1.f, sup = FIRST_UP;
    auto maxima = [&](int slot) {
        float mq = 0.f, md = 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            mq = absmax8(xq[i], mq);
            md = absmax8(xd[i], md);
        }
        f4 m = {0.f, 0.f, 0.f, 0.f};
        if (__any(mq > good_for(qup1) || md > good_for(dup1))) {
            m[0] = wave_max(mq);
            m[1] = wave_max(md);
        }
        if (wave == 0) {
            const float dm = max2(fabsf(r1[0]), fabsf(r1[1]));
            float dall = 0.f;
            if (__any(!(ds_bound<W>(r1[2], vmax, dm) * sup1 < 2.0f))) {
                m[2] = wave_max(r1[2]);
                dall = wave_max(dm);
            }
            m[3] = wave_over(max2(r0[1], fabsf(r0[3] * r1[3])), ml);
            if (lane == 0) tdmax[slot] = dall;
        }
        if (lane == 0) tmax[slot][wave] = m;
    };
    if (ntile) load();

    // the lane's key and value: the map's half of their channels
    Half2 k[KS], v[KS];
    float kdown, vdown;
    const long long krow = (long long)b * g.tk + min(key, g.tk - 1);
    {
        const int k0 = min(w_first, g.tk - 1), rows = min(g.tk - k0, 32);
        const float *kvp = g.kv + ((long long)b * g.tk + k0) * g.kvstride + 2 * kh * g.dh;
        const auto rk = rows_rsrc(kvp + g.koff, rows, g.kvstride, dw);
        const auto rv = rows_rsrc(kvp + g.voff, rows, g.kvstride, dw);
        const uint32_t off = (uint32_t)(key - k0) * (uint32_t)g.kvstride;
        RowFrag<KS> kf, vf;
        kf.template load<VEC>(rk, off + map * g.dh, live ? g.dh : 0);
        vf.template load<VEC>(rv, off + map * DHP, live ? dw - map * DHP : 0);
        kdown = kf.split(k) * (g.scale * LOG2E);
        // (a key's two halves share their power of two)
        float mv = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) mv = absmax8(vf.v[s], mv);
        mv = pair32(mv, max2);
        if (lh == 0) vkey[wave][lr] = mv;
        const float mx = wave_max(mv);
        if (lane == 0) vmaxs[wave] = mx;
        if (ntile) maxima(0);
        __syncthreads();
        const float up = up_of(max2(mv, vkey[wave ^ 1][lr]));
#pragma unroll
        for (int s = 0; s < KS; s++) v[s] = half_split(vf.v[s], up);
        vdown = down_of(up);
    }
    f32x16 dk[CT], dv[VT];
#pragma unroll
    for (int r = 0; r < 16; r++) {
#pragma unroll
        for (int c = 0; c < CT; c++) dk[c][r] = 0.f;
#pragma unroll
        for (int c = 0; c < VT; c++) dv[c][r] = 0.f;
    }
    const int flip = flip_at(ntile);
    auto stage = [&](int t) {
        float mq = 0.f, md = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const f4 m = tmax[t & 1][i];
            mq = max2(mq, m[0]);
            md = max2(md, m[1]);
            if (i) continue;
            ml = max2(ml, m[3]);
            sup1 = ds_up(ds_bound<W>(m[2], vmax, tdmax[t & 1]), sup1);
        }
        qup1 = sticky_up(mq, qup1);
        dup1 = sticky_up(md, dup1);
        pup1 = p_up(ml);
        if (stager) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                _Float16 *p = lds[t & 1] + row_pos(sr + i * Stage::RPP) * Tile::STRIDE + sc;
                const Half2 hq = half_split(xq[i], qup1), hd = half_split(xd[i], dup1);
                *(h8 *)p = hq.hi;
                *(h8 *)(p + Tile::PART) = hq.lo;
                *(h8 *)(p + Tile::HALVES) = hd.hi;
                *(h8 *)(p + Tile::HALVES + Tile::PART) = hd.lo;
            }
        }
        if (threadIdx.x < TR) {
            float(*rc)[TR] = rec[t & 1];
            const float u = t >= flip ? -pup1 : pup1;
            rc[0][threadIdx.x] = -r0[0];
            rc[1][threadIdx.x] = r0[1] * u;
            rc[2][threadIdx.x] = -r0[2];
            rc[3][threadIdx.x] = -r0[3] * r1[3] * u;
            rc[4][threadIdx.x] = -r1[0] * sup1;
            rc[5][threadIdx.x] = -r1[1] * sup1;
        }
    };
    if (ntile) {
        vmax = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) vmax = max2(vmax, vmaxs[i]);
        stage(0);
        if (ntile > 1) {
            load();
            maxima(1);
        }
    }
    for (int t = 0; t < ntile; t++) {
        __syncthreads();
        float rv = down_of(pup) * pup1 * (down_of(dup) * dup1);
        float rk = down_of(pup) * pup1 * (down_of(qup) * qup1) * (down_of(sup) * sup1);
        qup = qup1;
        dup = dup1;
        pup = pup1;
        sup = sup1;
        if (t == flip) {
            rv = -rv;
            rk = -rk;
        }
        if (t + 1 < ntile) stage(t + 1);
        if (t + 2 < ntile) load();
        const int tq0 = cq0, x0 = cx0;
        next(cq0, cx0);
        const _Float16 *const qt = lds[t & 1], *const dt = qt + Tile::HALVES;
        const float(*rc)[TR] = &rec[t & 1][2 * map];
        f32x16 s, da;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = da[r] = 0.f;
        dot_along<Tile>(qt, map * DHP, k, s);
        dot_along<Tile>(dt, map * DHP, v, da);
        read_ahead<2 * KS, 2, 3>();
        const float f = down_of(qup) * kdown;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 m4 = *(const f32x4 *)&rc[0][2 * r + 4 * lh], l4 = *(const f32x4 *)&rc[1][2 * r + 4 * lh];
#pragma unroll
            for (int e = 0; e < 4; e++)
                s[r + e] = exp_below(__builtin_fmaf(s[r + e], f, m4[e])) * l4[e];
        }
        // rows past the last carry il = 0, keys past the last are not stored
        const bool whole = !(g.causal && w_first + 31 > tq0 + shift) &&
                           !(g.diag && w_first <= tq0 + (x0 + TR - 1) / g.group && tq0 <= w_first + 31);
        if (!whole) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int x = x0 + 8 * (r >> 2) + 4 * lh + (r & 3);
                const int i = tq0 + (int)(((float)x + 0.5f) * ginv);
                const bool in = !(g.causal && key > i + shift) && !(g.diag && key == i);
                s[r] = in ? s[r] : 0.f;
            }
        }
        const float fd = da_unit(vdown, down_of(dup), sup);
        f32x4 *const mine = &ex[wave][0][lane], *const other = &ex[wave ^ 1][0][lane];
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f32x4 p, d;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[e] = s[r + e];
                d[e] = da[r + e];
            }
            mine[16 * r] = p;
            mine[16 * r + 256] = d;
        }
        __syncthreads();
        // P_1 - lambda P_2 (P_2's sign is in its rec) and dA, the same in both waves
        f32x16 a;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 p = other[16 * r], d = other[16 * r + 256];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                a[r + e] = s[r + e] + p[e];
                da[r + e] += d[e];
            }
        }
        rc = &rec[t & 1][4 + map];
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 D = *(const f32x4 *)&rc[0][2 * r + 4 * lh];
#pragma unroll
            for (int e = 0; e < 4; e++) s[r + e] *= __builtin_fmaf(da[r + e], fd, D[e]) * sown;
        }
        float mx = absmax16(s);
        if (__builtin_expect(__any(mx >= 0x1p15f || rk != 1.0f || rv != 1.0f), 0)) {
            scale_all(dk, ds_fit(s, mx, sown) * rk);
            scale_all(dv, rv);
        }
        {
            Half2 ah[2], ds[2];
            split16(a, ah);
#pragma unroll
            for (int c = 0; c < VT; c++)
                if (VT * 32 * 2 == W || map * VT + c < W / 32)
                    dot_across<Tile>(dt, 32 * (map * VT + c), ah, dv[c]);
            split16(s, ds);
#pragma unroll
            for (int c = 0; c < CT; c++) dot_across<Tile>(qt, map * DHP + 32 * c, ds, dk[c]);
        }
        read_ahead<2 * (VT + CT), 4, 3>();
        if (t + 2 < ntile) maxima(t & 1);
    }
    if (key >= g.tk) return;
    float *kd = g.dkv + krow * g.kvstride + g.koff + (2 * kh + map) * g.dh;
    float *vd = g.dkv + krow * g.kvstride + g.voff + 2 * kh * g.dh;
    const float sgn = ntile > flip ? -1.0f : 1.0f;
    const float fk = down_of(qup) * (g.scale * sgn), fk2 = down_of(pup) * down_of(sup);
    scale_all(dk, down_of(sown));
#pragma unroll
    for (int c = 0; c < CT; c++)
        put_channels<VEC>(kd, g.dh, 32 * c, dk[c], fk, fk2, live, g.acc_kv);
#pragma unroll
    for (int c = 0; c < VT; c++)
        if (VT * 32 * 2 == W || map * VT + c < W / 32)
            put_channels<VEC>(vd, 2 * g.dh, 32 * (map * VT + c), dv[c], down_of(dup) * sgn,
                              down_of(pup), live, g.acc_kv);
}

// acc += over 64 rows: columns ca .. ca + 31 of one tile (accumulator rows) times
// columns cb .. cb + 31 of another (lanes).
template <class TA, class TB>
__device__ __forceinline__ void dot_tiles(const _Float16 *ta, int ca, const _Float16 *tb, int cb,
                                          f32x16 &acc) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const h8 ah = TA::across(ta, 16 * s, ca), al = TA::across(ta + TA::PART, 16 * s, ca);
        const h8 bh = TB::across(tb, 16 * s, cb), bl = TB::across(tb + TB::PART, 16 * s, cb);
        acc = mm(al, bh, acc);
        acc = mm(ah, bl, acc);
        acc = mm(ah, bh, acc);
    }
}

// dQ, dK and dV of problems of at most 64 rows, a workgroup of four waves each,
// over tiles of 64 keys: Q and dO are read and split once, K and V once for all
// three.  Wave (rg, kg) has the scores of 32 rows with 32 keys, both maps, and sums
// dQ as diff_dq_kernel does; P_1 - lambda P_2 and dS_m go through LDS where the tile
// has been read for the last time, row by row, and come back transposed as
// operands of dV and dK, whose blocks of 32 keys and 32 channels the waves share
// out.  dO and dS have powers of two by row where a sum runs along one (dA, dQ), and
// common ones where it runs over the rows (dV through P's, dK with dS split again).
// ONE: one tile holds the keys.  A tile's chain of loads, splits, products and six
// barriers bounds it, with two workgroups a CU up to 32 channels: 128 x 4 heads of 64
// rows and keys, dh 32, 22 us (60 MB; 12 at a copy's rate) where dQ and dK/dV apart
// take 19.0 + 18.7; 64 rows on 256 keys 47 us (160 MB; 32) instead of 29.3 + 52.9.
template <int DHP, bool ONE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DHP <= 32 ? 2 : 1))) void
diff_bwd_rows_kernel(DiffArgs g) {
    constexpr int W = 2 * DHP, KS = DHP / 16, VS = W / 16, CT = (DHP + 31) / 32;
    using Tile = HalfTile<64, W>;
    using PTile = HalfTile<64, 64>;
    using Stage = StagePlan<64, W, 256>;
    constexpr int CH = Stage::PASSES;
    // (a map's last 32-channel tile may run past the row: into the padding)
    constexpr int EX = 2 * 2 * CT * 16 * 64 * 2;  // dQ's halves, in halves
    constexpr int SLOT = std::max({Tile::HALVES + 32, PTile::HALVES, EX});
    __shared__ __align__(16) _Float16 lds[4][SLOT];  // K, V, Q, dO
    __shared__ float rec[6][64];  // as in diff_dkv_kernel
    __shared__ f4 rmax[4];
    __shared__ float rdo[64];  // |dO|_2 of the rows
    __shared__ f2 tmax[4];
    __shared__ f4 psum[2][ONE ? 64 : 1];  // sums of P_m and of P_m dA over 32 keys
    __shared__ f2 smax[4];                // largest |dS_m| of a wave's part of the tile
    const int np = params_blocks(g);
    if ((int)blockIdx.x < np) {
        bwd_params<256>(g, (int)blockIdx.x, (double *)lds);
        return;
    }
    const int lane = threadIdx.x & 63, wave = wave_index(), lr = lane & 31, lh = lane >> 5;
    const int prob = (int)(g.first + xcd_order(blockIdx.x - np, gridDim.x - np));
    const int b = prob / g.hkv, kh = prob % g.hkv;
    const int nq = len_of(g.qlen, b, g.tq), nk = len_of(g.klen, b, g.tk), shift = nk - nq;
    const int dw = 2 * g.dh;
    _Float16 *const kt = lds[0], *const vt = lds[1], *const qt = lds[2], *const dt = lds[3];

    KvStage<DHP, 64, 256, true> st(g, b, kh, nk);
    st.load(0);
    const int sc = (int)threadIdx.x % Stage::C8 * 8, sr = (int)threadIdx.x / Stage::C8;
    const bool stager = st.stager();
    float xq[CH][8], xd[CH][8];
    f32x4 r0, r1;
    {
        const int run = sc >= DHP ? 1 : 0;
        const long long img = (long long)b * g.tq;
        const auto rq = rows_rsrc(g.q + img * g.qstride + 2 * kh * g.group * g.dh, nq, g.qstride,
                                  2 * g.group * g.dh);
        const auto rd = rows_rsrc(g.dout + (img * g.h + kh * g.group) * dw, nq,
                                  (long long)g.h * dw, g.group * dw);
        const auto rr = rows_rsrc(g.rec + (img * g.h + kh * g.group) * 8, nq, (long long)g.h * 8,
                                  g.group * 8);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int x = sr + i * Stage::RPP, i0 = x / g.group, hd = x - i0 * g.group;
            load8<true>(rq, (uint32_t)i0 * (uint32_t)g.qstride + 2 * hd * g.dh + run * g.dh + sc - run * DHP,
                        stager ? g.dh - (sc - run * DHP) : 0, xq[i]);
            load8<true>(rd, (uint32_t)(i0 * g.h + hd) * dw + sc, stager ? dw - sc : 0, xd[i]);
        }
        const int i0 = lane / g.group;
        const uint32_t at = (uint32_t)(i0 * g.h + lane - i0 * g.group) * 32u;
        r0 = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, at, 0, 0));
        r1 = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rr, at + 16u, 0, 0));
    }
    {
        f4 m = {0.f, 0.f, r1[2], max2(r0[1], fabsf(r0[3] * r1[3]))};
#pragma unroll
        for (int i = 0; i < CH; i++) m[0] = absmax8(xq[i], m[0]);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i != 1) m[i] = wave_max(m[i]);
        if (lane == 0) rmax[wave] = m;
        if (wave == 0) rdo[lane] = r1[2];
    }
    __syncthreads();
    f4 mx = rmax[0];
#pragma unroll
    for (int i = 1; i < 4; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) mx[e] = max2(mx[e], rmax[i][e]);
    // dO has a power of two of its row, that of the largest (dup) where it is 0
    const float qup = up_of(mx[0]), dup = up_of(mx[2]), pup = p_up(mx[3]);
    auto dup_of = [&](int row) { return rdo[row] > 0.f ? up_of(rdo[row]) : dup; };
    if (stager) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            _Float16 *p = qt + row_pos(sr + i * Stage::RPP) * Tile::STRIDE + sc;
            const Half2 hq = half_split(xq[i], qup), hd = half_split(xd[i], dup_of(sr + i * Stage::RPP));
            *(h8 *)p = hq.hi;
            *(h8 *)(p + Tile::PART) = hq.lo;
            *(h8 *)(p + SLOT) = hd.hi;
            *(h8 *)(p + SLOT + Tile::PART) = hd.lo;
        }
    }
    if (wave == 0) {
        rec[0][lane] = -r0[0];
        rec[1][lane] = r0[1] * pup;
        rec[2][lane] = -r0[2];
        rec[3][lane] = -r0[3] * r1[3] * pup;
        rec[4][lane] = -r1[0];
        rec[5][lane] = -r1[1];
    }
    const int rg = wave & 1, kg = wave >> 1, row = 32 * rg + lr;
    const int qi = row / g.group, head = kh * g.group + row % g.group;
    // the row's power of two of dO, what takes it to the rows' common one in dV (P has
    // it) and back in dS, and what bounds its dS
    const float ddown = down_of(dup_of(row)), pcommon = dup * ddown, nd = rdo[row];
    // 32 keys of the wave's row, in the order of an accumulator's registers
    auto put = [&](_Float16 *t, const Half2 (&x)[2]) {
        _Float16 *p = t + row_pos(row) * PTile::STRIDE + 32 * kg + 4 * lh;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            *(h4 *)(p + 16 * i) = __builtin_shufflevector(x[i].hi, x[i].hi, 0, 1, 2, 3);
            *(h4 *)(p + 16 * i + 8) = __builtin_shufflevector(x[i].hi, x[i].hi, 4, 5, 6, 7);
            *(h4 *)(p + PTile::PART + 16 * i) = __builtin_shufflevector(x[i].lo, x[i].lo, 0, 1, 2, 3);
            *(h4 *)(p + PTile::PART + 16 * i + 8) = __builtin_shufflevector(x[i].lo, x[i].lo, 4, 5, 6, 7);
        }
    };
    auto zero = [](f32x16 &x) {
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = 0.f;
    };
    f32x16 dq[2][CT];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int c = 0; c < CT; c++) zero(dq[m][c]);
    // keys that some row sees; the others' gradients are zeros
    const int kend = g.causal ? min(nk, nq + shift) : nq ? nk : 0;
    const int nt = ONE ? 1 : (g.tk + 63) / 64, flip = flip_at((max(kend, 0) + 63) / 64);
    // the largest value so far and powers of two (sup, own: of the lane's row), sgn: the
    // accumulators' sign
    float vmax = 0.f, kup = FIRST_UP, sup = FIRST_UP, sgn = 1.f, own[2] = {DS_START, DS_START};
    for (int t = 0; t < nt; t++) {
        const int k0 = 64 * t, key = k0 + 32 * rg + lr;  // of the wave's blocks of dK and dV
        const bool live = key < nk;
        float *const kv = g.dkv + ((long long)b * g.tk + min(key, g.tk - 1)) * g.kvstride + 2 * kh * g.dh;
        if (k0 >= kend) {  // (the accumulators are left as they are)
            f32x16 z;
            zero(z);
            for (int c = kg; c < W / 32 && key < g.tk; c += 2)
                put_channels<true>(kv + g.voff, dw, 32 * c, z, 0.f, 0.f, live, g.acc_kv);
            for (int c = 0; c < CT && key < g.tk; c++)
                put_channels<true>(kv + g.koff + kg * g.dh, g.dh, 32 * c, z, 0.f, 0.f, live, g.acc_kv);
            continue;
        }
        st.maxima(tmax, good_for(kup), vmax);
        __syncthreads();  // dS is read
        float mk = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mk = max2(mk, tmax[i][0]);
            vmax = max2(vmax, tmax[i][1]);
        }
        const float kup1 = sticky_up(mk, kup), vup = up_of(vmax);
        // (ONE: D is a mean of this tile's dA)
        const float dmax = ONE ? 0.f : max2(fabsf(rec[4][row]), fabsf(rec[5][row]));
        const float sup1 = ds_up(ds_bound<W>(nd, vmax, dmax), sup);
        float ratio = down_of(kup) * kup1 * (down_of(sup) * sup1);
        kup = kup1;
        sup = sup1;
        if (t == flip) {
            sgn = -1.f;
            ratio = -ratio;
        }
        st.store(kt, kup, vup, SLOT);
        if (!ONE && k0 + 64 < kend) st.load(k0 + 64);
        __syncthreads();
        const _Float16 *const k1 = kt + 32 * kg * Tile::STRIDE;
        Half2 ah[2], ds[2][2];
        f32x16 s[2];
        // what takes dS from the row's units, own's apart, to itself
        const float units = dup_of(row) * down_of(dup) * down_of(sup) * down_of(pup);
        {
            f32x16 da;
#pragma unroll
            for (int r = 0; r < 16; r++) s[0][r] = s[1][r] = da[r] = 0.f;
#pragma unroll
            for (int m = 0; m < 2; m++) {
                Half2 q[KS];
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    q[i].hi = Tile::along(qt, row, m * DHP + 16 * i + 8 * lh);
                    q[i].lo = Tile::along(qt + Tile::PART, row, m * DHP + 16 * i + 8 * lh);
                }
                dot_along<Tile>(k1, m * DHP, q, s[m]);
            }
            Half2 d[VS];
#pragma unroll
            for (int i = 0; i < VS; i++) {
                d[i].hi = Tile::along(dt, row, 16 * i + 8 * lh);
                d[i].lo = Tile::along(dt + Tile::PART, row, 16 * i + 8 * lh);
            }
            dot_along<Tile>(vt + 32 * kg * Tile::STRIDE, 0, d, da);
            const float f = down_of(kup) * (down_of(qup) * (g.scale * LOG2E));
            const float fd = da_unit(down_of(vup), ddown, sup);
            const float fd1 = fminf(fd * own[0], 0x1.fffffep127f), fd2 = fminf(fd * own[1], 0x1.fffffep127f);
            const float nm1 = rec[0][row], il1 = rec[1][row] * pcommon * sgn;
            const float nm2 = rec[2][row], il2 = rec[3][row] * pcommon * sgn;
            f32x16 a;
            auto softmax = [&](int r, float &p1, float &p2) {
                const int j = k0 + 32 * kg + 8 * (r >> 2) + 4 * lh + (r & 3);
                const bool in = j < nk && !(g.causal && j > qi + shift) && !(g.diag && j == qi);
                p1 = in ? exp_below(__builtin_fmaf(s[0][r], f, nm1)) * il1 : 0.f;
                p2 = in ? exp_below(__builtin_fmaf(s[1][r], f, nm2)) * il2 : 0.f;
                a[r] = p1 + p2;
            };
            if constexpr (ONE) {
                // D_m as the mean of these dA, whose rounding it shares: a row that sees
                // one key has dS = 0, and nothing but rounding would be left of it
                f4 ps = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float p1, p2;
                    softmax(r, p1, p2);
                    s[0][r] = p1;
                    s[1][r] = p2;
                    ps[0] += p1;
                    ps[1] = __builtin_fmaf(p1, da[r], ps[1]);
                    ps[2] += p2;
                    ps[3] = __builtin_fmaf(p2, da[r], ps[3]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) ps[i] = pair32(ps[i], add2);
                if (lh == 0) psum[kg][row] = ps;
                __syncthreads();
                ps = psum[0][row] + psum[1][row];
                const float D1 = ps[0] != 0.f ? -fd1 * (ps[1] / ps[0]) : 0.f;
                const float D2 = ps[2] != 0.f ? -fd2 * (ps[3] / ps[2]) : 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[0][r] *= __builtin_fmaf(da[r], fd1, D1);
                    s[1][r] *= __builtin_fmaf(da[r], fd2, D2);
                }
            } else {
                const float D1 = rec[4][row] * sup * own[0], D2 = rec[5][row] * sup * own[1];
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float p1, p2;
                    softmax(r, p1, p2);
                    s[0][r] = p1 * __builtin_fmaf(da[r], fd1, D1);
                    s[1][r] = p2 * __builtin_fmaf(da[r], fd2, D2);
                }
            }
            split16(a, ah);
            float m[2] = {absmax16(s[0]), absmax16(s[1])};
            if (__builtin_expect(__any(max2(m[0], m[1]) >= 0x1p15f || ratio != 1.0f), 0)) {
#pragma unroll
                for (int i = 0; i < 2; i++) scale_all(dq[i], ds_fit(s[i], m[i], own[i]) * ratio);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[i] = wave_max(m[i] * (down_of(own[i]) * units));
                split16(s[i], ds[i]);
            }
            if (lane == 0) smax[wave] = f2{m[0], m[1]};
        }
        __syncthreads();  // V is read
        put(vt, ah);
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int c = 0; c < CT; c++)
                dot_across<Tile>(k1, m * DHP + 32 * c, ds[m], dq[m][c]);
        // dK's sums run over the rows: dS once more, with one power of two for the tile
        float tup[2];
#pragma unroll
        for (int m = 0; m < 2; m++) {
            tup[m] = p_up(max2(max2(smax[0][m], smax[1][m]), max2(smax[2][m], smax[3][m])));
            const float f = tup[m] * (down_of(own[m]) * units);
#pragma unroll
            for (int r = 0; r < 16; r++) s[m][r] *= f;
            split16(s[m], ds[m]);
        }
        __syncthreads();  // K is read, P_1 - lambda P_2 there
        put(kt, ds[1]);
        for (int c = kg; c < W / 32; c += 2) {
            f32x16 dv;
            zero(dv);
            dot_tiles<Tile, PTile>(dt, 32 * c, vt, 32 * rg, dv);
            if (key < g.tk)
                put_channels<true>(kv + g.voff, dw, 32 * c, dv, down_of(dup) * sgn, down_of(pup),
                                   live, g.acc_kv);
        }
        __syncthreads();  // P_1 - lambda P_2 is read
        put(vt, ds[0]);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; c++) {
            f32x16 dk;
            zero(dk);
            dot_tiles<Tile, PTile>(qt, kg * DHP + 32 * c, kg ? kt : vt, 32 * rg, dk);
            if (key < g.tk)
                put_channels<true>(kv + g.koff + kg * g.dh, g.dh, 32 * c, dk,
                                   down_of(qup) * (g.scale * sgn),
                                   down_of(kg ? tup[1] : tup[0]), live, g.acc_kv);
        }
    }
    // the halves of dQ that waves (rg, 0) and (rg, 1) have, dS's own powers of two off
#pragma unroll
    for (int m = 0; m < 2; m++) scale_all(dq[m], down_of(own[m]) * (dup_of(row) * down_of(dup)));
    __syncthreads();
    float *const ex = (float *)kt + rg * 2 * CT * 16 * 64 + lane;
    auto each = [&](auto &&f) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int r = 0; r < 16; r++) f(ex[((m * CT + c) * 16 + r) * 64], dq[m][c], r);
    };
    if (kg) each([](float &e, f32x16 &v, int r) { e = v[r]; });
    __syncthreads();
    if (kg || qi >= g.tq) return;
    each([](float &e, f32x16 &v, int r) { v[r] += e; });
    float *dst = g.dq + ((long long)b * g.tq + qi) * g.qstride + 2 * head * g.dh;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int c = 0; c < CT; c++)
            put_channels<true>(dst + m * g.dh, g.dh, 32 * c, dq[m][c],
                               down_of(kup) * (g.scale * sgn), down_of(sup) * down_of(pup), qi < nq,
                               g.acc_q);
}

// The backward's first pass: lanes of a unit and blocks, so that the groups of
// lanes are a multiple of the heads and take about four units each.
struct PrePlan {
    int lpu;
    size_t blocks;
};
PrePlan plan_pre(const rnn_diff_attn_desc *d, size_t n, bool vec) {
    PrePlan p;
    p.lpu = !vec ? 64 : d->dh <= 16 ? 8 : d->dh <= 32 ? 16 : 32;
    const size_t gpb = 256 / p.lpu;
    size_t a = gpb, b = d->h;
    while (b) {
        const size_t r = a % b;
        a = b;
        b = r;
    }
    const size_t mult = d->h / a, units = n * d->tq * d->h;
    p.blocks = std::max<size_t>(1, std::min<size_t>(rnn_div_up(units, 4 * gpb), 1024) / mult) * mult;
    return p;
}

// Row groups of 32 a workgroup of the forward, and the splits of the keys: a
// power of two of groups up to four, keys split where the rows leave half of the
// CUs idle (2 x 8 causal heads of 1568 rows and keys, dh 64, 208 workgroups: 111 us
// unsplit, 124 and 24 for the join with two splits), down to a tile a split where
// the partial sums are small (11 x 1 query over 473 keys, dh 64, 12 + 4 us; with four
// tiles 24.5 + 4).  Above 32 channels, where LDS holds one workgroup a CU, two row
// groups with two waves on each row where four would not fill the CUs (208
// workgroups: 90 us against 122; 8 heads of 2048: 110 against 157; 256 workgroups, 8
// heads of 4096: 390 against 333; at 32 channels 8 x 6 heads of 577: 46.9 against
// 36.2).
struct FwdPlan {
    int qg, splits, split_keys;
    bool halves;  // two waves share a row's keys
    size_t blocks;
};
FwdPlan plan_fwd(const rnn_diff_attn_desc *d, size_t n, bool vec) {
    FwdPlan p;
    const size_t R = (size_t)d->tq * (d->h / d->hkv), probs = n * d->hkv;
    p.qg = !vec ? 4 : R <= 32 ? 1 : R <= 64 ? 2 : 4;
    p.blocks = probs * rnn_div_up(R, (size_t)32 * p.qg);
    const size_t tiles = rnn_div_up(d->tk, (size_t)64);
    const size_t least = p.blocks <= 16 ? 1 : p.blocks <= 64 ? 2 : 4;  // tiles of a split
    size_t s = p.blocks && p.blocks < 128 && tiles >= 4 ? std::min(tiles / least, 512 / p.blocks) : 1;
    s = std::max<size_t>(1, std::min<size_t>(s, 64));
    const size_t per = rnn_div_up(std::max<size_t>(tiles, 1), s);
    p.split_keys = (int)per * 64;
    p.splits = (int)rnn_div_up(std::max<size_t>(tiles, 1), per);
    p.halves = false;
    if (p.qg == 4 && vec && d->dh > 32 && p.splits == 1 && p.blocks < 256) {
        p.halves = true;
        p.qg = 2;
        p.blocks = probs * rnn_div_up(R, (size_t)64);
    }
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
        size_t part = 0;  // whichever alignment the operands turn out to have
        for (int vec = 0; vec < 2; vec++) {
            const PrePlan p = plan_pre(d, n, vec != 0);
            part = std::max(part, p.blocks * (2 * d->dh + 256 / p.lpu));
        }
        w.part = cv.take(part * sizeof(double));
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
    const size_t lim = 0x3fffffffu;  // (a grid's stride past a row's number stays an int)
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

// Blocks in launches of at most 2^31 threads (a grid holds below 2^32): f(g, blocks)
// with g.first their first.
template <typename F>
void in_launches(DiffArgs g, size_t blocks, size_t threads, F &&f) {
    const size_t most = ((size_t)1 << 31) / threads;
    for (size_t b = 0; b < blocks; b += most) {
        g.first = (long long)b;
        f(g, (unsigned)std::min(most, blocks - b));
    }
}

template <int DHP, bool VEC, int QG, int KH = 1>
void launch_fwd_qg(rnn_ctx *ctx, const DiffArgs &g, const FwdPlan &p) {
    if constexpr (KH == 1) {
        if (p.splits > 1) {
            const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
            diff_fwd_kernel<DHP, VEC, QG, 1, true><<<grid, 128 * QG, 0, ctx->stream>>>(g);
            return;
        }
    }
    in_launches(g, p.blocks, 128 * QG * KH, [&](const DiffArgs &a, unsigned blocks) {
        diff_fwd_kernel<DHP, VEC, QG, KH, false><<<blocks, 128 * QG * KH, 0, ctx->stream>>>(a);
    });
}
template <int DHP>
void launch_fwd(rnn_ctx *ctx, const DiffArgs &g, const FwdPlan &p, bool vec) {
    if (!vec)
        launch_fwd_qg<DHP, false, 4>(ctx, g, p);
    else if (p.qg == 1)
        launch_fwd_qg<DHP, true, 1>(ctx, g, p);
    else if (DHP > 32 && p.halves)
        launch_fwd_qg<DHP, true, 2, (DHP > 32 ? 2 : 1)>(ctx, g, p);
    else if (p.qg == 2)
        launch_fwd_qg<DHP, true, 2>(ctx, g, p);
    else
        launch_fwd_qg<DHP, true, 4>(ctx, g, p);
}

// The blocks for the parameters' gradients, params_blocks on the host.
unsigned params_of(const DiffArgs &g) {
    return g.first ? 0u : (g.dgain ? (2u * g.dh + 15u) / 16u : 0u) + (unsigned)g.lam_heads;
}

template <int DHP, bool VEC, int RG, int KG, int NM = 2>
void launch_dq(rnn_ctx *ctx, const DiffArgs &g) {
    const size_t R = (size_t)g.tq * g.group;
    constexpr int threads = 128 / NM * RG * KG;
    in_launches(g, (size_t)g.n * g.hkv * rnn_div_up(R, 32 * RG), threads, [&](const DiffArgs &a, unsigned blocks) {
        diff_dq_kernel<DHP, VEC, RG, KG, NM><<<blocks + params_of(a), threads, 0, ctx->stream>>>(a);
    });
}
template <int DHP, bool VEC, int KG>
void launch_dkv(rnn_ctx *ctx, const DiffArgs &g) {
    const size_t total = (size_t)g.n * g.hkv * rnn_div_up((size_t)g.tk, 32 * KG);
    in_launches(g, total, 128 * KG, [&](const DiffArgs &a, unsigned blocks) {
        diff_dkv_kernel<DHP, VEC, KG><<<blocks, 128 * KG, 0, ctx->stream>>>(a);
    });
}
// Joint kernel for up to 64 rows where one tile holds the keys or problems fill the
// CUs (128 x 4 heads of 64 rows on 256 keys 47 us, apart 29 + 53).
// dQ: two waves share 32 rows where four groups of 32 would not fill the CUs (2 x 8
// causal heads of 1568, dh 64: 108 us against 173; 8 x 6 of 577, dh 32: 42.0 against
// 42.4; 4 x 8 of 2048, dh 64: 503 against 500; 32 x 8 of 256, dh 64: 123 against 91).
// dK and dV: four waves on two groups of 32 keys; above 32 channels, where a CU
// holds one workgroup, eight on four where those fill the CUs (eight against four in
// the same cases: 195 against 182 us; 58.3 against 59.0; 569 against 917; 103 against
// 159).  Operands that are not whole float4s take one plan each, unmeasured.
template <int DHP>
void launch_bwd(rnn_ctx *ctx, const DiffArgs &g, bool vec) {
    const size_t probs = (size_t)g.n * g.hkv, R = (size_t)g.tq * g.group;
    if (vec && g.tq && R <= 64 && g.tk && (g.tk <= 64 || probs >= 256)) {
        in_launches(g, probs, 256, [&](const DiffArgs &a, unsigned blocks) {
            if (g.tk <= 64)
                diff_bwd_rows_kernel<DHP, true><<<blocks + params_of(a), 256, 0, ctx->stream>>>(a);
            else
                diff_bwd_rows_kernel<DHP, false><<<blocks + params_of(a), 256, 0, ctx->stream>>>(a);
        });
        return;
    }
    if (g.tq) {
        if (!vec)
            launch_dq<DHP, false, 4, 1>(ctx, g);
        else if (R <= 32)
            launch_dq<DHP, true, 1, 2>(ctx, g);
        else if (R <= 64 || probs * rnn_div_up(R, 128) < 256)
            launch_dq<DHP, true, 2, 2, (DHP <= 32 ? 2 : 1)>(ctx, g);
        else
            launch_dq<DHP, true, 4, 1>(ctx, g);
    }
    if (g.tk) {
        if (!vec)
            launch_dkv<DHP, false, 2>(ctx, g);
        else if (g.tk <= 32)
            launch_dkv<DHP, true, 1>(ctx, g);
        else if (DHP > 32 && probs * rnn_div_up((size_t)g.tk, 128) >= 256)
            launch_dkv<DHP, true, (DHP > 32 ? 4 : 2)>(ctx, g);
        else
            launch_dkv<DHP, true, 2>(ctx, g);
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
        const size_t units = n * d->tq * d->h;
        if (p.splits > 4)
            diff_join_kernel<4><<<(unsigned)units, 256, 0, ctx->stream>>>(g, p.splits);
        else
            diff_join_kernel<1><<<(unsigned)rnn_div_up(units, 4), 256, 0, ctx->stream>>>(g, p.splits);
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
    g.dlam = dlam;
    g.dgain = dgain;
    const bool vec = rows_vec(g);
    const size_t rows = n * d->tq;
    if (rows) {
        const PrePlan p = plan_pre(d, n, vec);
        const unsigned nblk = (unsigned)p.blocks;
        g.nblk = (int)nblk;
        g.gpb = 256 / p.lpu;
        if (p.lpu == 8)
            diff_bwd_pre_kernel<8><<<nblk, 256, 0, ctx->stream>>>(g);
        else if (p.lpu == 16)
            diff_bwd_pre_kernel<16><<<nblk, 256, 0, ctx->stream>>>(g);
        else if (p.lpu == 32)
            diff_bwd_pre_kernel<32><<<nblk, 256, 0, ctx->stream>>>(g);
        else
            diff_bwd_pre_kernel<64><<<nblk, 256, 0, ctx->stream>>>(g);
        RNN_LAUNCHED(ctx);
    }
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
