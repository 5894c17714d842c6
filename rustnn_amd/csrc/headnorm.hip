// Norms of heads: with the rotary position in the same pass (rnn_norm_rotary),
// and times SiLU of a gate (rnn_head_gate); forward and backward.  No
// counterpart in the reference.
//
//   x^ = x / sqrt(mean x^2 + eps) over a head's channels, u = gain x^
//   du -> dgain = sum du x^, t = du gain, dx = (t - x^ mean(t x^)) / sqrt(..)
//
// One read of each input and one write of each output: HBM-bound.  A head is
// owned by L lanes (a power of two) of eight channels each, held in registers
// between the sum and its use; groups of L lanes take consecutive heads, so
// that a wave reads whole lines; the next head's loads are in flight while one is
// worked on.  Squares are summed in 64 bits: a square passes a float's range from
// 2^64 on and falls below it from 2^-75.  So are the sums over lanes and rows.
//
// 25088 rows, where a copy of that size runs at 5.0 TB/s: norm and turn of 24 heads
// of 64 channels 58 us forward (5.3 TB/s) and 104 us backward (4.5), 8 gated heads
// of 64 channels 26 us (5.8: they stay in the last cache) and 48 (5.3), each
// backward 5 us more for the gains' gradient.  64 rows take 6 us, a launch's least.
#include "rnn_overlap.h"
#include "rotary_angle.h"

#include <algorithm>

namespace {

constexpr int MAX_HEAD = 256;      // channels of a head with rotary positions
constexpr int MAX_GATE = 512;      // channels of a gated head
constexpr int MAX_BLOCKS = 1024;   // of a forward: 4 a CU
constexpr int MAX_PARTS = 768;     // of a backward: 3 a CU, each leaving its part of dgain
constexpr int TABLE = 512;         // sines and cosines of a block's rows

// The sum over the L lanes of a group, every lane receiving it, in a fixed tree.
__device__ __forceinline__ double group_sum(double v, int L) {
    if (L > 1) v += rnn_dpp_d<0xB1>(v);
    if (L > 2) v += rnn_dpp_d<0x4E>(v);
    if (L > 4) v += rnn_dpp_d<0x141>(v);
    if (L > 8) v += rnn_dpp_d<0x140>(v);
    if (L > 16) v += __shfl_xor(v, 16, 64);
    if (L > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// 1 / sqrt(v): the instruction's approximation, within 2^-23, and a Newton step on
// it, which leaves 3/2 of its square: 1.5 2^-46.  0 of infinity.
__device__ __forceinline__ double inv_sqrt(double v) {
    const double r = __builtin_amdgcn_rsq(v), s = fma(0.5 * r, fma(-v * r, r, 1.0), r);
    return r == 0.0 ? r : s;
}

// sigma(z) = 1 / (1 + exp(-z)) = s down, s within 6.5 U (U = 2^-24).  exp(-z) as a power
// of two, its exponent in two parts, so that far gates lose nothing: the
// instruction's 2 U and two products; the sum's U; its reciprocal by the instruction
// (2 U) and a Newton step on it: 1.5 U.  From exp(-z) = 2^100 on (z = -69) all of it is
// taken 2^64 smaller, down = 2^-64, so that the reciprocal, which gives 0 for what is
// below the normal range, stays in it: z sigma, a normal number down to z = -91, is right
// to its last bit below that.  `down` is multiplied last; s z and s alone are below
// 1 where it is not 1.  From -120 on z sigma is below half of the least number: s = 0.
struct Sigma {
    float s, down;
    __device__ __forceinline__ explicit Sigma(float z) {
        const float c = __builtin_amdgcn_fmed3f(z, -120.f, 104.f);
        const float t = c * -1.44269504f;
        const float lo = __builtin_fmaf(c, -1.44269504f, -t) + c * -1.92596299e-8f;
        const bool far = t > 100.f;
        down = far ? 0x1p-64f : 1.f;
        const float e = __builtin_amdgcn_exp2f(far ? t - 64.f : t) * __builtin_fmaf(lo, 0.69314718f, 1.f);
        const float d = down + e, r = __builtin_amdgcn_rcpf(d);
        s = z < -120.f ? 0.f : __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r);
    }
};

// x^ in 32 bits whatever the head's size: 1 / norm as a float of [1, 2) times a
// power of two, which the channels take first.
struct Norm32 {
    float r, up;  // 1 / norm = r up
    __device__ __forceinline__ explicit Norm32(double rn) {
        const int e = (int)((uint64_t)__double_as_longlong(rn) >> 52) - 1023;
        const int k = max(-126, min(e, 126));
        up = __uint_as_float((uint32_t)(k + 127) << 23);
        r = (float)(rn * (double)__uint_as_float((uint32_t)(127 - k) << 23));
    }
    __device__ __forceinline__ float operator()(float v) const { return v * up * r; }
};

// Eight sums a lane over the groups of a block (256 threads), to out[e] by the
// first group's lanes: store(lane of the group, e, sum).
template <typename F>
__device__ __forceinline__ void block_sum8(double (&v)[8], int L, F store) {
    __shared__ double red[4 * 64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < 8; e++)
        for (int m = L; m < 64; m <<= 1) v[e] += __shfl_xor(v[e], m, 64);
    __syncthreads();
    if (lane < L) {
#pragma unroll
        for (int e = 0; e < 8; e++) red[(wave * 64 + lane) * 8 + e] = v[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < L * 8; i += 256) {
        double s = red[i];
        for (int w = 1; w < 4; w++) s += red[w * 512 + i];
        store(i >> 3, i & 7, s);
    }
}

// ------------------------------------------------------ norm and rotary
struct NrArgs {
    const float *x, *pos, *gain, *dy;
    float *y;      // the backward's dx
    double *part;  // [blocks][2][dh]
    long long xstride, ystride, dystride;
    int rows, t, h, hq, dh, axes, npairs;
    int p0, p1;  // pairs of the first two axes
    int g1, g2;  // grid sides of the last two axes
    int lanes, rpb, span;  // a block's rows, of which rpb at a time
    double eps;
    double w[MAX_PAIRS];  // quarter turns per unit of position of every pair
};

// Four channels at p, of which the first n are there.  16-byte accesses need 4-byte
// alignment alone.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void load4(const float *p, int n, float *v) {
    if (n == 4) {
        const f4u t = *(const f4u *)p;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = e < n ? p[e] : 0.f;
    }
}
__device__ __forceinline__ void store4(float *p, int n, const float *v) {
    if (n == 4) {
        *(f4u *)p = f4u{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < n) p[e] = v[e];
    }
}

// A lane's channels: two runs of four, from ca and cb on (na and nb of them are
// there), neighbouring lanes' runs next to each other, so that an access takes whole
// lines (eight channels a lane in one piece: a gate's forward 60 us against 32).
// Lanes before T hold four pairs: (j, j + R) of the two runs, or, alternating, two
// pairs of each run, which then are two halves of the pairs where those are a
// multiple of four; lanes past them channels that do not turn.  As elements, e < 4
// is the first channel of the lane's pair e and e >= 4 the second one of pair e - 4.
template <bool INTER>
struct NrLane {
    int ca, cb, na, nb, u, R;
    bool turned, halves;
    __device__ __forceinline__ NrLane(const NrArgs &g, int lane) : u(lane), R(g.npairs) {
        const int T = (R + 3) / 4, n = (g.dh - 2 * R + 7) / 8, v = u - T;
        turned = u < T;
        halves = R % 4 == 0;
        if (turned) {
            const int pairs = min(R - 4 * u, 4);
            ca = INTER && !halves ? 8 * u : 4 * u;
            cb = INTER && !halves ? 8 * u + 4 : R + 4 * u;
            na = INTER ? min(2 * pairs, 4) : pairs;
            nb = INTER ? 2 * pairs - na : pairs;
        } else {
            ca = 2 * R + 4 * v;
            cb = 2 * R + 4 * (n + v);
            na = v < n ? min(max(g.dh - ca, 0), 4) : 0;
            nb = v < n ? min(max(g.dh - cb, 0), 4) : 0;
        }
    }
    // the pair of elements q and q + 4
    __device__ __forceinline__ int pair(int q) const {
        return INTER && halves ? (q < 2 ? 2 * u + q : R / 2 + 2 * u + q - 2) : 4 * u + q;
    }
    // element e's place in the two runs, and its channel; -1: none
    static __device__ __forceinline__ constexpr int place(int e) {
        return INTER ? (e < 4 ? 2 * e : 2 * e - 7) : e;
    }
    __device__ __forceinline__ int channel(int e) const {
        const int p = place(e);
        return p < 4 ? (p < na ? ca + p : -1) : p - 4 < nb ? cb + p - 4 : -1;
    }
    __device__ __forceinline__ void load(const float *p, float (&v)[8]) const {
        float t[8];
        load4(p + ca, na, t);
        load4(p + cb, nb, t + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = t[place(e)];
    }
    __device__ __forceinline__ void store(float *p, const float (&v)[8]) const {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[place(e)] = v[e];
        store4(p + ca, na, t);
        store4(p + cb, nb, t + 4);
    }
};

// A block has `span` rows, of which it takes `rpb` at a time: their sines and cosines
// into LDS, formed once for all heads while the first heads' loads are in flight, then
// every head.  Four blocks of a forward a CU: for five the loads ahead do not fit the
// registers (25088 rows 64 us against 58, 8177 rows of 52 channels 18 against 12).
// Queries and then keys go over the lane groups in rounds, whose last ones may be
// partly empty: 8 rows of 6 + 2 heads on 32 groups take three for the work of two.
template <bool INTER, bool BACK>
__global__ __launch_bounds__(256, BACK ? 3 : 4) void norm_rotary_kernel(NrArgs g) {
    __shared__ __attribute__((aligned(16))) float2 tab[TABLE];
    const int L = g.lanes, R = g.npairs;
    const int ng = 256 / L, grp = threadIdx.x / L;
    using Lane = NrLane<INTER>;
    const Lane own(g, threadIdx.x & (L - 1));
    float gain[2][8];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = own.channel(e);
            gain[k][e] = c < 0 ? 0.f : g.gain ? g.gain[k * g.dh + c] : 1.f;
        }
    double acc[2][8];
    if constexpr (BACK) {
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) acc[k][e] = 0.0;
    }
    const double inv = 1.0 / g.dh;
    const long long begin = (long long)blockIdx.x * g.span, end = min(begin + g.span, (long long)g.rows);
    float v[8], d[8], nv[8], nd[8];
    long long r, nr;
    int hd, lr, nhd, nlr;
    for (long long row0 = begin; row0 < end; row0 += g.rpb) {
        const int nrow = (int)min((long long)g.rpb, end - row0);
        // item `it` of the queries' (k = 0) or the keys' heads, into the next registers
        const auto fetch = [&](int k, int it) {
            const int hn = k ? g.h - g.hq : g.hq;
            it = min(it, nrow * hn - 1);
            nlr = it / hn;
            nhd = it - nlr * hn + k * g.hq;
            nr = row0 + nlr;
            own.load(g.x + nr * g.xstride + nhd * g.dh, nv);
            if constexpr (BACK) own.load(g.dy + nr * g.dystride + nhd * g.dh, nd);
        };
        fetch(g.hq ? 0 : 1, grp);
        __syncthreads();
        for (int e = threadIdx.x; e < nrow * R; e += 256) {
            const int lr = e / R, j = e - lr * R;
            float sn, cs;
            rot_sincos(rot_position(g, (int)row0 + lr, j) * g.w[j], &sn, &cs);
            tab[e] = make_float2(cs, BACK ? -sn : sn);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int items = nrow * (k ? g.h - g.hq : g.hq);
            for (int i0 = 0; i0 < items; i0 += ng) {
                const bool live = i0 + grp < items;
                r = nr, hd = nhd, lr = nlr;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[e] = nv[e];
                    if constexpr (BACK) d[e] = nd[e];
                }
                if (i0 + ng < items)
                    fetch(k, i0 + ng + grp);
                else if (k == 0 && g.hq < g.h)
                    fetch(1, grp);
                double s = 0.0;
#pragma unroll
                for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
                const double rn = inv_sqrt(group_sum(s, L) * inv + g.eps);
                float o[8];
                if constexpr (!BACK) {
#pragma unroll
                    for (int e = 0; e < 8; e++) d[e] = (float)(v[e] * rn) * gain[k][e];
                }
                if (own.turned) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const float2 w = tab[lr * R + min(own.pair(q), R - 1)];
                        o[q] = __builtin_fmaf(d[q], w.x, -(d[q + 4] * w.y));
                        o[q + 4] = __builtin_fmaf(d[q + 4], w.x, d[q] * w.y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = d[e];
                }
                if constexpr (BACK) {
                    const Norm32 hat32(rn);
                    float hat[8], m32 = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        hat[e] = hat32(v[e]);
                        if (live) acc[k][e] = fma((double)o[e], (double)hat[e], acc[k][e]);
                        o[e] *= gain[k][e];
                        m32 = __builtin_fmaf(o[e], hat[e], m32);
                    }
                    m32 = (float)(group_sum((double)m32, L) * inv);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        o[e] = hat32(__builtin_fmaf(-hat[e], m32, o[e]));
                }
                if (live) own.store(g.y + r * g.ystride + hd * g.dh, o);
            }
        }
    }
    if constexpr (BACK) {
        if (!g.part) return;
#pragma unroll
        for (int k = 0; k < 2; k++)
            block_sum8(acc[k], L, [&](int lane, int e, double s) {
                const int c = Lane(g, lane).channel(e);
                if (c >= 0) g.part[((long long)blockIdx.x * 2 + k) * g.dh + c] = s;
            });
    }
}

// ------------------------------------------------------------ gated heads
struct GateArgs {
    const float *x, *z, *gain, *dy;
    float *y, *dz;  // y: the backward's dx
    double *part;   // [splits][h * d]
    long long zstride, dzstride;
    long long rows;
    int h, d, lanes;
    double eps;
};

// Block b: head b % h, rows (b / h) * groups + group, and every splits * groups
// further, so that dgain's sums stay with one head's channels.
template <bool BACK>
__global__ __launch_bounds__(256) void head_gate_kernel(GateArgs g) {
    const int L = g.lanes, ng = 256 / L, at = threadIdx.x / L, u = threadIdx.x & (L - 1);
    const int head = blockIdx.x % g.h, split = blockIdx.x / g.h, splits = gridDim.x / g.h;
    // four channels from c on, and four from c2 on
    const int c = 4 * u, c2 = 4 * (L + u), col = head * g.d;
    const int n1 = min(max(g.d - c, 0), 4), n2 = min(max(g.d - c2, 0), 4);
    const auto load = [&](const float *p, float (&v)[8]) {
        load4(p + col + c, n1, v);
        load4(p + col + c2, n2, v + 4);
    };
    const auto store = [&](float *p, const float (&v)[8]) {
        store4(p + col + c, n1, v);
        store4(p + col + c2, n2, v + 4);
    };
    const long long w = (long long)g.h * g.d;
    float gain[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int at = e < 4 ? c + e : c2 + e - 4;
        gain[e] = at >= g.d ? 0.f : g.gain ? g.gain[col + at] : 1.f;
    }
    double acc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.0;
    const double inv = 1.0 / g.d;
    const long long step = (long long)splits * ng;
    float v[8], z[8], d[8], nv[8], nz[8], nd[8];
    long long r, nr;
    auto fetch = [&](long long at) {
        nr = min(at, g.rows - 1);
        load(g.x + nr * w, nv);
        load(g.z + nr * g.zstride, nz);
        if constexpr (BACK) load(g.dy + nr * w, nd);
    };
    fetch((long long)split * ng + at);
    for (long long r0 = (long long)split * ng; r0 < g.rows; r0 += step) {
        const bool live = r0 + at < g.rows;
        r = nr;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = nv[e], z[e] = nz[e];
            if constexpr (BACK) d[e] = nd[e];
        }
        if (r0 + step < g.rows) fetch(r0 + step + at);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
        const double rn = inv_sqrt(group_sum(s, L) * inv + g.eps);
        float o[8];
        if constexpr (!BACK) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const Sigma sg(z[e]);
                o[e] = (float)(v[e] * rn) * gain[e] * (z[e] * sg.s) * sg.down;
            }
        } else {
            const Norm32 hat32(rn);
            float dz[8], hat[8], m32 = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const Sigma sg(z[e]);
                const float f = 1.f + z[e] * __builtin_fmaf(-sg.s, sg.down, 1.f);
                hat[e] = hat32(v[e]);
                dz[e] = d[e] * (hat[e] * gain[e]) * (sg.s * f) * sg.down;
                o[e] = d[e] * (z[e] * sg.s) * sg.down;
                if (live) acc[e] = fma((double)o[e], (double)hat[e], acc[e]);
                o[e] *= gain[e];
                m32 = __builtin_fmaf(o[e], hat[e], m32);
            }
            m32 = (float)(group_sum((double)m32, L) * inv);
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = hat32(__builtin_fmaf(-hat[e], m32, o[e]));
            if (live) store(g.dz + r * g.dzstride, dz);
        }
        if (live) store(g.y + r * w, o);
    }
    if constexpr (BACK) {
        if (!g.part) return;
        block_sum8(acc, L, [&](int lane, int e, double s) {
            const int at = e < 4 ? 4 * lane + e : 4 * (L + lane) + e - 4;
            if (at < g.d) g.part[split * w + col + at] = s;
        });
    }
}

// out[j] += the sum of part [nrow][len]'s column j, four columns a block: each over
// 64 groups of rows in order, then over the groups.
__global__ __launch_bounds__(256) void gain_reduce_kernel(int nrow, int len, const double *part,
                                                          float *out) {
    __shared__ double red[64][4];
    const int q = threadIdx.x >> 2, j = threadIdx.x & 3, col = (int)blockIdx.x * 4 + j;
    const int G = (nrow + 63) / 64, k0 = min(nrow, q * G), k1 = min(nrow, k0 + G);
    double s = 0.0;
    for (int k = k0; k < k1; k += 16) {
        double v[16];
#pragma unroll
        for (int i = 0; i < 16; i++)
            v[i] = k + i < k1 && col < len ? part[(size_t)(k + i) * len + col] : 0.0;
#pragma unroll
        for (int i = 0; i < 16; i++) s += v[i];
    }
    red[q][j] = s;
    __syncthreads();
    if (threadIdx.x >= 4 || col >= len) return;
    double t = red[0][j];
    for (int i = 1; i < 64; i++) t += red[i][j];
    out[col] += (float)t;
}

// ---------------------------------------------------------------- plans
int pow2_lanes(int units) {
    int L = 1;
    while (L < units) L *= 2;
    return L;
}

// Blocks for `all` pieces of work, at most `most`, with as many pieces each.
size_t even_blocks(size_t all, size_t most) { return rnn_div_up(all, rnn_div_up(all, most)); }

struct NrPlan {
    int lanes, rpb, span, blocks;
};
NrPlan nr_plan(const rnn_rotary_desc *d, size_t rows, size_t most) {
    NrPlan p;
    const int R = (int)(d->p0 + d->p1 + d->p2);
    p.lanes = pow2_lanes((R + 3) / 4 + ((int)d->dh - 2 * R + 7) / 8);
    // a row's blocks at most, as many rows each; of those, enough at a time for a
    // sine and cosine a thread
    p.span = (int)rnn_div_up(rows, most);
    p.rpb = std::min(p.span, R ? std::min(32, (int)rnn_div_up(256, R)) : 8);
    p.blocks = (int)rnn_div_up(rows, p.span);
    return p;
}

int nr_check(rnn_ctx *ctx, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n, size_t t,
             bool have_pos) {
    const int rc = rnn_rotary_checked(ctx, d, n, t, have_pos);
    if (rc) return rc;
    if (hq > d->h)
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: %u query heads of %u", hq, d->h);
    if (!(eps > 0.0f) || !std::isfinite(eps))
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: eps %g", (double)eps);
    if (d->dh > (uint32_t)MAX_HEAD)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "norm_rotary: %u channels a head (up to %d)", d->dh,
                        MAX_HEAD);
    return RNN_OK;
}

void nr_fill(NrArgs &g, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n, size_t t,
             const float *x, const float *gain, const float *pos, float *y) {
    g.x = x + d->xoff;
    g.pos = pos;
    g.gain = gain;
    g.dy = nullptr;
    g.y = y + d->yoff;
    g.part = nullptr;
    g.xstride = (long long)d->xstride;
    g.ystride = (long long)d->ystride;
    g.dystride = 0;
    g.rows = (int)(n * t);
    g.t = (int)t;
    g.h = (int)d->h;
    g.hq = (int)hq;
    g.dh = (int)d->dh;
    g.axes = (int)d->axes;
    g.npairs = (int)(d->p0 + d->p1 + d->p2);
    g.p0 = (int)d->p0;
    g.p1 = (int)d->p1;
    g.g1 = (int)d->g1;
    g.g2 = (int)d->g2;
    g.eps = (double)eps;
    rot_frequencies(d, g.w);
}

template <bool BACK>
void nr_launch(rnn_ctx *ctx, const NrArgs &g, int blocks, bool inter) {
    if (inter)
        norm_rotary_kernel<true, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
    else
        norm_rotary_kernel<false, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
}

struct GatePlan {
    int lanes;
    size_t splits, parts;  // of a forward, of a backward
};
GatePlan gate_plan(size_t rows, size_t h, size_t d) {
    GatePlan p;
    p.lanes = pow2_lanes((int)rnn_div_up(d, 8));
    const size_t all = rnn_div_up(rows, 256 / p.lanes);
    p.splits = even_blocks(all, std::max<size_t>(1, MAX_BLOCKS / h));
    p.parts = even_blocks(all, std::max<size_t>(1, MAX_PARTS / h));
    return p;
}

int gate_check(rnn_ctx *ctx, size_t rows, size_t h, size_t d, size_t zstride, size_t zoff, float eps) {
    if (!h || !d) return rnn_fail(ctx, RNN_E_INVALID, "head_gate: zero heads or channels");
    if (!(eps > 0.0f) || !std::isfinite(eps))
        return rnn_fail(ctx, RNN_E_INVALID, "head_gate: eps %g", (double)eps);
    if (d > MAX_GATE)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "head_gate: %zu channels a head (up to %d)", d, MAX_GATE);
    if (h > 65536) return rnn_fail(ctx, RNN_E_UNSUPPORTED, "head_gate: %zu heads", h);
    if (zoff > zstride || zstride - zoff < h * d)
        return rnn_fail(ctx, RNN_E_INVALID, "head_gate: %zu channels do not fit a row", h * d);
    if (zstride > ((size_t)1 << 31) || rows > ((size_t)1 << 31))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "head_gate: %zu rows of %zu", rows, zstride);
    return RNN_OK;
}

int ws_checked(rnn_ctx *ctx, const char *what, size_t need, const void *ws, size_t bytes) {
    if (!need) return RNN_OK;
    if (!ws) return rnn_fail(ctx, RNN_E_NULL, "%s: workspace is null", what);
    if (bytes < need)
        return rnn_fail(ctx, RNN_E_INVALID, "%s: workspace of %zu bytes, needs %zu", what, bytes, need);
    if ((uintptr_t)ws & 255) return rnn_fail(ctx, RNN_E_INVALID, "%s: workspace not 256-byte aligned", what);
    return RNN_OK;
}

}  // namespace

extern "C" {

int rnn_norm_rotary_workspace(const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n, size_t t,
                              int have_pos, size_t *bytes) {
    const int rc = nr_check(nullptr, d, hq, eps, n, t, have_pos != 0);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    const size_t rows = n * t;
    *bytes = rows ? (size_t)nr_plan(d, rows, MAX_PARTS).blocks * 2 * d->dh * sizeof(double) : 0;
    return RNN_OK;
}

int rnn_norm_rotary_forward(rnn_ctx *ctx, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n,
                            size_t t, const float *x, const float *gain, const float *pos, float *y) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    const int rc = nr_check(ctx, d, hq, eps, n, t, pos != nullptr);
    if (rc) return rc;
    if (!(n * t)) return RNN_OK;
    if (!x || !y) return rnn_fail(ctx, RNN_E_NULL, "norm_rotary: null operand");
    const size_t width = (size_t)d->h * d->dh;
    const bool in_place = x + d->xoff == y + d->yoff && d->xstride == d->ystride;
    const RnnRows ins[] = {{in_place ? nullptr : x + d->xoff, n * t, d->xstride, width},
                           rnn_block(gain, 2 * (size_t)d->dh),
                           rnn_block(pos, n * t * d->axes)};
    const RnnRows outs[] = {{y + d->yoff, n * t, d->ystride, width}};
    if (rnn_any_overlap(outs, ins)) return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: y over an operand");
    RNN_ON_DEVICE(ctx);
    NrArgs g;
    nr_fill(g, d, hq, eps, n, t, x, gain, pos, y);
    const NrPlan p = nr_plan(d, n * t, MAX_BLOCKS);
    g.lanes = p.lanes;
    g.rpb = p.rpb;
    g.span = p.span;
    nr_launch<false>(ctx, g, p.blocks, d->interleaved != 0);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_norm_rotary_backward(rnn_ctx *ctx, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n,
                             size_t t, const float *x, const float *gain, const float *pos,
                             const float *dy, size_t dystride, size_t dyoff, void *ws, size_t ws_bytes,
                             float *dx, float *dgain) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = nr_check(ctx, d, hq, eps, n, t, pos != nullptr);
    if (rc) return rc;
    const size_t width = (size_t)d->h * d->dh;
    if (dyoff > dystride || dystride - dyoff < width)
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: %zu channels do not fit a row of dy", width);
    if (!(n * t)) return RNN_OK;
    if (!x || !dy || !dx) return rnn_fail(ctx, RNN_E_NULL, "norm_rotary: null operand");
    if (!gain && dgain) return rnn_fail(ctx, RNN_E_NULL, "norm_rotary: dgain without gain");
    const bool in_place = dx + d->yoff == dy + dyoff && d->ystride == dystride;
    const RnnRows ins[] = {{x + d->xoff, n * t, d->xstride, width},
                           {in_place ? nullptr : dy + dyoff, n * t, dystride, width},
                           rnn_block(gain, 2 * (size_t)d->dh),
                           rnn_block(pos, n * t * d->axes),
                           rnn_block(dgain, 2 * (size_t)d->dh)};
    const RnnRows outs[] = {{dx + d->yoff, n * t, d->ystride, width}};
    if (rnn_any_overlap(outs, ins))
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: dx over another operand");
    const NrPlan p = nr_plan(d, n * t, MAX_PARTS);
    rc = ws_checked(ctx, "norm_rotary", dgain ? (size_t)p.blocks * 2 * d->dh * sizeof(double) : 0, ws,
                    ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    NrArgs g;
    nr_fill(g, d, hq, eps, n, t, x, gain, pos, dx);
    g.dy = dy + dyoff;
    g.dystride = (long long)dystride;
    g.part = dgain ? (double *)ws : nullptr;
    g.lanes = p.lanes;
    g.rpb = p.rpb;
    g.span = p.span;
    nr_launch<true>(ctx, g, p.blocks, d->interleaved != 0);
    RNN_LAUNCHED(ctx);
    if (dgain) {
        const size_t len = 2 * (size_t)d->dh;
        gain_reduce_kernel<<<(unsigned)rnn_div_up(len, 4), 256, 0, ctx->stream>>>(p.blocks, (int)len,
                                                                                  g.part, dgain);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

int rnn_head_gate_workspace(size_t rows, size_t h, size_t d, size_t *bytes) {
    const int rc = gate_check(nullptr, rows, h, d, h * d, 0, 1.0f);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    *bytes = rows ? gate_plan(rows, h, d).parts * h * d * sizeof(double) : 0;
    return RNN_OK;
}

int rnn_head_gate_forward(rnn_ctx *ctx, size_t rows, size_t h, size_t d, float eps, const float *x,
                          const float *z, size_t zstride, size_t zoff, const float *gain, float *y) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    const int rc = gate_check(ctx, rows, h, d, zstride, zoff, eps);
    if (rc) return rc;
    if (!rows) return RNN_OK;
    if (!x || !z || !y) return rnn_fail(ctx, RNN_E_NULL, "head_gate: null operand");
    const RnnRows ins[] = {rnn_block(y == x ? nullptr : x, rows * h * d),
                           {z + zoff, rows, zstride, h * d},
                           rnn_block(gain, h * d)};
    const RnnRows outs[] = {rnn_block(y, rows * h * d)};
    if (rnn_any_overlap(outs, ins))
        return rnn_fail(ctx, RNN_E_INVALID, "head_gate: y over another operand");
    RNN_ON_DEVICE(ctx);
    const GatePlan p = gate_plan(rows, h, d);
    GateArgs g = {x, z + zoff, gain, nullptr, y, nullptr, nullptr, (long long)zstride, 0, (long long)rows,
                  (int)h, (int)d, p.lanes, (double)eps};
    const unsigned grid = (unsigned)(p.splits * h);
    head_gate_kernel<false><<<grid, 256, 0, ctx->stream>>>(g);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_head_gate_backward(rnn_ctx *ctx, size_t rows, size_t h, size_t d, float eps, const float *x,
                           const float *z, size_t zstride, size_t zoff, const float *gain,
                           const float *dy, void *ws, size_t ws_bytes, float *dx, float *dz,
                           size_t dzstride, size_t dzoff, float *dgain) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = gate_check(ctx, rows, h, d, zstride, zoff, eps);
    if (!rc) rc = gate_check(ctx, rows, h, d, dzstride, dzoff, eps);
    if (rc) return rc;
    if (!rows) return RNN_OK;
    if (!x || !z || !dy || !dx || !dz) return rnn_fail(ctx, RNN_E_NULL, "head_gate: null operand");
    if (!gain && dgain) return rnn_fail(ctx, RNN_E_NULL, "head_gate: dgain without gain");
    if (dz == z && (dzstride != zstride || dzoff != zoff))
        return rnn_fail(ctx, RNN_E_INVALID, "head_gate: in place with two layouts");
    const bool over_z = dz + dzoff == z + zoff && dzstride == zstride;
    // what dx or dz may take the place of is met by the other one as dx or dz
    const RnnRows ins[] = {rnn_block(dx == x ? nullptr : x, rows * h * d),
                           rnn_block(dx == dy ? nullptr : dy, rows * h * d),
                           {over_z ? nullptr : z + zoff, rows, zstride, h * d},
                           rnn_block(gain, h * d),
                           rnn_block(dgain, h * d)};
    const RnnRows outs[] = {rnn_block(dx, rows * h * d), {dz + dzoff, rows, dzstride, h * d}};
    if (rnn_any_overlap(outs, ins))
        return rnn_fail(ctx, RNN_E_INVALID, "head_gate: a gradient over another operand");
    const GatePlan p = gate_plan(rows, h, d);
    rc = ws_checked(ctx, "head_gate", dgain ? p.parts * h * d * sizeof(double) : 0, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    const long long w = (long long)(h * d);
    GateArgs g = {x, z + zoff, gain, dy, dx, dz + dzoff, dgain ? (double *)ws : nullptr,
                  (long long)zstride, (long long)dzstride, (long long)rows, (int)h, (int)d, p.lanes,
                  (double)eps};
    const unsigned grid = (unsigned)(p.parts * h);
    head_gate_kernel<true><<<grid, 256, 0, ctx->stream>>>(g);
    RNN_LAUNCHED(ctx);
    if (dgain) {
        gain_reduce_kernel<<<(unsigned)rnn_div_up((size_t)w, 4), 256, 0, ctx->stream>>>((int)p.parts, (int)w,
                                                                                        g.part, dgain);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

}  // extern "C"
