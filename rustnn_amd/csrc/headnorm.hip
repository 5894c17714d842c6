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
// that a wave reads whole lines.  Squares, dots and what they are multiplied
// with are in 64 bits: a square passes a float's range from 2^64 on and falls
// below it from 2^-75, and 64-bit additions run at the rate of 32-bit ones here.
#include "rotary_angle.h"

#include <algorithm>

namespace {

constexpr int MAX_HEAD = 256;      // channels of a head with rotary positions
constexpr int MAX_GATE = 512;      // channels of a gated head
constexpr int MAX_BLOCKS = 8192;   // of a forward: 32 a CU
constexpr int MAX_PARTS = 1024;    // of a backward, each leaving its part of dgain
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
    int lanes, rpb;
    double eps;
    double w[MAX_PAIRS];  // quarter turns per unit of position of every pair
};

// A lane's channels: element e < 4 is the first channel of its pair e, e >= 4
// the second one of pair e - 4; lanes past the pairs hold eight channels that
// do not turn.  -1: no such channel.
template <bool INTER>
__device__ __forceinline__ int nr_channel(const NrArgs &g, int u, int e) {
    const int R = g.npairs, T = (R + 3) / 4;
    const int p = INTER ? (e < 4 ? 2 * e : 2 * e - 7) : e;
    if (u < T) {
        if (4 * u + (e & 3) >= R) return -1;
        return INTER ? 8 * u + p : e < 4 ? 4 * u + e : R + 4 * u + e - 4;
    }
    const int c = 2 * R + 8 * (u - T) + p;
    return c < g.dh ? c : -1;
}

// VEC: 16-byte accesses; whole groups of four pairs and of four other
// channels, rows and heads aligned.
template <bool VEC, bool INTER>
__device__ __forceinline__ void nr_load(const NrArgs &g, const float *p, int u, float (&v)[8]) {
    if constexpr (VEC) {
        const int R = g.npairs, T = R / 4;
        const int ca = u < T ? (INTER ? 8 * u : 4 * u) : 2 * R + 8 * (u - T);
        const int cb = u < T && !INTER ? R + 4 * u : ca + 4;
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 a = ca < g.dh ? *(const float4 *)(p + ca) : z;
        const float4 b = cb < g.dh ? *(const float4 *)(p + cb) : z;
        if constexpr (INTER) {
            v[0] = a.x, v[4] = a.y, v[1] = a.z, v[5] = a.w;
            v[2] = b.x, v[6] = b.y, v[3] = b.z, v[7] = b.w;
        } else {
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = nr_channel<INTER>(g, u, e);
            v[e] = c >= 0 ? p[c] : 0.f;
        }
    }
}

template <bool VEC, bool INTER>
__device__ __forceinline__ void nr_store(const NrArgs &g, float *p, int u, const float (&v)[8]) {
    if constexpr (VEC) {
        const int R = g.npairs, T = R / 4;
        const int ca = u < T ? (INTER ? 8 * u : 4 * u) : 2 * R + 8 * (u - T);
        const int cb = u < T && !INTER ? R + 4 * u : ca + 4;
        float4 a, b;
        if constexpr (INTER) {
            a = make_float4(v[0], v[4], v[1], v[5]);
            b = make_float4(v[2], v[6], v[3], v[7]);
        } else {
            a = make_float4(v[0], v[1], v[2], v[3]);
            b = make_float4(v[4], v[5], v[6], v[7]);
        }
        if (ca < g.dh) *(float4 *)(p + ca) = a;
        if (cb < g.dh) *(float4 *)(p + cb) = b;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = nr_channel<INTER>(g, u, e);
            if (c >= 0) p[c] = v[e];
        }
    }
}

// A block takes `rpb` rows at a time: their sines and cosines into LDS, formed
// once for all heads, then every head.
template <bool VEC, bool INTER, bool BACK>
__global__ __launch_bounds__(256) void norm_rotary_kernel(NrArgs g) {
    __shared__ __attribute__((aligned(16))) float2 tab[TABLE];
    const int L = g.lanes, R = g.npairs, T = (R + 3) / 4;
    const int ng = 256 / L, grp = threadIdx.x / L, u = threadIdx.x & (L - 1);
    const bool turned = u < T;
    float gain[2][8];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = nr_channel<INTER>(g, u, e);
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
    for (long long row0 = (long long)blockIdx.x * g.rpb; row0 < g.rows;
         row0 += (long long)gridDim.x * g.rpb) {
        const int nrow = (int)min((long long)g.rpb, g.rows - row0);
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
            const int hn = k ? g.h - g.hq : g.hq, items = nrow * hn;
            for (int i0 = 0; i0 < items; i0 += ng) {
                const bool live = i0 + grp < items;
                const int it = live ? i0 + grp : items - 1;
                const int lr = it / hn, hd = it - lr * hn + k * g.hq;
                const long long r = row0 + lr;
                float v[8], d[8];
                nr_load<VEC, INTER>(g, g.x + r * g.xstride + hd * g.dh, u, v);
                if constexpr (BACK) nr_load<VEC, INTER>(g, g.dy + r * g.dystride + hd * g.dh, u, d);
                double s = 0.0;
#pragma unroll
                for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
                const double rn = 1.0 / sqrt(group_sum(s, L) * inv + g.eps);
                float o[8];
                if constexpr (!BACK) {
#pragma unroll
                    for (int e = 0; e < 8; e++) d[e] = (float)(v[e] * rn) * gain[k][e];
                }
                if (turned) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const float2 w = tab[lr * R + min(4 * u + q, R - 1)];
                        o[q] = __builtin_fmaf(d[q], w.x, -(d[q + 4] * w.y));
                        o[q + 4] = __builtin_fmaf(d[q + 4], w.x, d[q] * w.y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = d[e];
                }
                if constexpr (BACK) {
                    double m = 0.0;
                    double hat[8], t[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        hat[e] = v[e] * rn;
                        if (live) acc[k][e] = fma((double)o[e], hat[e], acc[k][e]);
                        t[e] = (double)o[e] * gain[k][e];
                        m = fma(t[e], hat[e], m);
                    }
                    m = group_sum(m, L) * inv;
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = (float)(fma(-hat[e], m, t[e]) * rn);
                }
                if (live) nr_store<VEC, INTER>(g, g.y + r * g.ystride + hd * g.dh, u, o);
            }
        }
    }
    if constexpr (BACK) {
        if (!g.part) return;
#pragma unroll
        for (int k = 0; k < 2; k++)
            block_sum8(acc[k], L, [&](int lane, int e, double s) {
                const int c = nr_channel<INTER>(g, lane, e);
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

template <bool VEC>
__device__ __forceinline__ void gate_load(const float *p, int c, int d, float (&v)[8]) {
    if constexpr (VEC) {
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        *(float4 *)v = c < d ? *(const float4 *)(p + c) : z;
        *(float4 *)(v + 4) = c + 4 < d ? *(const float4 *)(p + c + 4) : z;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = c + e < d ? p[c + e] : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void gate_store(float *p, int c, int d, const float (&v)[8]) {
    if constexpr (VEC) {
        if (c < d) *(float4 *)(p + c) = *(const float4 *)v;
        if (c + 4 < d) *(float4 *)(p + c + 4) = *(const float4 *)(v + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c + e < d) p[c + e] = v[e];
    }
}

// Block b: head b % h, rows (b / h) * groups + group, and every splits * groups
// further, so that dgain's sums stay with one head's channels.
template <bool VEC, bool BACK>
__global__ __launch_bounds__(256) void head_gate_kernel(GateArgs g) {
    const int L = g.lanes, ng = 256 / L, grp = threadIdx.x / L, u = threadIdx.x & (L - 1);
    const int head = blockIdx.x % g.h, split = blockIdx.x / g.h, splits = gridDim.x / g.h;
    const int c = 8 * u, col = head * g.d;
    const long long w = (long long)g.h * g.d;
    float gain[8];
#pragma unroll
    for (int e = 0; e < 8; e++) gain[e] = c + e >= g.d ? 0.f : g.gain ? g.gain[col + c + e] : 1.f;
    double acc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.0;
    const double inv = 1.0 / g.d;
    for (long long r0 = (long long)split * ng; r0 < g.rows; r0 += (long long)splits * ng) {
        const bool live = r0 + grp < g.rows;
        const long long r = live ? r0 + grp : g.rows - 1;
        float v[8], z[8], d[8];
        gate_load<VEC>(g.x + r * w + col, c, g.d, v);
        gate_load<VEC>(g.z + r * g.zstride + col, c, g.d, z);
        if constexpr (BACK) gate_load<VEC>(g.dy + r * w + col, c, g.d, d);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
        const double rn = 1.0 / sqrt(group_sum(s, L) * inv + g.eps);
        float o[8];
        if constexpr (!BACK) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                o[e] = (float)(v[e] * rn) * gain[e] * (z[e] / (1.f + expf(-z[e])));
        } else {
            float dz[8];
            double hat[8], t[8], m = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float sig = 1.f / (1.f + expf(-z[e]));
                hat[e] = v[e] * rn;
                dz[e] = d[e] * ((float)hat[e] * gain[e]) * (sig * (1.f + z[e] * (1.f - sig)));
                const double du = (double)d[e] * (z[e] * sig);
                if (live) acc[e] = fma(du, hat[e], acc[e]);
                t[e] = du * gain[e];
                m = fma(t[e], hat[e], m);
            }
            m = group_sum(m, L) * inv;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = (float)(fma(-hat[e], m, t[e]) * rn);
            if (live) gate_store<VEC>(g.dz + r * g.dzstride + col, c, g.d, dz);
        }
        if (live) gate_store<VEC>(g.y + r * w + col, c, g.d, o);
    }
    if constexpr (BACK) {
        if (!g.part) return;
        block_sum8(acc, L, [&](int lane, int e, double s) {
            if (8 * lane + e < g.d) g.part[split * w + col + 8 * lane + e] = s;
        });
    }
}

__global__ __launch_bounds__(256) void gain_reduce_kernel(int nrow, size_t len, const double *part,
                                                          float *out) {
    rnn_colsum_red_block(nrow, len, len, part, out, out, blockIdx.x);
}

// ---------------------------------------------------------------- plans
int pow2_lanes(int units) {
    int L = 1;
    while (L < units) L *= 2;
    return L;
}

struct NrPlan {
    int lanes, rpb, blocks, parts;  // blocks of a forward, of a backward
};
NrPlan nr_plan(const rnn_rotary_desc *d, size_t rows) {
    NrPlan p;
    const int R = (int)(d->p0 + d->p1 + d->p2);
    p.lanes = pow2_lanes((R + 3) / 4 + ((int)d->dh - 2 * R + 7) / 8);
    // rows enough for a sine and cosine a thread, fewer where that would leave
    // CUs idle
    const int most = R ? std::min(32, (int)rnn_div_up(256, R)) : 8;
    p.rpb = (int)std::max<size_t>(1, std::min<size_t>(most, rows / 512));
    const size_t b = rnn_div_up(rows, p.rpb);
    p.blocks = (int)std::min<size_t>(b, MAX_BLOCKS);
    p.parts = (int)std::min<size_t>(b, MAX_PARTS);
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

bool aligned16(const float *p, long long stride) {
    return ((uintptr_t)p & 15) == 0 && stride % 4 == 0;
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
void nr_launch(rnn_ctx *ctx, const NrArgs &g, int blocks, bool vec, bool inter) {
    if (vec && inter)
        norm_rotary_kernel<true, true, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
    else if (vec)
        norm_rotary_kernel<true, false, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
    else if (inter)
        norm_rotary_kernel<false, true, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
    else
        norm_rotary_kernel<false, false, BACK><<<blocks, 256, 0, ctx->stream>>>(g);
}

struct GatePlan {
    int lanes;
    size_t splits, parts;  // of a forward, of a backward
};
GatePlan gate_plan(size_t rows, size_t h, size_t d) {
    GatePlan p;
    p.lanes = pow2_lanes((int)rnn_div_up(d, 8));
    const size_t all = rnn_div_up(rows, 256 / p.lanes);
    p.splits = std::min(all, std::max<size_t>(1, MAX_BLOCKS / h));
    p.parts = std::min(all, std::max<size_t>(1, MAX_PARTS / h));
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
    *bytes = rows ? (size_t)nr_plan(d, rows).parts * 2 * d->dh * sizeof(double) : 0;
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
    if (x == y && (d->xstride != d->ystride || d->xoff != d->yoff))
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: in place with two layouts");
    RNN_ON_DEVICE(ctx);
    NrArgs g;
    nr_fill(g, d, hq, eps, n, t, x, gain, pos, y);
    const NrPlan p = nr_plan(d, n * t);
    g.lanes = p.lanes;
    g.rpb = p.rpb;
    const bool vec = g.npairs % 4 == 0 && g.dh % 4 == 0 && aligned16(g.x, g.xstride) &&
                     aligned16(g.y, g.ystride);
    nr_launch<false>(ctx, g, p.blocks, vec, d->interleaved != 0);
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
    if (dx == x) return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: dx is x");
    if (dx == dy && (d->ystride != dystride || d->yoff != dyoff))
        return rnn_fail(ctx, RNN_E_INVALID, "norm_rotary: in place with two layouts");
    const NrPlan p = nr_plan(d, n * t);
    rc = ws_checked(ctx, "norm_rotary", dgain ? (size_t)p.parts * 2 * d->dh * sizeof(double) : 0, ws,
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
    const bool vec = g.npairs % 4 == 0 && g.dh % 4 == 0 && aligned16(g.x, g.xstride) &&
                     aligned16(g.y, g.ystride) && aligned16(g.dy, g.dystride);
    nr_launch<true>(ctx, g, p.parts, vec, d->interleaved != 0);
    RNN_LAUNCHED(ctx);
    if (dgain) {
        const size_t len = 2 * (size_t)d->dh;
        gain_reduce_kernel<<<(unsigned)rnn_div_up(len, 16), 256, 0, ctx->stream>>>(p.parts, len, g.part,
                                                                                   dgain);
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
    RNN_ON_DEVICE(ctx);
    const GatePlan p = gate_plan(rows, h, d);
    const long long w = (long long)(h * d);
    GateArgs g = {x, z + zoff, gain, nullptr, y, nullptr, nullptr, (long long)zstride, 0, (long long)rows,
                  (int)h, (int)d, p.lanes, (double)eps};
    const bool vec = d % 4 == 0 && aligned16(x, w) && aligned16(g.z, g.zstride) && aligned16(y, w);
    const unsigned grid = (unsigned)(p.splits * h);
    if (vec)
        head_gate_kernel<true, false><<<grid, 256, 0, ctx->stream>>>(g);
    else
        head_gate_kernel<false, false><<<grid, 256, 0, ctx->stream>>>(g);
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
    const GatePlan p = gate_plan(rows, h, d);
    rc = ws_checked(ctx, "head_gate", dgain ? p.parts * h * d * sizeof(double) : 0, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    const long long w = (long long)(h * d);
    GateArgs g = {x, z + zoff, gain, dy, dx, dz + dzoff, dgain ? (double *)ws : nullptr,
                  (long long)zstride, (long long)dzstride, (long long)rows, (int)h, (int)d, p.lanes,
                  (double)eps};
    const bool vec = d % 4 == 0 && aligned16(x, w) && aligned16(g.z, g.zstride) && aligned16(dy, w) &&
                     aligned16(dx, w) && aligned16(g.dz, g.dzstride);
    const unsigned grid = (unsigned)(p.parts * h);
    if (vec)
        head_gate_kernel<true, true><<<grid, 256, 0, ctx->stream>>>(g);
    else
        head_gate_kernel<false, true><<<grid, 256, 0, ctx->stream>>>(g);
    RNN_LAUNCHED(ctx);
    if (dgain) {
        gain_reduce_kernel<<<(unsigned)rnn_div_up((size_t)w, 16), 256, 0, ctx->stream>>>(
            (int)p.parts, (size_t)w, g.part, dgain);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

}  // extern "C"
