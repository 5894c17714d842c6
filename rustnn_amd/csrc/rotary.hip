// Rotary positions with up to three axes (time, height, width) on the heads
// of a token row (rnn_rotary).  No counterpart in the reference.
//
// Each output carries the rounding of sine and cosine (rotary_angle.h), of one
// product and of one fused multiply-add.
//
// The work is one read and one write of the heads: HBM-bound.  A thread owns
// a group of pairs of one token in up to four heads, so that the 64-bit part
// (about 45 instructions a pair) serves them together; consecutive lanes take
// the groups of a head, then the next head, so that a wave reads whole lines.
#include "rotary_angle.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int HPT = 4;  // heads of a thread: hl, hl + HL, ... (HL = ceil(h / HPT))

struct RotArgs {
    const float *x, *pos;
    float *y;
    long long xstride, ystride;
    int rows, t, h, dh, axes, npairs, hl;
    int p0, p1;  // pairs of the first two axes
    int g1, g2;  // grid sides of the last two axes
    int rpb;     // rows of a block
    int first;   // the launch's first row
    float sign;  // -1: the inverse
    // quarter turns per unit of position of every pair
    double w[MAX_PAIRS];
};

// G pairs a thread (4: 16-byte accesses, R, dh and the strides multiples of 4;
// 1: any layout), channels past 2R copied G at a time.
template <int G, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs g) {
    const int R = g.npairs, turned = R / G, ng = turned + (g.dh - 2 * R) / G;
    const int units = g.hl * ng;
    const int row0 = g.first + (int)blockIdx.x * g.rpb, nrow = min(g.rpb, g.rows - row0);
    for (int e = threadIdx.x; e < nrow * units; e += 256) {
        const int lr = e / units, u = e - lr * units;
        const int hl = u / ng, grp = u - hl * ng;
        const int r = row0 + lr;
        const float *x = g.x + r * g.xstride;
        float *y = g.y + r * g.ystride;
        if (grp >= turned) {
            const int c = 2 * R + (grp - turned) * G;
#pragma unroll
            for (int i = 0; i < HPT; i++) {
                const int hd = hl + i * g.hl;
                if (hd >= g.h) break;
                if constexpr (G == 4)
                    *(float4 *)(y + hd * g.dh + c) = *(const float4 *)(x + hd * g.dh + c);
                else
                    y[hd * g.dh + c] = x[hd * g.dh + c];
            }
            continue;
        }
        const int j0 = grp * G;
        // the first and second channels of the group's pairs in a head: two
        // runs of G, or one of 2G with the two alternating
        const int ca = INTER ? 2 * j0 : j0, cb = INTER ? 2 * j0 + G : j0 + R;
        float va[HPT][G], vb[HPT][G];
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int hd = min(hl + i * g.hl, g.h - 1);
            if constexpr (G == 4) {
                *(float4 *)va[i] = *(const float4 *)(x + hd * g.dh + ca);
                *(float4 *)vb[i] = *(const float4 *)(x + hd * g.dh + cb);
            } else {
                va[i][0] = x[hd * g.dh + ca];
                vb[i][0] = x[hd * g.dh + cb];
            }
        }
        float sn[G], cs[G];
#pragma unroll
        for (int k = 0; k < G; k++) {
            rot_sincos(rot_position(g, r, j0 + k) * g.w[j0 + k], &sn[k], &cs[k]);
            sn[k] *= g.sign;
        }
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int hd = hl + i * g.hl;
            if (hd >= g.h) break;
            float oa[G], ob[G];
#pragma unroll
            for (int k = 0; k < G; k++) {
                if constexpr (INTER && G == 4) {
                    // pair k: element 2k of the run of 8
                    const float a = k < 2 ? va[i][2 * k] : vb[i][2 * k - 4];
                    const float b = k < 2 ? va[i][2 * k + 1] : vb[i][2 * k - 3];
                    float *o = k < 2 ? &oa[2 * k] : &ob[2 * k - 4];
                    o[0] = __builtin_fmaf(a, cs[k], -(b * sn[k]));
                    o[1] = __builtin_fmaf(b, cs[k], a * sn[k]);
                } else {
                    oa[k] = __builtin_fmaf(va[i][k], cs[k], -(vb[i][k] * sn[k]));
                    ob[k] = __builtin_fmaf(vb[i][k], cs[k], va[i][k] * sn[k]);
                }
            }
            if constexpr (G == 4) {
                *(float4 *)(y + hd * g.dh + ca) = *(const float4 *)oa;
                *(float4 *)(y + hd * g.dh + cb) = *(const float4 *)ob;
            } else {
                y[hd * g.dh + ca] = oa[0];
                y[hd * g.dh + cb] = ob[0];
            }
        }
    }
}

}  // namespace

int rnn_rotary_checked(rnn_ctx *ctx, const rnn_rotary_desc *d, size_t n, size_t t, bool have_pos) {
    if (!d) return rnn_fail(ctx, RNN_E_NULL, "rotary: desc is null");
    if (!d->h || !d->dh) return rnn_fail(ctx, RNN_E_INVALID, "rotary: zero heads or channels");
    if (d->axes < 1 || d->axes > 3)
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: %u axes (1 to 3)", d->axes);
    if ((d->axes < 2 && d->p1) || (d->axes < 3 && d->p2))
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: pairs beyond the %u axes", d->axes);
    const uint64_t pairs = (uint64_t)d->p0 + d->p1 + d->p2;
    if (2 * pairs > d->dh)
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: %llu pairs in %u channels",
                        (unsigned long long)pairs, d->dh);
    if (pairs > MAX_PAIRS)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "rotary: more than %d pairs", MAX_PAIRS);
    if (!(d->base > 0.0f) || !std::isfinite(d->base))
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: base %g", (double)d->base);
    const uint64_t width = (uint64_t)d->h * d->dh;
    if (width > (1u << 24)) return rnn_fail(ctx, RNN_E_UNSUPPORTED, "rotary: row too wide");
    if (d->xoff > d->xstride || d->xstride - d->xoff < width || d->yoff > d->ystride ||
        d->ystride - d->yoff < width)
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: %llu channels do not fit a row",
                        (unsigned long long)width);
    if (!have_pos) {
        if (!d->g0 || !d->g1 || !d->g2 || (d->axes < 2 && d->g1 != 1) ||
            (d->axes < 3 && d->g2 != 1))
            return rnn_fail(ctx, RNN_E_INVALID, "rotary: grid %u x %u x %u with %u axes", d->g0,
                            d->g1, d->g2, d->axes);
        const uint64_t plane = (uint64_t)d->g1 * d->g2;
        if (plane > 0x7fffffffu || d->g0 > 0x7fffffffu / plane || (uint64_t)d->g0 * plane != t)
            return rnn_fail(ctx, RNN_E_INVALID, "rotary: %zu tokens on a grid of %u x %u x %u", t,
                            d->g0, d->g1, d->g2);
    }
    if (t > 0x7fffffffu || (t && n > 0x7fffffffu / t))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "rotary: too many rows");
    return RNN_OK;
}

extern "C" {

int rnn_rotary_check(const rnn_rotary_desc *d, size_t n, size_t t, int have_pos) {
    return rnn_rotary_checked(nullptr, d, n, t, have_pos != 0);
}

int rnn_rotary(rnn_ctx *ctx, const rnn_rotary_desc *d, size_t n, size_t t, const float *x,
               const float *pos, float *y, int inverse) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    const int rc = rnn_rotary_checked(ctx, d, n, t, pos != nullptr);
    if (rc) return rc;
    const size_t rows = n * t;
    if (!rows) return RNN_OK;
    if (!x || !y) return rnn_fail(ctx, RNN_E_NULL, "rotary: null operand");
    if (x == y && (d->xstride != d->ystride || d->xoff != d->yoff))
        return rnn_fail(ctx, RNN_E_INVALID, "rotary: in place with two layouts");
    RNN_ON_DEVICE(ctx);
    RotArgs g;
    g.x = x + d->xoff;
    g.y = y + d->yoff;
    g.pos = pos;
    g.xstride = (long long)d->xstride;
    g.ystride = (long long)d->ystride;
    g.rows = (int)rows;
    g.t = (int)t;
    g.h = (int)d->h;
    g.dh = (int)d->dh;
    g.axes = (int)d->axes;
    g.npairs = (int)(d->p0 + d->p1 + d->p2);
    g.hl = (g.h + HPT - 1) / HPT;
    g.p0 = (int)d->p0;
    g.p1 = (int)d->p1;
    g.g1 = (int)d->g1;
    g.g2 = (int)d->g2;
    g.sign = inverse ? -1.0f : 1.0f;
    rot_frequencies(d, g.w);
    // 16-byte accesses: whole groups of four pairs and of four copied
    // channels, every head's start aligned
    auto al = [](const float *p, long long stride) {
        return ((uintptr_t)p & 15) == 0 && stride % 4 == 0;
    };
    const bool vec = g.npairs % 4 == 0 && g.dh % 4 == 0 && al(g.x, g.xstride) && al(g.y, g.ystride);
    const int G = vec ? 4 : 1;
    const int units = g.hl * (g.npairs / G + (g.dh - 2 * g.npairs) / G);
    g.rpb = std::max(1, 256 / units);
    // launches of at most 2^23 blocks, 2^31 threads (a grid holds below 2^32)
    const size_t most = ((size_t)1 << 23) * (size_t)g.rpb;
    for (size_t r = 0; r < rows; r += most) {
        g.first = (int)r;
        const unsigned grid = (unsigned)rnn_div_up(std::min(rows - r, most), (size_t)g.rpb);
        if (vec && d->interleaved)
            rotary_kernel<4, true><<<grid, 256, 0, ctx->stream>>>(g);
        else if (vec)
            rotary_kernel<4, false><<<grid, 256, 0, ctx->stream>>>(g);
        else if (d->interleaved)
            rotary_kernel<1, true><<<grid, 256, 0, ctx->stream>>>(g);
        else
            rotary_kernel<1, false><<<grid, 256, 0, ctx->stream>>>(g);
    }
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

}  // extern "C"
