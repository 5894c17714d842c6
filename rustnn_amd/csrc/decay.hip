// Linear attention with a decay for each head (rnn_decay_attn_*).  No
// counterpart in the reference.
//
// Forward and gradients are one form, in which a, b and c change their parts:
//   lin(a, b, c)_i = sum_(l <= i) gamma^(i-l) (a_i . b_l) c_l
//   y = scale lin(q, k, v)         dq = scale lin(dy, v, k)
//   dk = scale lin'(v, dy, q)      dv = scale lin'(k, q, dy)
// (lin': from the other end.)  With a state T = sum gamma^(..) b^T c of da x dc
// carried over the tokens, lin_i = a_i T.  The forward's direction holds S (dq: its
// transpose), the other one R, the gradient of the state before a token, which
// begins as the gradient of the last state and ends as the first one's:
//   S_i = gamma S_(i-1) + k_i^T v_i,   R^_i = gamma (R^_(i+1) + scale q_i^T dy_i)
// The rates' gradient is g dL/dg, g = -exp(rate) = log gamma: with Z = dS/dg,
// Z_i = gamma (Z_(i-1) + S_(i-1)), dL/dg = scale sum q_i . (Z^T-weighted sum of k),
// that is, dq's form with each term times i - l, dotted with q; and <Z_last, R^>.
#include "rnn_internal.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MAX_D = 128;

struct DecayJob {
    const float *a, *b, *c;
    float *y;
    const float *s0;    // [n][h] states before the first token; null: 0
    float *s1;          // states after the last; null: not wanted
    const float *dot;   // the rates' gradient: what the weighted sums are dotted with
    const float *s1g;   // and the gradient of the last state
    long long as, bs, cs, ys, ds;  // row strides
    int da, dc;         // channels
    int ga, gb, gc, gy; // query heads that share a head of the operand
    int si, sj;         // a state's strides along da and dc
    float sa, sb;       // factors of a and of b
    int rev, acc;       // from the last token; y accumulates
};

struct DecayArgs {
    DecayJob job[3];
    const float *rate;
    const uint32_t *lens;
    double *part;  // [n][h] parts of dL/dg
    int n, t, h, reverse;
};

// log gamma of a head: at most 0, and finite, so that its multiple by 0 is 0.
__device__ __forceinline__ double log_gamma(float rate) {
    const double g = -exp((double)rate);
    return g < -1e30 ? -1e30 : g;
}

// s gamma, gamma in two parts.
__device__ __forceinline__ float decayed(float s, float gam, float rest) {
    return __builtin_fmaf(s, gam, s * rest);
}

// Token by token: a block holds a head's state, wave w rows 32 w .. 32 w + 31,
// a lane columns lane and lane + 64.
template <bool SLOPE>
__global__ __launch_bounds__(256) void decay_tokens_kernel(DecayArgs g) {
    __shared__ float red[2][4][MAX_D];
    __shared__ double dred[4];
    const DecayJob &q = g.job[blockIdx.y];
    const bool slope = SLOPE && q.dot;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int heads = g.h / q.gy;
    const int b = blockIdx.x / heads, ho = blockIdx.x % heads;
    const int len = g.lens ? (int)min(g.lens[b], (uint32_t)g.t) : g.t;
    for (int r = 0; r < q.gy; r++) {
        const int hd = ho * q.gy + r;
        const bool back = (hd >= g.h - g.reverse) != (q.rev != 0);
        // gamma in two floats: one rounded alone would be off by its last bit to
        // the power of the tokens
        const double g64 = exp(log_gamma(g.rate[hd]));
        const float gam = (float)g64, rest = (float)(g64 - (double)gam);
        const long long st = ((long long)b * g.h + hd) * q.da * q.dc;
        float s[32][2], z[32][2];
#pragma unroll
        for (int i = 0; i < 32; i++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int ia = 32 * wave + i, jc = lane + 64 * k;
                s[i][k] = q.s0 && ia < q.da && jc < q.dc ? q.s0[st + ia * q.si + jc * q.sj] : 0.f;
                z[i][k] = 0.f;
            }
        double dg = 0.0;
        for (int i = 0; i < g.t; i++) {
            if (i >= len) {
                if (!q.acc && r == 0 && wave < 2 && threadIdx.x < q.dc)
                    q.y[((long long)b * g.t + i) * q.ys + (hd / q.gy) * q.dc + threadIdx.x] = 0.f;
                continue;
            }
            const long long row = (long long)b * g.t + (back ? len - 1 - i : i);
            const float *a = q.a + row * q.as + (hd / q.ga) * q.da;
            const float *bb = q.b + row * q.bs + (hd / q.gb) * q.da;
            const float *c = q.c + row * q.cs + (hd / q.gc) * q.dc;
            float cv[2], o[2] = {0.f, 0.f}, oz[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 2; k++) cv[k] = lane + 64 * k < q.dc ? c[lane + 64 * k] : 0.f;
#pragma unroll
            for (int e = 0; e < 32; e++) {
                const int ia = 32 * wave + e;
                const float av = ia < q.da ? a[ia] : 0.f, bv = ia < q.da ? q.sb * bb[ia] : 0.f;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    if (SLOPE) z[e][k] = decayed(z[e][k] + s[e][k], gam, rest);
                    const float old = q.rev ? s[e][k] : decayed(s[e][k], gam, rest);
                    s[e][k] = __builtin_fmaf(bv, cv[k], old);
                    o[k] = __builtin_fmaf(av, s[e][k], o[k]);
                    if (SLOPE) oz[k] = __builtin_fmaf(av, z[e][k], oz[k]);
                    if (q.rev) s[e][k] = decayed(s[e][k], gam, rest);
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; k++) {
                red[0][wave][lane + 64 * k] = o[k];
                if (SLOPE) red[1][wave][lane + 64 * k] = oz[k];
            }
            __syncthreads();
            const int jc = threadIdx.x;
            if (jc < q.dc) {
                float v = 0.f, vz = 0.f;
                for (int w = 0; w < 4; w++) {
                    v += red[0][w][jc];
                    if (SLOPE) vz += red[1][w][jc];
                }
                float *y = q.y + row * q.ys + (hd / q.gy) * q.dc + jc;
                *y = (q.acc || r > 0 ? *y : 0.f) + q.sa * v;
                if (slope) dg += (double)(q.sa * vz) * q.dot[row * q.ds + hd * q.dc + jc];
            }
        }
#pragma unroll
        for (int i = 0; i < 32; i++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int ia = 32 * wave + i, jc = lane + 64 * k;
                if (ia >= q.da || jc >= q.dc) continue;
                if (q.s1) q.s1[st + ia * q.si + jc * q.sj] = s[i][k];
                if (slope && q.s1g) dg += (double)z[i][k] * q.s1g[st + ia * q.si + jc * q.sj];
            }
        if (slope) {
            dg = rnn_wave_sum_d(dg);
            __syncthreads();
            if (lane == 0) dred[wave] = dg;
            __syncthreads();
            if (threadIdx.x == 0)
                g.part[(long long)b * g.h + hd] = dred[0] + dred[1] + dred[2] + dred[3];
        }
    }
}

// drate[j] += g sum of the head's parts, in a fixed order.
__global__ __launch_bounds__(256) void decay_rate_kernel(const double *part, int rows, int h,
                                                         const float *rate, float *drate) {
    __shared__ double red[4];
    const int j = blockIdx.x;
    double s = 0.0;
    for (int i = threadIdx.x; i < rows; i += 256) s += part[(long long)i * h + j];
    s = rnn_wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        drate[j] += (float)(log_gamma(rate[j]) * (red[0] + red[1] + red[2] + red[3]));
}

struct DecayWs {
    size_t part = 0, bytes = 0;
};
DecayWs plan_ws(const rnn_decay_attn_desc *d, size_t n, size_t t, bool backward) {
    DecayWs w;
    WsCarve c;
    if (backward) w.part = c.take(n * d->h * sizeof(double));
    w.bytes = c.off;
    return w;
}

int decay_check(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t) {
    if (!d) return rnn_fail(ctx, RNN_E_NULL, "decay_attn: desc is null");
    if (!d->h || !d->hkv || !d->dk || !d->dv)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: zero heads or channels");
    if (d->h % d->hkv)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: %u heads on %u key heads", d->h, d->hkv);
    if (d->reverse > d->h)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: %u of %u heads reversed", d->reverse, d->h);
    if (!std::isfinite(d->scale))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: scale %g", (double)d->scale);
    if (d->dk > MAX_D || d->dv > MAX_D)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "decay_attn: heads of %u and %u channels (up to %d)",
                        d->dk, d->dv, MAX_D);
    const uint64_t qw = (uint64_t)d->h * d->dk, kw = (uint64_t)d->hkv * d->dk,
                   vw = (uint64_t)d->hkv * d->dv;
    if (d->qstride > (1u << 22) || d->kvstride > (1u << 22))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "decay_attn: row stride above 2^22");
    if (d->qoff > d->qstride || d->qstride - d->qoff < qw || d->koff > d->kvstride ||
        d->kvstride - d->koff < kw || d->voff > d->kvstride || d->kvstride - d->voff < vw)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: heads do not fit a row");
    if (d->koff < d->voff + vw && d->voff < d->koff + kw)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: keys and values overlap");
    const uint64_t lim = 1ull << 31, per = (uint64_t)d->h * std::max<uint64_t>(t, (uint64_t)d->dk * d->dv);
    if (t >= lim || per >= lim || (n && n > (lim - 1) / per))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "decay_attn: too many tokens or states");
    return RNN_OK;
}

int check_ws(rnn_ctx *ctx, const DecayWs &w, const void *ws, size_t bytes) {
    if (!w.bytes) return RNN_OK;
    if (!ws) return rnn_fail(ctx, RNN_E_NULL, "decay_attn: workspace is null");
    if (bytes < w.bytes)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: workspace of %zu bytes, needs %zu", bytes, w.bytes);
    if ((uintptr_t)ws & 255)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: workspace not 256-byte aligned");
    return RNN_OK;
}

// One of the form's operands: where its rows are, and how many query heads share
// one of its heads.
struct Operand {
    const float *p;
    size_t stride;
    int share;
};

DecayJob make_job(const Operand &a, const Operand &b, int da, const Operand &c, int dc, float *y,
                  size_t ys, int gy) {
    DecayJob j = {};
    j.a = a.p, j.b = b.p, j.c = c.p, j.y = y;
    j.as = (long long)a.stride, j.bs = (long long)b.stride, j.cs = (long long)c.stride;
    j.ys = (long long)ys;
    j.da = da, j.dc = dc;
    j.ga = a.share, j.gb = b.share, j.gc = c.share, j.gy = gy;
    j.si = dc, j.sj = 1;
    j.sa = j.sb = 1.f;
    return j;
}

void fill_args(DecayArgs &g, const rnn_decay_attn_desc *d, size_t n, size_t t, const float *rate,
               const uint32_t *lens) {
    g.rate = rate;
    g.lens = lens;
    g.part = nullptr;
    g.n = (int)n;
    g.t = (int)t;
    g.h = (int)d->h;
    g.reverse = (int)d->reverse;
}

}  // namespace

extern "C" {

int rnn_decay_attn_workspace(const rnn_decay_attn_desc *d, size_t n, size_t t, int backward,
                             size_t *bytes) {
    const int rc = decay_check(nullptr, d, n, t);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    *bytes = plan_ws(d, n, t, backward != 0).bytes;
    return RNN_OK;
}

int rnn_decay_attn_forward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                           const float *q, const float *kv, const float *rate, const uint32_t *lens,
                           const float *state_in, void *ws, size_t ws_bytes, float *y,
                           float *state_out) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = decay_check(ctx, d, n, t);
    if (rc) return rc;
    if (!n || (!t && !state_out)) return RNN_OK;
    if ((t && (!q || !kv || !y)) || !rate) return rnn_fail(ctx, RNN_E_NULL, "decay_attn_forward: null operand");
    const DecayWs w = plan_ws(d, n, t, false);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    DecayArgs g;
    fill_args(g, d, n, t, rate, lens);
    const int grp = (int)(d->h / d->hkv);
    const Operand Q = {q + d->qoff, d->qstride, 1}, K = {kv + d->koff, d->kvstride, grp},
                  V = {kv + d->voff, d->kvstride, grp};
    DecayJob &j = g.job[0];
    j = make_job(Q, K, (int)d->dk, V, (int)d->dv, y, (size_t)d->h * d->dv, 1);
    j.s0 = state_in;
    j.s1 = state_out;
    j.sa = d->scale;
    decay_tokens_kernel<false><<<dim3((unsigned)(n * d->h), 1), 256, 0, ctx->stream>>>(g);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_decay_attn_backward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                            const float *q, const float *kv, const float *rate, const uint32_t *lens,
                            const float *state_in, const float *dy, const float *dstate_out, void *ws,
                            size_t ws_bytes, float *dq, float *dkv, float *drate, float *dstate_in,
                            uint32_t flags) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = decay_check(ctx, d, n, t);
    if (rc) return rc;
    if (flags & ~(uint32_t)(RNN_ATTN_SET_DQ | RNN_ATTN_SET_DKV))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn_backward: unknown flags 0x%x", flags);
    if (!n || (!t && !dstate_in)) return RNN_OK;
    if ((t && (!q || !kv || !dy || !dq || !dkv)) || !rate)
        return rnn_fail(ctx, RNN_E_NULL, "decay_attn_backward: null operand");
    if (dstate_in && (dstate_in == dstate_out || dstate_in == state_in))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn_backward: dstate_in is an operand");
    const DecayWs w = plan_ws(d, n, t, true);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    DecayArgs g;
    fill_args(g, d, n, t, rate, lens);
    const int grp = (int)(d->h / d->hkv), dk = (int)d->dk, dv = (int)d->dv;
    const Operand Q = {q + d->qoff, d->qstride, 1}, K = {kv + d->koff, d->kvstride, grp},
                  V = {kv + d->voff, d->kvstride, grp}, O = {dy, (size_t)d->h * d->dv, 1};
    g.part = (double *)((char *)ws + w.part);
    DecayJob &jq = g.job[0], &jk = g.job[1], &jv = g.job[2];
    jq = make_job(O, V, dv, K, dk, dq + d->qoff, d->qstride, 1);
    jq.si = 1, jq.sj = dv;
    jq.s0 = state_in;
    jq.sa = d->scale;
    jq.acc = !(flags & RNN_ATTN_SET_DQ);
    if (drate) {
        jq.dot = Q.p;
        jq.ds = (long long)d->qstride;
        jq.s1g = dstate_out;
    }
    jk = make_job(V, O, dv, Q, dk, dkv + d->koff, d->kvstride, grp);
    jk.si = 1, jk.sj = dv;
    jv = make_job(K, Q, dk, O, dv, dkv + d->voff, d->kvstride, grp);
    jk.s0 = jv.s0 = dstate_out;
    jk.sb = jv.sb = d->scale;
    jk.rev = jv.rev = 1;
    jk.acc = jv.acc = !(flags & RNN_ATTN_SET_DKV);
    jv.s1 = dstate_in;
    // one launch a job: of shared heads, dk and dv have fewer blocks
    for (int k = 0; k < 3; k++) {
        DecayArgs one = g;
        one.job[0] = g.job[k];
        const unsigned blocks = (unsigned)(n * (k ? d->hkv : d->h));
        if (k == 0 && drate)
            decay_tokens_kernel<true><<<dim3(blocks, 1), 256, 0, ctx->stream>>>(one);
        else
            decay_tokens_kernel<false><<<dim3(blocks, 1), 256, 0, ctx->stream>>>(one);
        RNN_LAUNCHED(ctx);
    }
    if (drate) {
        decay_rate_kernel<<<(unsigned)d->h, 256, 0, ctx->stream>>>(g.part, (int)n, (int)d->h, rate, drate);
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

}  // extern "C"
