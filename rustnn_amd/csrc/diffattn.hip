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
    double *part; // partials of dgain and dlambda, [blocks][2 dh + h]
    long long qstride, kvstride;
    int n, h, hkv, dh, tq, tk, koff, voff, lam_heads, diag, causal, group;
    int acc_q, acc_kv, rpb;
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

// One wave per (image, query, head).
__global__ __launch_bounds__(256) void diff_fwd_row_kernel(DiffArgs g) {
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
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    const int last = i < see.nq ? (g.causal ? min(see.nk, i + see.shift + 1) : see.nk) : 0;
    for (int j0 = 0; j0 < last; j0 += 64) {
        const int j = j0 + lane;
        const bool in = see(i, j);
        const float *kr = k0 + (long long)min(j, see.nk - 1) * g.kvstride;
        float p[2];
        for (int mp = 0; mp < 2; mp++) {
            float s = 0.f;
            for (int c = 0; c < g.dh; c++)
                s = __builtin_fmaf(q[mp * g.dh + c], kr[mp * g.dh + c], s);
            s = in ? s * g.scale : -INFINITY;
            const float mn = fmaxf(m[mp], wave_max(s));
            const float base = mn == -INFINITY ? 0.f : mn;
            const float al = exp2f((m[mp] - base) * LOG2E);
            p[mp] = in ? exp2f((s - base) * LOG2E) : 0.f;
            l[mp] = l[mp] * al + wave_sum(p[mp]);
            o[mp][0] *= al;
            o[mp][1] *= al;
            m[mp] = mn;
        }
        const int cnt = min(64, last - j0);
        for (int t = 0; t < cnt; t++) {
            const float p1 = __shfl(p[0], t, 64), p2 = __shfl(p[1], t, 64);
            const float *vr = v0 + (long long)(j0 + t) * g.kvstride;
            for (int u = 0; u < 2; u++) {
                const int c = lane + 64 * u;
                const float v = c < dv && see(i, j0 + t) ? vr[c] : 0.f;
                o[0][u] = __builtin_fmaf(p1, v, o[0][u]);
                o[1][u] = __builtin_fmaf(p2, v, o[1][u]);
            }
        }
    }
    double e1, e2;
    lambda_terms(g.lam, g.lam_heads, g.dh, hd, &e1, &e2);
    const float lam = (float)(e1 - e2 + (double)g.lam_init);
    float il[2];
    for (int mp = 0; mp < 2; mp++) {
        il[mp] = l[mp] > 0.f ? 1.0f / l[mp] : 0.f;
        if (m[mp] == -INFINITY) m[mp] = 0.f;
    }
    float out[2], ss = 0.f;
    for (int u = 0; u < 2; u++) {
        o[0][u] *= il[0];
        o[1][u] *= il[1];
        out[u] = o[0][u] - lam * o[1][u];
        if (lane + 64 * u < dv) ss += out[u] * out[u];
    }
    const float r = 1.0f / sqrtf(wave_sum(ss) / (float)dv + g.eps);
    for (int u = 0; u < 2; u++) {
        const int c = lane + 64 * u;
        if (c >= dv) continue;
        g.y[w * dv + c] = g.gain ? out[u] * r * (g.gain[c] * (1.0f - g.lam_init)) : out[u];
        if (g.o12) {
            g.o12[(w * 2) * dv + c] = o[0][u];
            g.o12[(w * 2 + 1) * dv + c] = o[1][u];
        }
    }
    if (g.stats && lane == 0) *(float4 *)(g.stats + w * 4) = make_float4(m[0], il[0], m[1], il[1]);
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
        const float p1 = in ? exp2f((s1 * g.scale - st.x) * LOG2E) * st.y : 0.f;
        const float p2 = in ? exp2f((s2 * g.scale - st.z) * LOG2E) * st.w : 0.f;
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
            const float p1 = in ? exp2f((s1 * g.scale - st.x) * LOG2E) * st.y : 0.f;
            const float p2 = in ? exp2f((s2 * g.scale - st.z) * LOG2E) * st.w : 0.f;
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

struct DiffWs {
    size_t dout = 0, dd = 0, part = 0, bytes = 0;
};

DiffWs plan_ws(const rnn_diff_attn_desc *d, size_t n, bool backward) {
    DiffWs w;
    WsCarve cv;
    if (backward) {
        const size_t rows = n * d->tq, heads = rows * d->h;
        w.dout = cv.take(heads * 2 * d->dh * sizeof(float));
        w.dd = cv.take(heads * 2 * sizeof(float));
        const size_t nblk = rows ? rnn_div_up(rows, (size_t)pre_rows(rows)) : 0;
        w.part = cv.take(nblk * (2 * d->dh + d->h) * sizeof(double));
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
    if (n > lim || d->tq > (1u << 26) || d->tk > (1u << 26) || d->kvstride > lim || d->qstride > lim ||
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
    const unsigned grid = (unsigned)rnn_div_up(n * d->tq * d->h, 4);
    diff_fwd_row_kernel<<<grid, 256, 0, ctx->stream>>>(g);
    RNN_LAUNCHED(ctx);
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
