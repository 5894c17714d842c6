// Linear with an activation and a residual (rnn_linear_act_*).  No counterpart
// in the reference, whose MLP is SwiGLU.
#include "rnn_internal.h"

#include <algorithm>
#include <cmath>

namespace {

template <uint32_t ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == RNN_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == RNN_ACT_GELU) return z * (0.5f * (1.0f + erff(z * 0.70710678118654752f)));
    if constexpr (ACT == RNN_ACT_GELU_TANH) {
        const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
        return 0.5f * z * (1.0f + tanhf(u));
    }
    if constexpr (ACT == RNN_ACT_SILU) return z / (1.0f + expf(-z));
    return z;
}

template <uint32_t ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == RNN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == RNN_ACT_GELU)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
               z * (0.39894228040143268f * expf(-0.5f * z * z));
    if constexpr (ACT == RNN_ACT_GELU_TANH) {
        // beyond 30 the slope is 0 or 1 to the last bit, and z^2 stays finite
        z = fminf(fmaxf(z, -30.0f), 30.0f);
        const float zz = z * z;
        const float th = tanhf(0.79788456080286536f * (z + 0.044715f * zz * z));
        return 0.5f * (1.0f + th) +
               0.5f * z * (1.0f - th * th) * (0.79788456080286536f * (1.0f + 0.134145f * zz));
    }
    if constexpr (ACT == RNN_ACT_SILU) {
        const float s = 1.0f / (1.0f + expf(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    return 1.0f;
}

// y = act(z) + res; z, res and y may be one.
template <uint32_t ACT>
__global__ __launch_bounds__(256) void act_fwd_kernel(size_t len, const float *z, const float *res,
                                                      float *y) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < len; i += (size_t)gridDim.x * 256) {
        const float v = act_value<ACT>(z[i]);
        y[i] = res ? v + res[i] : v;
    }
}

// dz = dy act'(z); dz may be z.
template <uint32_t ACT>
__global__ __launch_bounds__(256) void act_bwd_kernel(size_t len, const float *dy, const float *z,
                                                      float *dz) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < len; i += (size_t)gridDim.x * 256)
        dz[i] = dy[i] * act_slope<ACT>(z[i]);
}

template <typename F>
int by_act(uint32_t act, F &&f) {
    switch (act) {
        case RNN_ACT_RELU: return f(std::integral_constant<uint32_t, RNN_ACT_RELU>());
        case RNN_ACT_GELU: return f(std::integral_constant<uint32_t, RNN_ACT_GELU>());
        case RNN_ACT_GELU_TANH: return f(std::integral_constant<uint32_t, RNN_ACT_GELU_TANH>());
        case RNN_ACT_SILU: return f(std::integral_constant<uint32_t, RNN_ACT_SILU>());
        default: return f(std::integral_constant<uint32_t, RNN_ACT_NONE>());
    }
}

unsigned ew_grid(size_t len) { return (unsigned)std::min<size_t>(rnn_div_up(len, 256), 4096); }

}  // namespace

extern "C" {

int rnn_linear_act_forward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                           const float *w, const float *b, uint32_t act, const float *res,
                           float *z, float *y) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (act > RNN_ACT_SILU)
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_forward: activation %u", act);
    if (rows == 0 || fout == 0) return RNN_OK;
    if ((fin && (!x || !w)) || !y) return rnn_fail(ctx, RNN_E_NULL, "linear_act_forward: null operand");
    if (y == x || (z && (z == x || z == y || z == res)))
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_forward: aliased operands");
    RNN_ON_DEVICE(ctx);
    float *t = z ? z : y;
    if (!z && res == y)
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "linear_act_forward: res is y without z");
    const int rc = rnn_linear_forward(ctx, rows, fin, fout, x ? x : t, w ? w : t, b, t);
    if (rc) return rc;
    const size_t len = rows * fout;
    by_act(act, [&](auto a) {
        act_fwd_kernel<decltype(a)::value><<<ew_grid(len), 256, 0, ctx->stream>>>(len, t, res, y);
        return 0;
    });
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_linear_act_backward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                            const float *x, const float *w, const float *z, uint32_t act,
                            float *dz, float *dw, float *db, float *dx, uint32_t flags) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (act > RNN_ACT_SILU)
        return rnn_fail(ctx, RNN_E_INVALID, "linear_act_backward: activation %u", act);
    RNN_ON_DEVICE(ctx);
    const size_t len = rows * fout;
    if (act != RNN_ACT_NONE && len) {
        if (!dy || !z || !dz) return rnn_fail(ctx, RNN_E_NULL, "linear_act_backward: null operand");
        if (dz == dx || dz == x || dz == w || dz == dy)
            return rnn_fail(ctx, RNN_E_INVALID, "linear_act_backward: dz aliases another operand");
        by_act(act, [&](auto a) {
            act_bwd_kernel<decltype(a)::value><<<ew_grid(len), 256, 0, ctx->stream>>>(len, dy, z, dz);
            return 0;
        });
        RNN_LAUNCHED(ctx);
        dy = dz;
    }
    return rnn_linear_backward_ex(ctx, rows, fin, fout, dy, x, w, dw, db, dx, flags);
}

}  // extern "C"
