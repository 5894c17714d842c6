// The angles of rotary positions, for the kernels that turn channel pairs.
//
// A pair (u, v) of axis a turns by pos_a w, w = base^(-p / p_a).  In 32 bits
// pos w alone is off by 2^-24 of itself, a fifth of a turn at a position of
// 2^23, so the angle is formed in 64 bits, in quarter turns: pos (w 2 / pi),
// its nearest whole number taken off exactly, and what remains, at most pi / 4,
// goes into the Taylor sums of sine and cosine up to x^13 and x^14 (the first
// term left out is below 3e-14 there), rounded once to 32 bits.
#pragma once

#include "rnn_internal.h"

#include <cmath>
#include <cstring>

constexpr int MAX_PAIRS = 256;

// RNN_OK, or the code with which a description is refused (ctx may be null).
int rnn_rotary_checked(rnn_ctx *ctx, const rnn_rotary_desc *d, size_t n, size_t t, bool have_pos);

// Quarter turns per unit of position of every pair.  The powers (50 ns each) are kept
// for the next call of the same shares and base.
inline void rot_frequencies(const rnn_rotary_desc *d, double (&w)[MAX_PAIRS]) {
    struct Kept {
        uint32_t np[3] = {0, 0, 0};
        float base = 0.f;
        double w[MAX_PAIRS];
    };
    static thread_local Kept kept;
    const uint32_t np[3] = {d->p0, d->p1, d->p2};
    const size_t all = (size_t)np[0] + np[1] + np[2];
    if (kept.base != d->base || std::memcmp(kept.np, np, sizeof(np))) {
        int j = 0;
        for (int a = 0; a < 3; a++)
            for (uint32_t p = 0; p < np[a]; p++)
                kept.w[j++] = std::pow((double)d->base, -(double)p / (double)np[a]) *
                              0.63661977236758134308;  // 2 / pi
        std::memcpy(kept.np, np, sizeof(np));
        kept.base = d->base;
    }
    std::memcpy(w, kept.w, all * sizeof(double));
}

// The position of row r on pair j's axis (g: a kernel's arguments).
template <typename G>
__device__ __forceinline__ double rot_position(const G &g, int r, int j) {
    const int ax = j < g.p0 ? 0 : j < g.p0 + g.p1 ? 1 : 2;
    if (g.pos) return g.pos[(long long)r * g.axes + ax];
    const int tt = r % g.t, q = tt / g.g2;
    return ax == 0 ? q / g.g1 : ax == 1 ? q % g.g1 : tt % g.g2;
}

// Sine and cosine of `q` quarter turns.
__device__ __forceinline__ void rot_sincos(double q, float *s, float *c) {
    const double k = rint(q);
    const double x = (q - k) * 1.57079632679489661923;
    const double z = x * x;
    double a = 1.0 / 6227020800.0;  // 1 / 13!
    a = fma(a, z, -1.0 / 39916800.0);
    a = fma(a, z, 1.0 / 362880.0);
    a = fma(a, z, -1.0 / 5040.0);
    a = fma(a, z, 1.0 / 120.0);
    a = fma(a, z, -1.0 / 6.0);
    const double sn = fma(a * z, x, x);
    double b = -1.0 / 87178291200.0;  // 1 / 14!
    b = fma(b, z, 1.0 / 479001600.0);
    b = fma(b, z, -1.0 / 3628800.0);
    b = fma(b, z, 1.0 / 40320.0);
    b = fma(b, z, -1.0 / 720.0);
    b = fma(b, z, 1.0 / 24.0);
    b = fma(b, z, -0.5);
    const double cs = fma(b, z, 1.0);
    // the quadrant: k mod 4 (k may be beyond an int)
    const int m = (int)(k - 4.0 * floor(k * 0.25));
    const double ss = (m & 1) ? cs : sn, cc = (m & 1) ? sn : cs;
    *s = (float)((m & 2) ? -ss : ss);
    *c = (float)((m == 1 || m == 2) ? -cc : cc);
}
