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
#include "mfma_half.h"
#include "rnn_overlap.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MAX_D = 128;
constexpr int C = 32;  // tokens of a chunk
constexpr size_t SIMDS = 1024;  // four of each of 256 compute units

// Division of numbers below 2^31 by d: (mulhi(x, m) + x) >> s.
struct Divider {
    uint32_t d = 1, m = 0, s = 0;
    Divider() = default;
    explicit Divider(uint32_t by) : d(by) {
        while ((1ull << s) < by) s++;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - by)) / by + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x, uint32_t &rest) const {
        const uint32_t q = (__umulhi(x, m) + x) >> s;
        rest = x - q * d;
        return q;
    }
};

struct DecayJob {
    const float *a, *b, *c;
    float *y;
    const float *s0;    // [n][h] states before the first token; null: 0
    float *s1;          // states after the last; null: not wanted
    const float *dot;   // the rates' gradient: what the weighted sums are dotted with
    const float *s1g;   // and the gradient of the last state
    float *seg;         // [nseg][n][h] states before each segment of the walk
    const float *segg;  // the rates' gradient: those of the walk the other way
    long long as, bs, cs, ys, ds;  // row strides
    int da, dc;         // channels
    int ga, gb, gc;     // query heads that share a head of the operand
    int si, sj;         // a state's strides along da and dc
    float sa, sb;       // factors of a and of b
    int rev, acc;       // from the last token; y accumulates
    Divider slices;     // c's channels, by 32
};

struct DecayArgs {
    DecayJob job[3];
    const float *rate;
    const uint32_t *lens;
    double *part;  // [n][nseg][slices][h] parts of dL/dg
    float *drate;  // their sums' place, added by `h` blocks past a launch's `walk` ones
    int parts, walk;
    int n, t, h, reverse;
    int nseg;  // segments of a sequence
    Divider segs, heads;
};

__device__ __forceinline__ int length(const DecayArgs &g, long long b) {
    return g.lens ? (int)min(g.lens[b], (uint32_t)g.t) : g.t;
}

// A sequence's segments: its chunks in as many runs, the first ones a chunk longer
// where they do not divide; a run is of rows, whatever a head's direction.
struct Segments {
    int len, longer, each;  // tokens, runs of each + 1 chunks, chunks
    __device__ __forceinline__ Segments(const DecayArgs &g, int tokens) : len(tokens) {
        uint32_t rest;
        each = (int)g.segs((uint32_t)(len + C - 1) / C, rest);
        longer = (int)rest;
    }
    __device__ __forceinline__ int first(int k) const {
        return min(C * (k * each + min(k, longer)), len);
    }
    // the last one that holds tokens; 0 if none does
    __device__ __forceinline__ int last(int nseg) const { return max(each ? nseg : longer, 1) - 1; }
};

// log gamma of a head: at most 0, and finite, so that its multiple by 0 is 0 (of a
// rate that is no number NaN).
__device__ __forceinline__ double log_gamma(float rate) {
    const double g = -exp((double)rate);
    return g < -1e30 ? -1e30 : g;
}

// gamma^m in 32 bits, as a power of two whose exponent m log2(gamma) is in two parts:
// the instruction's ulp and a product's rounding.
struct Power {
    float hi, lo;
    __device__ __forceinline__ explicit Power(double lg) {
        const double l2 = lg * 1.4426950408889634;
        hi = (float)l2;
        lo = (float)(l2 - (double)hi);
    }
    __device__ __forceinline__ float operator()(int m) const {
        const float f = (float)m, t = f * hi;
        const float rest = t < -200.f ? 0.f : __builtin_fmaf(f, hi, -t) + f * lo;
        return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(rest, 0.69314718f, 1.f);
    }
};

// s gamma, gamma in two parts.
__device__ __forceinline__ float decayed(float s, float gam, float rest) {
    return __builtin_fmaf(s, gam, s * rest);
}

// Token by token, forward: a block holds a head's state, four channels of v a
// thread in every RP-th row, RP = 256 / G, G groups of four channels (a power of
// two).  Its read and write are the work: 16 bytes an access (VEC: dv a multiple of
// four, states aligned), all of them in flight at once: 64 streams of 8 heads of 64 x
// 128 8.6 us, 3.9 TB/s; one of 4 heads of 64 x 64 4.0, a launch's least.  (Four bytes an
// access: 16.3.)
template <bool VEC, int G>
__global__ __launch_bounds__(256) void decay_tokens_kernel(DecayArgs g) {
    constexpr int RP = 256 / G, K = MAX_D / RP;
    __shared__ __attribute__((aligned(16))) float red[RP][4 * G], ab[2][MAX_D];
    const DecayJob &q = g.job[0];
    const int c4 = 4 * (threadIdx.x & (G - 1)), r0 = threadIdx.x / G;
    const int b = blockIdx.x / g.h, hd = blockIdx.x % g.h;
    const long long st = ((long long)b * g.h + hd) * q.da * q.dc;
    f32x4 s[K];
    const auto each = [&](auto f) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (r0 + k * RP < q.da && c4 < q.dc) f(k, st + (long long)(r0 + k * RP) * q.dc + c4);
    };
#pragma unroll
    for (int k = 0; k < K; k++) s[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (q.s0)
        each([&](int k, long long at) {
            if constexpr (VEC) {
                s[k] = *(const f32x4 *)(q.s0 + at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) s[k][e] = c4 + e < q.dc ? q.s0[at + e] : 0.f;
            }
        });
    const int len = length(g, b);
    const bool back = hd >= g.h - g.reverse;
    // gamma in two floats: one rounded alone would be off by its last bit to
    // the power of the tokens
    const double g64 = exp(log_gamma(g.rate[hd]));
    const float gam = (float)g64, rest = (float)(g64 - (double)gam);
    const int tid = threadIdx.x;
    for (int i = 0; i < g.t; i++) {
        if (i >= len) {
            if (tid < q.dc) q.y[((long long)b * g.t + i) * q.ys + hd * q.dc + tid] = 0.f;
            continue;
        }
        const long long row = (long long)b * g.t + (back ? len - 1 - i : i);
        const float *c = q.c + row * q.cs + (hd / q.gc) * q.dc;
        if (tid < q.da)
            ab[0][tid] = q.a[row * q.as + hd * q.da + tid];
        else if (tid >= 128 && tid - 128 < q.da)
            ab[1][tid - 128] = q.b[row * q.bs + (hd / q.gb) * q.da + tid - 128];
        f32x4 cv, o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; e++) cv[e] = c4 + e < q.dc ? c[c4 + e] : 0.f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int r = r0 + k * RP;
            if (r >= q.da) continue;
            const float av = ab[0][r], bv = ab[1][r];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[k][e] = __builtin_fmaf(bv, cv[e], decayed(s[k][e], gam, rest));
                o[e] = __builtin_fmaf(av, s[k][e], o[e]);
            }
        }
        *(f32x4 *)&red[r0][c4] = o;
        __syncthreads();
        if (tid < q.dc) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < RP; k++) v += red[k][tid];
            q.y[row * q.ys + hd * q.dc + tid] = q.sa * v;
        }
    }
    if (q.s1)
        each([&](int k, long long at) {
            if constexpr (VEC) {
                *(f32x4 *)(q.s1 + at) = s[k];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c4 + e < q.dc) q.s1[at + e] = s[k][e];
            }
        });
}

__device__ __forceinline__ f32x16 mm32(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// Register r of a 32 x 32 accumulator holds row tile_row(r) + 4 (lane / 32) of
// column lane % 32.  Taken as an operand of a product, register r stands for the
// k's tile_row(r) and tile_row(r) + 4: accumulators are operands as they are.
__device__ __forceinline__ constexpr int tile_row(int r) { return (r & 3) + 8 * (r >> 2); }

// Rows of a head in the order of a walk: the p-th token from `first` on.
struct Walk {
    long long first;
    int dir;  // +1, -1
};

// Past the end of every resource here (32 rows of at most 2^24 bytes), whatever
// rows and channels are added to it or taken from it.
constexpr uint32_t NOWHERE = 0x50000000u;

// Keeps what depends on v in the loop: hoisted out of it, the comparisons of a
// chunk's places and channels fill the scalar registers.
__device__ __forceinline__ int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A chunk's rows of an operand or a result: L of them, the resource beginning at
// the lowest; what lies outside reads as 0 and is not written.
struct ChunkRows {
    __amdgpu_buffer_rsrc_t rs;
    uint32_t stride;  // bytes
    int lim, step, L;
    __device__ __forceinline__ ChunkRows(const float *p, long long st, int width, const Walk &w, int c0,
                                         int n)
        : stride((uint32_t)st * 4u), lim(width), step(w.dir), L(n) {
        const long long low = w.dir < 0 ? w.first - c0 - (n - 1) : w.first + c0;
        rs = rows_rsrc(p + low * st, n, st, width);
    }
    // Byte offset of channel ch at place p.  Places past the end come out beyond
    // the resource either way, rows below it as offsets near 2^32.
    __device__ __forceinline__ uint32_t at(int p, int ch) const {
        const uint32_t c = ch < lim ? 4u * (uint32_t)ch : NOWHERE;
        return c + (uint32_t)(step < 0 ? L - 1 - p : p) * stride;
    }
    // From the offset of place p, that of place p + k.
    __device__ __forceinline__ uint32_t go(uint32_t at, int k) const {
        return at + (uint32_t)(step * k) * stride;
    }
    __device__ __forceinline__ float load(uint32_t at) const {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0));
    }
    __device__ __forceinline__ void store(uint32_t at, float v) const {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rs, at, 0, 0);
    }
};

// An operand's k's along the channels: register 4 k + e of lane l is channel 8 k +
// 4 (l / 32) + e of the row at place l % 32, as accumulators order their rows.
template <int DAT>
__device__ __forceinline__ void load_rows(const ChunkRows &x, int ln, int half, f32x4 (&v)[4 * DAT]) {
    const uint32_t at = ln < x.L ? x.at(ln, 0) + 4u * (uint32_t)half : NOWHERE;
#pragma unroll
    for (int k = 0; k < 4 * DAT; k++)
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x.rs, at + 32 * k, 0, 0));
}
// Channels from `lim` on, which are another head's, as 0 (FULL: there are none).
template <int DAT, bool FULL>
__device__ __forceinline__ void cut_rows(int lim, int half, f32x4 (&v)[4 * DAT]) {
    if (FULL) return;
    const int t = opaque(half - lim);
#pragma unroll
    for (int k = 0; k < 4 * DAT; k++) {
        u32x4 w = __builtin_bit_cast(u32x4, v[k]);
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] &= (uint32_t)((t + 8 * k + e) >> 31);
        v[k] = __builtin_bit_cast(f32x4, w);
    }
}
// Sixteen places of channel ch: k's along the tokens.
__device__ __forceinline__ void load_cols(const ChunkRows &x, int half, int ch, float (&v)[16]) {
    const uint32_t at = x.at(half, ch);
#pragma unroll
    for (int r = 0; r < 16; r++) v[r] = x.load(x.go(at, tile_row(r)));
}

// A state in memory, as the walk's accumulators hold it: register r of tile d is
// row 32 d + tile_row(r) + half of column col.
struct StateRows {
    __amdgpu_buffer_rsrc_t rs;
    uint32_t si, base;  // bytes
    int rows;           // rows from `half` on
    __device__ __forceinline__ StateRows(const float *p, const DecayJob &q, int half, int col)
        : rs(make_rsrc(p, (uint32_t)(q.da * q.dc) * 4u)), si((uint32_t)q.si * 4u),
          base(col < q.dc ? (uint32_t)(col * q.sj + half * q.si) * 4u : NOWHERE), rows(q.da - half) {}
    __device__ __forceinline__ uint32_t at(int d, int r) const {
        const int i = 32 * d + tile_row(r);
        return i < opaque(rows) ? base + (uint32_t)i * si : NOWHERE;
    }
    __device__ __forceinline__ float load(int d, int r) const {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at(d, r), 0, 0));
    }
    __device__ __forceinline__ void store(int d, int r, float v) const {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rs, at(d, r), 0, 0);
    }
};

// A head's powers of gamma in LDS, of a wave's own.
struct Powers {
    float near[C];      // gamma^m
    float first[C];     // gamma^(p + e) sa
    float left[C];      // gamma^(L - p - e) sb, of a chunk of L places
};

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Sixteen places' entries of a table, as an accumulator's rows.
__device__ __forceinline__ void places(const float *tab, int half, float (&v)[16]) {
    const float *t = tab + opaque(half);
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const f32x4 w = *(const f32x4 *)(t + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * q + e] = w[e];
    }
}

// o + p c over a chunk, where p (register r: the keys of operand register r) is 0
// for keys behind the query: a value of c that is no number makes its column's
// rows from its own on NaN, and none before.
__device__ __forceinline__ f32x16 tri_product(const f32x16 &p, const float (&c)[16], f32x16 o, int half) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) m = __builtin_fmaf(c[r], 0.f, m);
    if (!__any(m != m)) {
#pragma unroll
        for (int r = 0; r < 16; r++) o = mm32(p[r], c[r], o);
        return o;
    }
    int bad = C;
#pragma unroll
    for (int r = 0; r < 16; r++) {  // the same sums in the same order
        const bool ok = c[r] * 0.f == 0.f;
        if (!ok) bad = min(bad, tile_row(r) + half);
        o = mm32(p[r], ok ? c[r] : 0.f, o);
    }
    bad = min(bad, __shfl_xor(bad, 32, 64));
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (tile_row(r) + half >= bad) o[r] = __builtin_nanf("");
    return o;
}

// drate[j] += g sum of the head's parts, in a fixed order, by a block among those of the
// next walk (a launch for it took 4 us more).
__device__ void sum_rate(const DecayArgs &g, int j) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < g.parts; i += 256) s += g.part[(long long)i * g.h + j];
    s = rnn_wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        g.drate[j] += (float)(log_gamma(g.rate[j]) * (red[0] + red[1] + red[2] + red[3]));
}

enum { WALK = 0, WALK_RATE = 1, STATE = 2 };

// A wave takes 32 of c's channels of a head through a segment, 32 tokens at a
// time, its part of the state (DAT tiles of 32 x 32) in accumulators:
//   P^T = b a^T, weighted by gamma^(i-l) and cut; y = gamma^(i + e) a T + P c;
//   T = gamma^32 T + (gamma^(32 - l - e) b)^T c        (e: 1, rev: 0)
// Rows come straight from global memory in the operands' layouts, the next
// chunk's into the registers that this one's products have freed; b's channels by
// tokens through the wave's own LDS.  A wave shares nothing with another one and
// waits for none.  WALK_RATE: the rates' gradient as well.  STATE: the segment's
// own T alone.
//
// Bound by the fp32 products, 16 + 48 DAT of 64 cycles a chunk (32 + 80 DAT with the
// rates): one wave a SIMD takes 4.5 us a chunk of 64 x 64 heads, 65 % of their rate at
// 2.4 GHz, two as much for each.  (Measured and not better: rows shared by a block's
// waves through LDS with barriers, products and other instructions interleaved by
// hand.)  8 clips of 1568 tokens, 8 heads of 64: forward 37 us and 23 for the states
// between segments, dq and the rates 67, dk and dv 64, their states 34; 128 images of
// 64 tokens, 4 heads: 15, 21 and 23.  Four tiles with the rates do not fit the
// registers, 66 or 68 of which go through scratch: 8 x 1568 tokens unpadded, 4 heads of
// 128 x 128 173 us, where the products come to 135 by those of 8 heads of 64 x 64 (74);
// three tiles fit but for one register at most (4 heads of 96 x 96: 78).
template <int DAT, bool FULL, int MODE>
__global__ __launch_bounds__(256, DAT <= (MODE == WALK_RATE ? 1 : 2) ? 2 : 1) void decay_walk_kernel(DecayArgs g) {
    // rows of b: 4 rows apart are half of the banks apart
    constexpr int BS = 32 * DAT + 8;
    __shared__ __attribute__((aligned(16))) Powers tables[4];
    __shared__ __attribute__((aligned(16))) float btile[MODE == STATE ? 1 : 4][MODE == STATE ? 4 : C * BS];
    const DecayJob &q = g.job[blockIdx.y];
    const int lane = threadIdx.x & 63, ln = lane & 31, half = 4 * (lane >> 5), wave = wave_index();
    // the arguments at once, not one after the other as they are needed (128 x 64
    // tokens 15.4 us against 14.9)
    asm volatile("" ::"s"(q.a), "s"(q.b), "s"(q.c), "s"(q.y), "s"(q.s0), "s"(q.as), "s"(q.bs), "s"(q.cs),
                 "s"(q.ys), "s"(q.da), "s"(q.ga), "s"(q.sa), "s"(q.rev), "s"(g.rate));
    if (MODE == WALK && (int)blockIdx.x >= g.walk) {  // of the launch after the one that left the parts
        if (blockIdx.y == 0) sum_rate(g, (int)blockIdx.x - g.walk);
        return;
    }
    uint32_t u = (uint32_t)xcd_order(blockIdx.x, g.walk) * 4 + wave, rest;  // fewer than 2^31 waves
    u = q.slices(u, rest);
    const int slice = (int)rest, col = slice * 32 + ln;
    u = g.segs(u, rest);
    const int seg = (int)rest;
    const long long b = g.heads(u, rest);
    const int hd = (int)rest;
    if (b >= g.n) return;
    const Segments runs(g, __builtin_amdgcn_readfirstlane(length(g, b)));
    const int t0 = runs.first(seg), t1 = runs.first(seg + 1), T = t1 - t0;
    const bool lastseg = seg == runs.last(g.nseg);
    constexpr bool slope = MODE == WALK_RATE;
    const int e0 = q.rev ? 0 : 1;
    const bool incol = col < q.dc;
    if (MODE != STATE && !q.acc && runs.len < g.t) {  // padding rows, shared among the runs
        const int pad = g.t - runs.len, each = (pad + g.nseg - 1) / g.nseg;
        const int z0 = min(seg * each, pad), z1 = min(z0 + each, pad);
        for (int i = runs.len + z0 + (lane >> 5); i < runs.len + z1; i += 2)
            if (incol) q.y[(b * g.t + i) * q.ys + hd * q.dc + col] = 0.f;
    }
    Powers &pw = tables[wave];
    float *bt = btile[MODE == STATE ? 0 : wave];
    double dg = 0.0;
    const long long st = (b * g.h + hd) * q.da * q.dc;
    const long long sg = ((long long)seg * g.n * g.h) * q.da * q.dc + st;
    const bool down = (hd >= g.h - g.reverse) != (q.rev != 0);
    const Walk w = {b * g.t + (down ? t1 - 1 : t0), down ? -1 : 1};
    const bool ends = down ? seg == 0 : lastseg;    // holds the walk's last token
    const bool begins = down ? lastseg : seg == 0;  // holds its first
    if (MODE == STATE && (T == 0 || ends)) return;
    const float *pa = q.a + (hd / q.ga) * q.da, *pb = q.b + (hd / q.gb) * q.da,
                *pc = q.c + (hd / q.gc) * q.dc;
    f32x4 af[4 * DAT], bf[4 * DAT];
    float cf[16], bcol[MODE == STATE ? DAT : 1][16];
    {
        const int L = min(C, T);
        const ChunkRows rb(pb, q.bs, q.da, w, 0, L);
        if constexpr (MODE != STATE) {
            load_rows<DAT>(rb, ln, half, bf);
            load_rows<DAT>(ChunkRows(pa, q.as, q.da, w, 0, L), ln, half, af);
        } else {
#pragma unroll
            for (int d = 0; d < DAT; d++) load_cols(rb, half, 32 * d + ln, bcol[d]);
        }
        load_cols(ChunkRows(pc, q.cs, q.dc, w, 0, L), half, col, cf);
    }
    // the state: rows 32 d + tile_row(r) + half, column col
    const float *s0 = MODE == STATE ? nullptr : g.nseg > 1 ? q.seg + sg : begins && q.s0 ? q.s0 + st : nullptr;
    f32x16 S[DAT], Z[MODE == WALK_RATE ? DAT : 1];
#pragma unroll
    for (int d = 0; d < DAT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            S[d][r] = 0.f;
            if (MODE == WALK_RATE) Z[d][r] = 0.f;
        }
    if (s0) {
        const StateRows x(s0, q, half, col);
#pragma unroll
        for (int d = 0; d < DAT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) S[d][r] = x.load(d, r);
    }
    const float *sgrad = !slope || !T ? nullptr : g.nseg > 1 ? q.segg + sg : q.s1g ? q.s1g + st : nullptr;
    bool any = s0 != nullptr;  // whether the state may be other than 0
    const double lg = log_gamma(g.rate[hd]);
    wave_sync();
    const Power pow(lg);
    if (lane < C) {
        pw.near[lane] = pow(lane);
        pw.first[lane] = pow(lane + e0) * q.sa;
    }
    float hi = 0.f, lo = 0.f;  // gamma^L, in two parts
    for (int c0 = 0; c0 < T; c0 += C) {
        const int L = min(C, T - c0), next = min(C, max(T - c0 - C, 0));
        if (c0 == 0 || L < C) {
            const double all = exp(lg * L);
            hi = (float)all;
            lo = (float)(all - (double)hi);
            wave_sync();
            if (lane < C) pw.left[lane] = pow(max(L - lane - e0, 0)) * q.sb;
            wave_sync();
        }
        // whether a reader of the state follows
        const bool goes = MODE == STATE || c0 + L < T || sgrad || (ends && q.s1);
        if constexpr (MODE != STATE) {
            f32x16 P, o, oz;
#pragma unroll
            for (int r = 0; r < 16; r++) P[r] = o[r] = oz[r] = 0.f;
            cut_rows<DAT, FULL>(q.da, half, af);
            cut_rows<DAT, FULL>(q.da, half, bf);
            wave_sync();
#pragma unroll
            for (int k = 0; k < 4 * DAT; k++) *(f32x4 *)(bt + ln * BS + 8 * k + half) = bf[k];
#pragma unroll
            for (int k = 0; k < 4 * DAT; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) P = mm32(bf[k][e], af[k][e], P);
            __builtin_amdgcn_sched_barrier(0);
            load_rows<DAT>(ChunkRows(pb, q.bs, q.da, w, c0 + C, next), ln, half, bf);
            __builtin_amdgcn_sched_barrier(0);
            const int query = opaque(ln - half);
            const float sab = q.sa * q.sb;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                // keys behind the query: 0, also of what is no number
                const int far = query - tile_row(r);
                const float v = __uint_as_float(__float_as_uint(P[r]) & ~(uint32_t)(far >> 31));
                P[r] = v * (pw.near[max(far, 0)] * sab);
            }
            if (any) {
                float row[16];
                places(pw.first, half, row);
#pragma unroll
                for (int d = 0; d < DAT; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o = mm32(af[4 * d + (r >> 2)][r & 3], S[d][r], o);
                if (slope) {
#pragma unroll
                    for (int d = 0; d < DAT; d++)
#pragma unroll
                        for (int r = 0; r < 16; r++) oz = mm32(af[4 * d + (r >> 2)][r & 3], Z[d][r], oz);
                    const float one = (float)(half + 1);
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        oz[r] = row[r] * __builtin_fmaf(one + (float)tile_row(r), o[r], oz[r]);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) o[r] *= row[r];
            }
            __builtin_amdgcn_sched_barrier(0);
            load_rows<DAT>(ChunkRows(pa, q.as, q.da, w, c0 + C, next), ln, half, af);
            float dot[16];
            if (slope) load_cols(ChunkRows(q.dot + hd * q.dc, q.ds, q.dc, w, c0, L), half, col, dot);
            __builtin_amdgcn_sched_barrier(0);
            o = tri_product(P, cf, o, half);
            const ChunkRows ry(q.y + hd * q.dc, q.ys, q.dc, w, c0, L);
            const uint32_t y_at = ry.at(half, col);
            if (q.acc) {
#pragma unroll
                for (int r = 0; r < 16; r++) o[r] += ry.load(ry.go(y_at, tile_row(r)));
            }
#pragma unroll
            for (int r = 0; r < 16; r++) ry.store(ry.go(y_at, tile_row(r)), o[r]);
            if (slope) {
                const float fq = (float)query;
#pragma unroll
                for (int r = 0; r < 16; r++) P[r] *= fq - (float)tile_row(r);
                oz = tri_product(P, cf, oz, half);
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) sum = __builtin_fmaf(oz[r], dot[r], sum);
                dg += (double)sum;
            }
        }
        if (goes) {
            // b's rows in LDS, which other lanes have written
            if (MODE != STATE) wave_sync();
            float left[16];
            places(pw.left, half, left);
#pragma unroll
            for (int r = 0; r < 16; r++) cf[r] *= left[r];
#pragma unroll
            for (int d = 0; d < DAT; d++) {
                float bd[16];
#pragma unroll
                for (int r = 0; r < 16; r++)
                    bd[r] = MODE == STATE ? bcol[MODE == STATE ? d : 0][r]
                                          : bt[(tile_row(r) + half) * BS + 32 * d + ln];
                if (slope) {
                    const float fl = (float)(L - 1 - half);
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        Z[d][r] = decayed(__builtin_fmaf((float)L, S[d][r], Z[d][r]), hi, lo);
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        Z[d] = mm32(bd[r], cf[r] * (fl - (float)tile_row(r)), Z[d]);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) S[d][r] = decayed(S[d][r], hi, lo);
#pragma unroll
                for (int r = 0; r < 16; r++) S[d] = mm32(bd[r], cf[r], S[d]);
                if constexpr (MODE == STATE)
                    load_cols(ChunkRows(pb, q.bs, q.da, w, c0 + C, next), half, 32 * d + ln, bcol[d]);
            }
            any = true;
        }
        __builtin_amdgcn_sched_barrier(0);
        load_cols(ChunkRows(pc, q.cs, q.dc, w, c0 + C, next), half, col, cf);
        __builtin_amdgcn_sched_barrier(0);
    }
    float *s1 = MODE == STATE ? q.seg + sg : ends && q.s1 ? q.s1 + st : nullptr;
    if (s1) {
        const StateRows x(s1, q, half, col);
#pragma unroll
        for (int d = 0; d < DAT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) x.store(d, r, S[d][r]);
    }
    if (MODE == WALK_RATE && sgrad) {
        const StateRows x(sgrad, q, half, col);
#pragma unroll
        for (int d = 0; d < DAT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) dg += (double)Z[d][r] * x.load(d, r);
    }
    if (slope) {
        dg = rnn_wave_sum_d(dg);
        if (lane == 0) g.part[((b * g.nseg + seg) * q.slices.d + slice) * g.h + hd] = dg;
    }
}

// The states before each segment, in the walk's direction, from the segments' own
// ones: one thread an element, over the segments in order.  A block's elements are
// one head's, so that lengths and factors are the same for all of them.
// Bound by the chain of loads: 64 segments of 8 heads of 64 x 128 11 us (3.0 TB/s; 16
// ahead 12.5, without the eight ahead 14), 8 of 64 of 64 x 64 6.3 (2.7).
__global__ __launch_bounds__(256) void decay_scan_kernel(DecayArgs g, int blocks) {
    const DecayJob &q = g.job[blockIdx.y];
    // `blocks` of them a head of a sequence
    const int per = q.da * q.dc, head = blockIdx.x / blocks;
    const int at = (int)(blockIdx.x - head * blocks) * 256 + threadIdx.x;
    const int b = head / g.h, hd = head - b * g.h;
    const Segments runs(g, length(g, b));
    const int last = runs.last(g.nseg);
    const bool down = (hd >= g.h - g.reverse) != (q.rev != 0);
    if (at >= per) return;
    const long long all = (long long)g.n * g.h * per, i = (long long)head * per + at;
    float s = q.s0 ? q.s0[i] : 0.f;
    // the k-th segment of the walk, eight of them loaded while the eight before are
    // worked on; the last one's own state has no reader
    float own[8], next[8];
    const auto fetch = [&](int k0) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int k = min(k0 + j, last);
            next[j] = q.seg[(long long)(down ? last - k : k) * all + i];
        }
    };
    fetch(0);
    const double lg = log_gamma(g.rate[hd]);
    // gamma to the tokens of a run: the last one's, a longer and another one's
    float hi[3], lo[3];
#pragma unroll
    for (int j = 0; j < 3; j++) {
        const double all64 = exp(lg * (j ? C * (runs.each + (j == 1)) : runs.len - runs.first(last)));
        hi[j] = (float)all64;
        lo[j] = (float)(all64 - (double)hi[j]);
    }
    for (int k0 = 0; k0 <= last; k0 += 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) own[j] = next[j];
        if (k0 + 8 <= last) fetch(k0 + 8);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int k = k0 + j;
            if (k > last) break;
            const int run = down ? last - k : k;
            q.seg[(long long)run * all + i] = s;
            const int len = run == last ? 0 : run < runs.longer ? 1 : 2;
            s = decayed(s, hi[len], lo[len]) + own[j];
        }
    }
}

// dk and dv of shared heads: the sum over the query heads' parts, in order.  Rows
// behind a sequence's end hold zeros, and stay as they are where dkv accumulates.
// (5 x 577 tokens, two key heads of 44 + 72 channels for three query heads each: 5 us,
// for which the query heads' walks run side by side; one after the other in a wave, all
// of this training pass took 378 us against 150.)
struct GroupArgs {
    const float *part[2];
    float *out[2];
    int d[2];
    const uint32_t *lens;
    long long stride[2];
    int t, hkv, grp, acc;
};
__global__ __launch_bounds__(256) void decay_group_kernel(GroupArgs g, long long rows) {
    const int k = blockIdx.y, d = g.d[k], w = g.hkv * d;
    const long long all = rows * w;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long row = i / w;
        const int at = (int)(i - row * w), hd = at / d;
        if (g.acc && g.lens && row % g.t >= (long long)g.lens[row / g.t]) continue;
        const float *p = g.part[k] + row * w * g.grp + (long long)hd * g.grp * d + (at - hd * d);
        float s = p[0];
        for (int r = 1; r < g.grp; r++) s += p[(long long)r * d];
        float *o = g.out[k] + row * g.stride[k] + at;
        *o = g.acc ? *o + s : s;
    }
}

// The form's walks over a sequence, and where a workspace's parts are.
struct DecayPlan {
    bool tokens = false;  // token by token
    int nseg = 1;
    size_t seg = 0, segr = 0, part = 0, part_k = 0, part_v = 0, bytes = 0;
};
// Segments of a walk of so many chunks by so many waves: a wave a SIMD, two of a
// forward whose registers leave room (two) and that keep four chunks each.  They cost
// a pass for the states, which are written, scanned and read, and pay where the
// chunks that a walk is spared come to more; in sixths of a chunk's time.  Four heads of
// 64 channels, us without / with them: one image of 64 tokens 12 / 16 forward and 31 /
// 41 backward, of 128 tokens 21 / 17 and 56 / 42; 64 sequences of 256 tokens 42 / 47 and
// 112 / 125, of 2048 tokens 320 / 230 and 821 / 661; 8 of 1024 tokens 149 / 31 and 407 /
// 81 (half and twice as many segments: 40, 36 and 94, 104).  Other heads' sizes have not
// been timed with and without; they do not enter.
size_t segments(size_t waves, size_t chunks, bool two, bool backward) {
    size_t k = SIMDS / waves;
    if (k < 2 || chunks < 2) return 1;  // 800 waves, 32 chunks: 106 us, in two 128
    if (two && chunks >= 4 * (2 * SIMDS / waves)) k = 2 * SIMDS / waves;
    // the scan takes them one after the other: beyond 64, two chunks each
    k = std::min(k, std::min(chunks, std::max<size_t>(64, chunks / 2)));
    const size_t each = rnn_div_up(chunks, k);
    return 6 * (chunks - each) > 10 + 2 * each + (backward ? 11 : 9) * (waves * k) / SIMDS ? k : 1;
}
DecayPlan plan_of(const rnn_decay_attn_desc *d, size_t n, size_t t, bool backward) {
    DecayPlan p;
    WsCarve c;
    // Few tokens: the state's read and write are all there is to do.  (Us with 1, 4, 8
    // and 12 tokens, by the walk: 64 streams of 8 heads of 64 x 128 17, 17, 18, 18, one of
    // 4 heads of 64 x 64 9 throughout; token by token 9, 12, 17, 22 and 4, 7, 10, 13: the
    // one stream's limit lies at 7, the many streams' at 9.)
    p.tokens = !backward && t <= 8;
    const size_t kt = rnn_div_up(d->dk, 32), vt = rnn_div_up(d->dv, 32);
    // the waves of the walk with the fewest
    const size_t waves = n * d->h * (backward ? std::min(kt, vt) : vt);
    if (!p.tokens && waves) p.nseg = (int)segments(waves, rnn_div_up(t, C), !backward && kt <= 2, backward);
    const size_t states = (size_t)p.nseg * n * d->h * d->dk * d->dv * sizeof(float);
    if (p.nseg > 1) {
        p.seg = c.take(states);
        if (backward) p.segr = c.take(states);
    }
    if (backward) p.part = c.take(n * p.nseg * rnn_div_up(d->dk, 32) * d->h * sizeof(double));
    if (backward && d->h != d->hkv) {
        p.part_k = c.take(n * t * d->h * d->dk * sizeof(float));
        p.part_v = c.take(n * t * d->h * d->dv * sizeof(float));
    }
    p.bytes = c.off;
    return p;
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
    if (d->qstride > (1u << 22) || d->kstride > (1u << 22) || d->vstride > (1u << 22) || (uint64_t)d->h * std::max(d->dk, d->dv) > (1u << 22))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "decay_attn: row stride above 2^22");
    if (d->qoff > d->qstride || d->qstride - d->qoff < qw || d->koff > d->kstride ||
        d->kstride - d->koff < kw || d->voff > d->vstride || d->vstride - d->voff < vw)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: heads do not fit a row");
    // places and segments in 32 bits, a grid's threads below 2^32
    const uint64_t heads = (uint64_t)n * d->h;
    if (t >= (1u << 29) || n >= (1u << 22) || heads >= (1u << 22) || heads * t >= (1ull << 31) ||
        heads * d->dk * d->dv >= (1ull << 31))
        return rnn_fail(ctx, RNN_E_UNSUPPORTED, "decay_attn: too many tokens, heads or states");
    return RNN_OK;
}

int check_ws(rnn_ctx *ctx, const DecayPlan &w, const void *ws, size_t bytes) {
    if (!w.bytes) return RNN_OK;
    if (!ws) return rnn_fail(ctx, RNN_E_NULL, "decay_attn: workspace is null");
    if (bytes < w.bytes)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: workspace of %zu bytes, needs %zu", bytes, w.bytes);
    if ((uintptr_t)ws & 255)
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn: workspace not 256-byte aligned");
    return RNN_OK;
}

// A call's operands as they lie in memory.
struct Layout {
    const rnn_decay_attn_desc *d;
    size_t n, rows;
    RnnRows q(const float *p) const {
        return {p ? p + d->qoff : p, rows, d->qstride, (size_t)d->h * d->dk};
    }
    RnnRows k(const float *p) const {
        return {p ? p + d->koff : p, rows, d->kstride, (size_t)d->hkv * d->dk};
    }
    RnnRows v(const float *p) const {
        return {p ? p + d->voff : p, rows, d->vstride, (size_t)d->hkv * d->dv};
    }
    RnnRows y(const float *p) const { return rnn_block(p, rows * d->h * d->dv); }
    RnnRows rates(const float *p) const { return rnn_block(p, d->h); }
    RnnRows lens(const uint32_t *p) const { return rnn_block(p, n); }
    RnnRows states(const float *p) const { return rnn_block(p, n * d->h * d->dk * d->dv); }
};

// One of the form's operands: where its rows are, and how many query heads share
// one of its heads.
struct Operand {
    const float *p;
    size_t stride;
    int share;
};

DecayJob make_job(const Operand &a, const Operand &b, int da, const Operand &c, int dc,
                  float *y, size_t ys) {
    DecayJob j{};
    j.a = a.p, j.b = b.p, j.c = c.p, j.y = y;
    j.as = (long long)a.stride, j.bs = (long long)b.stride, j.cs = (long long)c.stride;
    j.ys = (long long)ys;
    j.da = da, j.dc = dc;
    j.ga = a.share, j.gb = b.share, j.gc = c.share;
    j.si = dc, j.sj = 1;
    j.sa = j.sb = 1.f;
    j.slices = Divider((uint32_t)(dc + 31) / 32);
    return j;
}

void fill_args(DecayArgs &g, const rnn_decay_attn_desc *d, const DecayPlan &p, size_t n, size_t t,
               const float *rate, const uint32_t *lens) {
    g.nseg = p.nseg;
    g.segs = Divider((uint32_t)p.nseg);
    g.heads = Divider(d->h);
    g.rate = rate;
    g.lens = lens;
    g.part = nullptr;
    g.drate = nullptr;
    g.parts = 0;
    g.n = (int)n;
    g.t = (int)t;
    g.h = (int)d->h;
    g.reverse = (int)d->reverse;
}

// Heads of whole tiles need no cut (8 x 1568 tokens, 8 heads of 64: forward 66 us, with
// the cut 68, backward 171 and 178; 1 x 16384 tokens, 64 x 128: 116 and 124); states take
// b by channels, where those past a head's read as 0.
template <int MODE>
void launch_walk(rnn_ctx *ctx, DecayArgs &g, int jobs) {
    size_t waves = 0;
    bool full = true;
    for (int k = 0; k < jobs; k++) {
        const DecayJob &q = g.job[k];
        waves = std::max(waves, (size_t)g.n * g.h * g.nseg * q.slices.d);
        full = full && q.da % 32 == 0;
    }
    g.walk = (int)rnn_div_up(waves, 4);
    const dim3 grid((unsigned)(g.walk + (g.drate ? g.h : 0)), (unsigned)jobs);
    hipStream_t s = ctx->stream;
#define WALK_AS(DAT)                                                                \
    (full ? decay_walk_kernel<DAT, true, MODE><<<grid, 256, 0, s>>>(g)              \
          : decay_walk_kernel<DAT, MODE == STATE, MODE><<<grid, 256, 0, s>>>(g))
    switch ((g.job[0].da + 31) / 32) {
        case 1: WALK_AS(1); break;
        case 2: WALK_AS(2); break;
        case 3: WALK_AS(3); break;
        default: WALK_AS(4); break;
    }
#undef WALK_AS
}

// The states between segments: every segment's own, then over the segments.
void launch_segments(rnn_ctx *ctx, DecayArgs &g, int jobs) {
    launch_walk<STATE>(ctx, g, jobs);
    const int blocks = (int)rnn_div_up(g.job[0].da * g.job[0].dc, 256);
    decay_scan_kernel<<<dim3((unsigned)(g.n * g.h * blocks), jobs), 256, 0, ctx->stream>>>(g, blocks);
}

}  // namespace

extern "C" {

int rnn_decay_attn_workspace(const rnn_decay_attn_desc *d, size_t n, size_t t, int backward,
                             size_t *bytes) {
    const int rc = decay_check(nullptr, d, n, t);
    if (rc) return rc;
    if (!bytes) return RNN_E_NULL;
    *bytes = plan_of(d, n, t, backward != 0).bytes;
    return RNN_OK;
}

int rnn_decay_attn_forward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                           const float *q, const float *k, const float *v, const float *rate,
                           const uint32_t *lens, const float *state_in, void *ws, size_t ws_bytes,
                           float *y, float *state_out) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = decay_check(ctx, d, n, t);
    if (rc) return rc;
    if (!n || (!t && !state_out)) return RNN_OK;
    if ((t && (!q || !k || !v || !y)) || !rate) return rnn_fail(ctx, RNN_E_NULL, "decay_attn_forward: null operand");
    const Layout at = {d, n, n * t};
    // the states may be handed on in place
    const RnnRows ins[] = {at.q(q), at.k(k), at.v(v), at.rates(rate), at.lens(lens),
                           at.states(state_in == state_out ? nullptr : state_in)};
    const RnnRows outs[] = {at.y(y), at.states(state_out)};
    if (rnn_any_overlap(outs, ins))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn_forward: a result over another operand");
    const DecayPlan w = plan_of(d, n, t, false);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    DecayArgs g;
    fill_args(g, d, w, n, t, rate, lens);
    const int grp = (int)(d->h / d->hkv);
    const Operand Q = {q + d->qoff, d->qstride, 1}, K = {k + d->koff, d->kstride, grp},
                  V = {v + d->voff, d->vstride, grp};
    DecayJob &j = g.job[0];
    j = make_job(Q, K, (int)d->dk, V, (int)d->dv, y, (size_t)d->h * d->dv);
    j.s0 = state_in;
    j.s1 = state_out;
    j.sa = d->scale;
    if (w.tokens) {
        const unsigned grid = (unsigned)(n * d->h);
        const bool vec = d->dv % 4 == 0 && (((uintptr_t)state_in | (uintptr_t)state_out) & 15) == 0;
#define TOKENS_AS(G)                                                              \
    (vec ? decay_tokens_kernel<true, G><<<grid, 256, 0, ctx->stream>>>(g)         \
         : decay_tokens_kernel<false, G><<<grid, 256, 0, ctx->stream>>>(g))
        if (d->dv > 64)
            TOKENS_AS(32);
        else if (d->dv > 32)
            TOKENS_AS(16);
        else
            TOKENS_AS(8);
#undef TOKENS_AS
        RNN_LAUNCHED(ctx);
        return RNN_OK;
    }
    if (w.nseg > 1) {
        j.seg = (float *)((char *)ws + w.seg);
        launch_segments(ctx, g, 1);
        RNN_LAUNCHED(ctx);
    }
    launch_walk<WALK>(ctx, g, 1);
    RNN_LAUNCHED(ctx);
    return RNN_OK;
}

int rnn_decay_attn_backward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                            const float *q, const float *k, const float *v, const float *rate,
                            const uint32_t *lens, const float *state_in, const float *dy,
                            const float *dstate_out, void *ws, size_t ws_bytes, float *dq, float *dk,
                            float *dv, float *drate, float *dstate_in, uint32_t flags) {
    if (!ctx) return RNN_E_NULL;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    int rc = decay_check(ctx, d, n, t);
    if (rc) return rc;
    if (flags & ~(uint32_t)(RNN_ATTN_SET_DQ | RNN_ATTN_SET_DKV))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn_backward: unknown flags 0x%x", flags);
    if (!n || (!t && !dstate_in)) return RNN_OK;
    if ((t && (!q || !k || !v || !dy || !dq || !dk || !dv)) || !rate)
        return rnn_fail(ctx, RNN_E_NULL, "decay_attn_backward: null operand");
    const Layout at = {d, n, n * t};
    const RnnRows ins[] = {at.q(q), at.k(k), at.v(v), at.rates(rate), at.lens(lens),
                           at.states(state_in), at.y(dy), at.states(dstate_out)};
    const RnnRows outs[] = {at.q(dq), at.k(dk), at.v(dv), at.rates(drate), at.states(dstate_in)};
    if (rnn_any_overlap(outs, ins))
        return rnn_fail(ctx, RNN_E_INVALID, "decay_attn_backward: a gradient over another operand");
    const DecayPlan w = plan_of(d, n, t, true);
    rc = check_ws(ctx, w, ws, ws_bytes);
    if (rc) return rc;
    RNN_ON_DEVICE(ctx);
    DecayArgs g;
    fill_args(g, d, w, n, t, rate, lens);
    const int grp = (int)(d->h / d->hkv), kd = (int)d->dk, vd = (int)d->dv;
    const Operand Q = {q + d->qoff, d->qstride, 1}, K = {k + d->koff, d->kstride, grp},
                  V = {v + d->voff, d->vstride, grp}, O = {dy, (size_t)d->h * d->dv, 1};
    g.part = (double *)((char *)ws + w.part);
    DecayJob &jq = g.job[0], &jk = g.job[1], &jv = g.job[2];
    jq = make_job(O, V, vd, K, kd, dq + d->qoff, d->qstride);
    jq.si = 1, jq.sj = vd;
    jq.s0 = state_in;
    jq.sa = d->scale;
    jq.acc = !(flags & RNN_ATTN_SET_DQ);
    if (drate) {
        jq.dot = Q.p;
        jq.ds = (long long)d->qstride;
        jq.s1g = dstate_out;
    }
    // keys and values that query heads share: each head's part, then their sum
    const bool share = grp > 1;
    float *part_k = (float *)((char *)ws + w.part_k), *part_v = (float *)((char *)ws + w.part_v);
    jk = make_job(V, O, vd, Q, kd, share ? part_k : dk + d->koff, share ? (size_t)d->h * kd : d->kstride);
    jk.si = 1, jk.sj = vd;
    jv = make_job(K, Q, kd, O, vd, share ? part_v : dv + d->voff, share ? (size_t)d->h * vd : d->vstride);
    jk.s0 = jv.s0 = dstate_out;
    jk.sb = jv.sb = d->scale;
    jk.rev = jv.rev = 1;
    const int acc = !(flags & RNN_ATTN_SET_DKV);
    jk.acc = jv.acc = share ? 0 : acc;
    jv.s1 = dstate_in;
    if (w.nseg > 1) {
        // S from the keys and values, R from the queries and dy
        DecayArgs sg = g;
        sg.job[0] = make_job(Q, K, kd, V, vd, nullptr, 0);
        sg.job[0].s0 = state_in;
        sg.job[0].seg = (float *)((char *)ws + w.seg);
        sg.job[1] = jv;
        sg.job[1].seg = (float *)((char *)ws + w.segr);
        launch_segments(ctx, sg, 2);
        RNN_LAUNCHED(ctx);
        jq.seg = sg.job[0].seg;
        jk.seg = jv.seg = sg.job[1].seg;
        jq.segg = sg.job[1].seg;
    }
    // dq: with the rates' gradient it takes twice the registers, by itself; dk and
    // dv together where their states have as many tiles
    DecayArgs one = g;
    if (drate) {
        launch_walk<WALK_RATE>(ctx, one, 1);
        RNN_LAUNCHED(ctx);
        one.job[0] = jk;
        one.job[1] = jv;
        one.drate = drate;  // dk's and dv's launch adds it
        one.parts = (int)(n * w.nseg * rnn_div_up(d->dk, 32));
    }
    const bool joint = (kd + 31) / 32 == (vd + 31) / 32;
    launch_walk<WALK>(ctx, one, (drate ? 1 : 2) + (joint ? 1 : 0));
    RNN_LAUNCHED(ctx);
    if (!joint) {
        one.job[0] = jv;
        one.drate = nullptr;
        launch_walk<WALK>(ctx, one, 1);
        RNN_LAUNCHED(ctx);
    }
    if (share && t) {
        GroupArgs ga = {{part_k, part_v}, {dk + d->koff, dv + d->voff}, {kd, vd}, lens,
                        {(long long)d->kstride, (long long)d->vstride}, (int)t, (int)d->hkv, grp, acc};
        const size_t each = n * t * d->hkv * (size_t)std::max(kd, vd);
        decay_group_kernel<<<dim3((unsigned)std::min<size_t>(rnn_div_up(each, 256), 4096), 2), 256, 0,
                             ctx->stream>>>(ga, (long long)(n * t));
        RNN_LAUNCHED(ctx);
    }
    return RNN_OK;
}

}  // extern "C"
