// Which operands of a call share memory, for entry points that refuse results
// over what they still read.  Host only, no device headers.
#pragma once

#include <cstddef>
#include <cstdint>

// n rows of w floats (or other 32-bit words), stride >= w of them apart; p null: none.
struct RnnRows {
    const void *p;
    size_t n, stride, w;
};
inline RnnRows rnn_block(const void *p, size_t words) { return {p, 1, words, words}; }

// Whether a and b share a word.  At once where one ends before the other begins or
// the strides are the same (columns of one buffer), else row by row.
inline bool rnn_overlap(const RnnRows &a, const RnnRows &b) {
    if (!a.p || !b.p || !a.n || !b.n || !a.w || !b.w) return false;
    const uint64_t pa = (uintptr_t)a.p / 4, pb = (uintptr_t)b.p / 4;
    if (pb >= pa + (a.n - 1) * a.stride + a.w || pa >= pb + (b.n - 1) * b.stride + b.w) return false;
    if (a.stride == b.stride) {
        // b's row j begins c words after a's row j + m does
        const int64_t s = (int64_t)a.stride, off = (int64_t)(pb - pa);
        const int64_t m = off >= 0 ? off / s : -((s - 1 - off) / s), c = off - m * s;
        const auto rows_meet = [&](int64_t k) { return k > -(int64_t)b.n && k < (int64_t)a.n; };
        return (c < (int64_t)a.w && rows_meet(m)) || (c + (int64_t)b.w > s && rows_meet(m + 1));
    }
    for (size_t i = 0, j = 0; i < a.n && j < b.n;) {
        const uint64_t ra = pa + i * a.stride, rb = pb + j * b.stride;
        if (ra + a.w <= rb)
            i++;
        else if (rb + b.w <= ra)
            j++;
        else
            return true;
    }
    return false;
}

// Whether one of the results shares a word with an operand or another result.
template <size_t O, size_t I>
bool rnn_any_overlap(const RnnRows (&out)[O], const RnnRows (&in)[I]) {
    for (size_t i = 0; i < O; i++) {
        for (size_t j = 0; j < I; j++)
            if (rnn_overlap(out[i], in[j])) return true;
        for (size_t j = i + 1; j < O; j++)
            if (rnn_overlap(out[i], out[j])) return true;
    }
    return false;
}
