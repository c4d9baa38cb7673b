// rope_dev.h - rotary positions of several axes: the cosines and sines of 8 elements of a head, made in registers.
//
// Element e turns by A_e = pos[axis(e)] rev[e] revolutions (rev: frequency times the axis's scale over 2 pi, made in more than 64 bits on the
// host). The turn is reduced in 64 bits, where dropping whole revolutions and quarters is exact, so that a position of a million is
// as good as one of ten; what is left, at most an eighth of a revolution, goes through the Taylor series of sine and cosine (in 64 bits, to x^15
// and x^16: the next terms are 5e-17 and 2e-18 at pi / 4) and is rounded to f32 once. The rotation itself is two f32 products, each rounded, and their rounded sum:
// a key has the same bits, and so the same 4-bit codes, whichever kernel rotates it.
#pragma once
#include "kernels.h"
#include "rows_dev.h"

namespace {

__device__ __forceinline__ void turn_of(double rev, int32_t pos, float & c, float & s) {
    double t = (double) pos * rev;
    t -= __builtin_rint(t);
    const double quarter = __builtin_rint(4.0 * t);
    const double x = (t - 0.25 * quarter) * 6.283185307179586476925, y = x * x;
    double a = -1.0 / 1307674368000.0, b = 1.0 / 20922789888000.0;      // 1 / 15!, 1 / 16!
    a = __builtin_fma(a, y, 1.0 / 6227020800.0);
    b = __builtin_fma(b, y, -1.0 / 87178291200.0);
    a = __builtin_fma(a, y, -1.0 / 39916800.0);
    b = __builtin_fma(b, y, 1.0 / 479001600.0);
    a = __builtin_fma(a, y, 1.0 / 362880.0);
    b = __builtin_fma(b, y, -1.0 / 3628800.0);
    a = __builtin_fma(a, y, -1.0 / 5040.0);
    b = __builtin_fma(b, y, 1.0 / 40320.0);
    a = __builtin_fma(a, y, 1.0 / 120.0);
    b = __builtin_fma(b, y, -1.0 / 720.0);
    a = __builtin_fma(a, y, -1.0 / 6.0);
    b = __builtin_fma(b, y, 1.0 / 24.0);
    a = __builtin_fma(a * y, x, x);
    b = __builtin_fma(b, y, -0.5);
    const float sine = (float) a, cosine = (float) __builtin_fma(b, y, 1.0);
    const int q = (int) quarter;      // -2 .. 2
    c = q & 1 ? sine : cosine;
    s = q & 1 ? cosine : sine;
    if ((q + 1) & 2) c = -c;      // quarters 1, 2 of -2 .. 2 as 0 .. 3
    if (q & 2) s = -s;
}

// the positions of a row, one for each axis
struct row_pos { int32_t p[4]; };
__device__ __forceinline__ row_pos pos_of(const int32_t * pos, int64_t row, int n_axes) {
    row_pos r;
    const int32_t * at = pos + row * n_axes;
    r.p[0] = at[0];
#pragma unroll
    for (int a = 1; a < 4; a++) r.p[a] = a < n_axes ? at[a] : 0;
    return r;
}
__device__ __forceinline__ int32_t axis_pos(const row_pos & r, int axis) { return axis == 0 ? r.p[0] : axis == 1 ? r.p[1] : axis == 2 ? r.p[2] : r.p[3]; }

// cosines and sines of elements e0 .. e0 + 7; elements that do not turn have cosine 1 and sine 0
__device__ __forceinline__ void turns8(const rope_map & m, const row_pos & r, int e0, float8 & c, float8 & s) {
    float cs[8], sn[8];
    if (m.form == 1) {      // a pair's elements turn by the same
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            turn_of(m.rev[e0 + j], axis_pos(r, m.axis[e0 + j]), cs[j], sn[j]);
            cs[j + 1] = cs[j];
            sn[j + 1] = sn[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) turn_of(m.rev[e0 + j], axis_pos(r, m.axis[e0 + j]), cs[j], sn[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) { c[j] = cs[j]; s[j] = sn[j]; }
}

// Neighbours turned: x'[2i] = x[2i] c[2i] - x[2i+1] s[2i], x'[2i+1] = x[2i+1] c[2i+1] + x[2i] s[2i+1]; backward is the transpose. `left`: how many of
// the 8 turn (the rest come out as they are, whatever lies beside them).
__device__ __forceinline__ float8 turn_neighbours(float8 x, float8 c, float8 s, int left, bool back) {
    float8 y = x;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float sa = back ? s[j + 1] : -s[j], sb = back ? -s[j] : s[j + 1];
        const float a = x[j] * c[j] + x[j + 1] * sa, b = x[j + 1] * c[j + 1] + x[j] * sb;
        if (j < left) { y[j] = a; y[j + 1] = b; }
    }
    return y;
}

}  // namespace
