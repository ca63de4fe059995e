// What the kernels over sequences of tokens share (gfx950).
#ifndef SPIO_TOKENS_H
#define SPIO_TOKENS_H
#include "spio_pointwise.h"
#include "spio_token_args.h"

namespace tk {

#if SPIO_DTYPE == 0
typedef _Float16 value_t;
#elif SPIO_DTYPE == 1
typedef __bf16 value_t;
#else
typedef float value_t;
#endif

constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

__device__ inline void barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

__device__ inline float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// The value of another lane of the row of 16: 0xB1 lane ^ 1, 0x4E lane ^ 2, 0x141 the mirrored lane of eight, 0x128 lane ^ 8
template <int CTRL>
__device__ inline float from(float v) {
    return pw::as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)pw::as_bits(v), CTRL, 0xf, 0xf, false));
}
// The sum over LANES neighbouring lanes (a power of two up to 16), in all of them
template <int LANES>
__device__ inline float sum_of(float v) {
    if (LANES >= 2) v += from<0xB1>(v);
    if (LANES >= 4) v += from<0x4E>(v);
    if (LANES >= 8) v += from<0x141>(v);
    if (LANES >= 16) v += from<0x128>(v);
    return v;
}

// Eight values that follow each other, on 16 bytes
__device__ inline pw::Unit load(const value_t* p) {
    pw::Unit u;
#pragma unroll
    for (int i = 0; i < pw::QUADS; ++i) u.q[i] = ((const pw_uint4*)p)[i];
    return u;
}
// ONCE: past the caches, for whole lines that nobody reads soon
template <bool ONCE>
__device__ inline void store(value_t* p, const pw::Unit& u) {
#pragma unroll
    for (int i = 0; i < pw::QUADS; ++i) {
        if (ONCE)
            __builtin_nontemporal_store(u.q[i], (pw_uint4*)p + i);
        else
            ((pw_uint4*)p)[i] = u.q[i];
    }
}
__device__ inline void values(const pw::Unit& u, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = pw::value(u, e);
}

// Sums over `rows` rows of float32 values [turned + rest][inner]: the first of them are stored as [inner][turned], the one or
// two [inner] behind these to `first` and `second`.
struct ColumnSums {
    const float* from;
    long long rows, inner, turned, rest;
    float *to, *first, *second;
};
// Partial sums added up: workgroup `group` of 256 threads takes 32 columns (a line of a row), 8 lanes each of which have
// every 8th row; in float64, since the rows may be many and their sums cancel.
constexpr int SUM_COLUMNS = 32;
__device__ inline void column_sums(const ColumnSums& a, long long group) {
    constexpr int LANES = 256 / SUM_COLUMNS;
    __shared__ double parts[LANES][SUM_COLUMNS];
    const int tid = (int)__builtin_amdgcn_workitem_id_x();
    const long long columns = (a.turned + a.rest) * a.inner;
    const long long column = group * SUM_COLUMNS + tid % SUM_COLUMNS;
    double sum = 0.;
    if (column < columns) {
#pragma unroll 8
        for (long long i = tid / SUM_COLUMNS; i < a.rows; i += LANES) sum += a.from[i * columns + column];
    }
    parts[tid / SUM_COLUMNS][tid % SUM_COLUMNS] = sum;
    barrier();
    if (tid >= SUM_COLUMNS || column >= columns) return;
    sum = 0.;
#pragma unroll
    for (int i = 0; i < LANES; ++i) sum += parts[i][tid];
    const long long k = column / a.inner, c = column % a.inner;
    *(k < a.turned ? a.to + c * a.turned + k : (k == a.turned ? a.first : a.second) + c) = (float)sum;
}

}  // namespace tk

#endif
