// Group norm with an activation over NHWC tensors (gfx950).
//
//   mean, var [n][g]  of the pixels and the C/G channels of a group      (float32)
//   rstd = rsqrt(var + eps)
//   out = act((in - mean) * rstd * weight[c] + bias[c])                  weight and bias float32, optional
//   stats[n][g] = mean, rstd (optional); codes, exponents = in in the 8-bit form (SPIO_GN_KEPT)
//
// The variance is that of the differences to the mean, never the difference of two large sums: a workgroup holds its
// pixels in registers and goes over them twice.
//
// HBM-bound: a value is read and written once where an image's slice of channels fits the registers of one
// workgroup (SPIO_GN_SPLIT 0: one launch).  Otherwise (SPIO_GN_SPLIT 1) images are cut into stretches: one launch
// leaves mean and sum of squared differences of every stretch and group, the second one combines them, in the
// same order always, while its own loads are on their way, and reads the input again, mostly from the memory-side cache.
#include "spio_group_norm.h"

namespace {

using namespace gn;

struct Chunk {
    pw::Unit v[UN];
    unsigned off[UN];
    int pixels;         // of the stretch from its first on
    long long first;    // pixel of the tensor that the offsets start from
};

template <int POLICY>
PW_DEVICE void load_chunk(Chunk& c, const void* in, const Place& p, long long pixels) {
    const long long begin = SPIO_GN_SPLIT ? (long long)p.stretch * SPAN : 0;
    const long long left = pixels - begin;
    c.pixels = (int)(left < SPAN ? left : SPAN);
    c.first = p.image * pixels + begin;
    const pw_rsrc rs = pw::buffer(reinterpret_cast<const unsigned char*>(in) + c.first * (C * pw::VALUE_BYTES),
                                  (unsigned)c.pixels * (C * pw::VALUE_BYTES));
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int pixel = p.row + u * ROWS;
        c.off[u] = p.live ? (unsigned)(pixel * C + p.channel) * pw::VALUE_BYTES : pw::OOB;
        c.v[u] = pw::load_unit<POLICY>(rs, c.off[u]);
    }
}

// mean[] and squares[] (sum of squared differences to it) of the groups of a chunk.
PW_DEVICE void moments(const Chunk& c, const Place& p, float* red, float* mean, float* squares) {
    float s[KEYS] = {};
#pragma unroll
    for (int u = 0; u < UN; ++u) {  // what lies behind the last pixel is zero
        float x[8];
        pw::unpack(x, c.v[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e / KEY_CHANNELS] += x[e];
    }
    group_sums(s, p, red, mean);
    const float count = 1.f / ((float)c.pixels * CG);
    float m[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        m[k] = mean[group_of(p, k) < GS ? group_of(p, k) : 0] * count;
        s[k] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        if (p.live && p.row + u * ROWS < c.pixels) {
            float x[8];
            pw::unpack(x, c.v[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = x[e] - m[e / KEY_CHANNELS];
                s[e / KEY_CHANNELS] = __builtin_fmaf(d, d, s[e / KEY_CHANNELS]);
            }
        }
    }
    group_sums(s, p, red, squares);
}

// out and the checkpoint of a chunk, from the lanes' means and rstds by key
PW_DEVICE void apply(const Chunk& c, const Place& p, void* out, unsigned char* codes, unsigned char* exponents,
                     const float (&mean)[KEYS], const float (&rstd)[KEYS], const float (&w)[8], const float (&b)[8]) {
    const unsigned bytes = (unsigned)c.pixels * (C * pw::VALUE_BYTES);
    const pw_rsrc rs_out = pw::buffer(reinterpret_cast<unsigned char*>(out) + c.first * (C * pw::VALUE_BYTES), bytes);
    const pw_rsrc rs_codes = pw::buffer(codes + c.first * C, SPIO_GN_KEPT ? (unsigned)c.pixels * C : 0);
    const pw_rsrc rs_exp = pw::buffer(exponents + c.first * BLOCKS, SPIO_GN_KEPT ? (unsigned)c.pixels * BLOCKS : 0);
    float scale[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) scale[e] = rstd[e / KEY_CHANNELS] * (SPIO_GN_HAS_WEIGHT ? w[e] : 1.f);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        float x[8], y[8];
        pw::unpack(x, c.v[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = x[e] - mean[e / KEY_CHANNELS];
            y[e] = pw::activate(SPIO_GN_HAS_BIAS ? __builtin_fmaf(d, scale[e], b[e]) : d * scale[e]);
        }
        pw::store_unit<pw::STREAM>(rs_out, c.off[u], pw::pack(y));
        if (SPIO_GN_KEPT) {
            const int pixel = p.row + u * ROWS;
            const unsigned ex = pw::block_exponent(c.v[u]);
            const pw_uint2 code = pw::encode(x, ex);
            __builtin_amdgcn_raw_buffer_store_b64(code, rs_codes, p.live ? pixel * C + p.channel : (int)pw::OOB, 0, pw::STREAM);
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)ex, rs_exp,
                                                 p.live && p.tid % 4 == 0 ? pixel * BLOCKS + p.channel / 32 : (int)pw::OOB, 0, 0);
        }
    }
}

PW_DEVICE float inverse_deviation(float squares, long long pixels) {
    return __builtin_amdgcn_rsqf(squares * (1.f / ((float)pixels * CG)) + SPIO_GN_EPS);
}

}  // namespace

#define SPIO_GN_CONCAT2(a, b) a##b
#define SPIO_GN_CONCAT(a, b) SPIO_GN_CONCAT2(a, b)
#define SPIO_GN_KERNEL extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS)))

#if !SPIO_GN_SPLIT

SPIO_GN_KERNEL SPIO_KERNEL_NAME(void* __restrict__ out, unsigned char* __restrict__ codes,
                                unsigned char* __restrict__ exponents, float* __restrict__ stats,
                                const void* __restrict__ in, const float* __restrict__ weight,
                                const float* __restrict__ bias, long long pixels, long long) {
    __shared__ float red[RED_FLOATS], sum[GS], squares[GS];
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), 1);
    Chunk c;
    load_chunk<pw::STREAM>(c, in, p, pixels);
    float w[8] = {}, b[8] = {};
    if (SPIO_GN_HAS_WEIGHT) load_vector(w, weight, p);
    if (SPIO_GN_HAS_BIAS) load_vector(b, bias, p);
    moments(c, p, red, sum, squares);
    const float count = 1.f / ((float)pixels * CG);
    float mean[KEYS], rstd[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        const int g = group_of(p, k) < GS ? group_of(p, k) : 0;
        mean[k] = sum[g] * count;
        rstd[k] = inverse_deviation(squares[g], pixels);
    }
    if (stats)
        for (int g = p.tid; g < GS && p.slice * GS + g < GROUPS; g += THREADS) {
            float* s = stats + ((long long)p.image * GROUPS + p.slice * GS + g) * 2;
            s[0] = sum[g] * count;
            s[1] = inverse_deviation(squares[g], pixels);
        }
    apply(c, p, out, codes, exponents, mean, rstd, w, b);
}

#else

// partials[image][group][stretch] = mean, sum of squared differences
SPIO_GN_KERNEL SPIO_KERNEL_NAME(void*, unsigned char*, unsigned char*, float* __restrict__ partials,
                                const void* __restrict__ in, const float*, const float*, long long pixels, long long) {
    __shared__ float red[RED_FLOATS], sum[GS], squares[GS];
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), stretches);
    Chunk c;
    load_chunk<0>(c, in, p, pixels);
    moments(c, p, red, sum, squares);
    const float count = 1.f / ((float)c.pixels * CG);
    for (int g = p.tid; g < GS && p.slice * GS + g < GROUPS; g += THREADS) {
        float* s = partials + (((long long)p.image * GROUPS + p.slice * GS + g) * stretches + p.stretch) * 2;
        s[0] = sum[g] * count;
        s[1] = squares[g];
    }
}

SPIO_GN_KERNEL SPIO_GN_CONCAT(SPIO_KERNEL_NAME, _apply)(
    float* __restrict__ stats, const float* __restrict__ partials, void* __restrict__ out,
    unsigned char* __restrict__ codes, unsigned char* __restrict__ exponents, const void* __restrict__ in,
    const float* __restrict__ weight, const float* __restrict__ bias, long long pixels, long long images) {
    __shared__ float means[GS], rstds[GS];
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    // the last stretches first: the first launch read them last
    const Place p = place((unsigned)images * stretches * SLICES - 1 - __builtin_amdgcn_workgroup_id_x(), stretches);
    Chunk c;
    load_chunk<pw::STREAM>(c, in, p, pixels);
    float w[8] = {}, b[8] = {};
    if (SPIO_GN_HAS_WEIGHT) load_vector(w, weight, p);
    if (SPIO_GN_HAS_BIAS) load_vector(b, bias, p);

    // The lanes of a wave share a group's stretches; sets of n values with means m and squares q join as
    // n = n1 + n2, m = m1 + (m2 - m1) n2/n, q = q1 + q2 + (m2 - m1)^2 n1 n2/n.
    constexpr int LANES = group_lanes();
    const int part = p.tid % LANES;
    for (int g = p.tid / LANES; g < GS; g += THREADS / LANES) {
        float n = 0.f, m = 0.f, q = 0.f;
        auto join = [&](float n2, float m2, float q2) {
            const float total = n + n2, share = total > 0.f ? n2 / total : 0.f, d = m2 - m;
            q += q2 + d * d * n * share;
            m += d * share;
            n = total;
        };
        if (p.slice * GS + g < GROUPS) {
            const float* s = partials + ((long long)p.image * GROUPS + p.slice * GS + g) * stretches * 2;
            for (unsigned i = part; i < stretches; i += LANES) {
                const long long left = pixels - (long long)i * SPAN;
                join((float)(left < SPAN ? left : SPAN) * CG, s[2 * i], s[2 * i + 1]);
            }
        }
        // (both lanes of a pair come to the same sums but for their order: the lower one's is passed on in the end)
#pragma unroll
        for (int step = 1; step < LANES; step <<= 1) {
            const float n2 = lane_xor(n, step), m2 = lane_xor(m, step), q2 = lane_xor(q, step);
            join(n2, m2, q2);
        }
        if (part == 0) {
            means[g] = m;
            rstds[g] = inverse_deviation(q, pixels);
            if (stats && p.stretch == 0 && p.slice * GS + g < GROUPS) {
                float* s = stats + ((long long)p.image * GROUPS + p.slice * GS + g) * 2;
                s[0] = m;
                s[1] = rstds[g];
            }
        }
    }
    sync();
    float mean[KEYS], rstd[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        const int g = group_of(p, k) < GS ? group_of(p, k) : 0;
        mean[k] = means[g];
        rstd[k] = rstds[g];
    }
    apply(c, p, out, codes, exponents, mean, rstd, w, b);
}

#endif
