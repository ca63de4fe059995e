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
// A value is read and written once where an image's slice of channels fits the registers of one workgroup (SPIO_GN_SPLIT 0:
// one launch).  128n 768c 7x7 without activation takes 6.1 us for 19 MB, 3 of which any launch and its first load take;
// 32n 192c 28x28 float32 with silu 11.6 us for 39 MB: 192 workgroups hold an image's slice each, all load at once, and none
// stores before its last value has come.
//
// Otherwise (SPIO_GN_SPLIT 1) images are cut into stretches: one launch leaves mean and sum of squared differences of
// every stretch and group, the second one combines them, in the same order always, while its own first loads are on
// their way, and reads the input again.  32n 48c 224x224 with silu: 27.8 us for 155 MB (5.6 TB/s) and 44.4 us for 309 MB (7.0
// TB/s, part of it from the memory-side cache), where one pass would be 52 us at the rate of a copy.  Workgroups of
// an image that hold their stretches and exchange sums through memory need no second read, but wait for each other: 79.5
// us where the pair took 73 to 78.  The second launch issues vector instructions for 75 % of that time (86 % where it writes 8
// bits too: 128n 96c 56x56 16.3 and 28.6 us): rounding, packing and the activation are what it has besides its loads.
//
// Loads: the first launch's leave lines in the caches for the second, whose own and whose stores are streamed (plain
// stores take the pair 10 to 25 % longer); the second launch has DEPTH units a lane under way, the first all of them.
#include "spio_group_norm.h"

namespace {

using namespace gn;

constexpr unsigned STEP = (unsigned)(ROWS * C) * pw::VALUE_BYTES;

// A stretch of an image (all of it where images are whole)
struct Stretch {
    int pixels;         // from its first on
    unsigned off;       // of the lane's first unit; the others follow STEP apart
    long long first;    // pixel of the tensors that the offsets start from
    pw_rsrc in;
};

PW_DEVICE Stretch stretch_of(const void* in, const Place& p, long long pixels) {
    const long long begin = SPIO_GN_SPLIT ? (long long)p.stretch * SPAN : 0;
    const long long left = pixels - begin;
    Stretch s;
    s.pixels = (int)(left < SPAN ? left : SPAN);
    s.first = p.image * pixels + begin;
    s.off = p.live ? (unsigned)(p.row * C + p.channel) * pw::VALUE_BYTES : pw::OOB;
    s.in = pw::buffer(reinterpret_cast<const unsigned char*>(in) + s.first * (C * pw::VALUE_BYTES),
                      (unsigned)s.pixels * (C * pw::VALUE_BYTES));
    return s;
}

// Units [0, COUNT) of it
template <int COUNT, int POLICY>
PW_DEVICE void load_units(pw::Unit (&v)[COUNT], const Stretch& s) {
#pragma unroll
    for (int u = 0; u < COUNT; ++u) v[u] = pw::load_unit<POLICY>(s.in, s.off + u * STEP);
}
PW_DEVICE void keep_packed(pw::Unit (&v)[UN]) {
#pragma unroll
    for (int u = 0; u < UN; ++u) pw::keep_packed(v[u]);
}

// The mean of a group from its sum over that many pixels
PW_DEVICE float mean_of(float sum, int pixels) {
    const float count = (float)pixels * CG;
    return pw::quotient(sum, count, pw::reciprocal(count));
}

// mean[] = sums and squares[] = sums of squared differences to the means of the groups of a stretch.
PW_DEVICE void moments(pw::Unit (&v)[UN], const Stretch& c, const Place& p, const pw::Constants& k, float* red,
                       float* mean, float* squares) {
    float s[KEYS] = {};
#pragma unroll
    for (int u = 0; u < UN; ++u) {  // what lies behind the last pixel is zero
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e / KEY_CHANNELS] = pw::plus(v[u], e, s[e / KEY_CHANNELS], k);
#pragma unroll
        for (int i = 0; i < KEYS; ++i) asm volatile("" : "+v"(s[i]));  // a unit is worked on when it is there, not when all are
    }
    group_sums(s, p, red, mean);
    keep_packed(v);
    float m[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        m[i] = mean_of(mean[group_of(p, i) < GS ? group_of(p, i) : 0], c.pixels);
        s[i] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        if (p.live && p.row + u * ROWS < c.pixels) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = pw::plus(v[u], e, -m[e / KEY_CHANNELS], k);
                s[e / KEY_CHANNELS] = __builtin_fmaf(d, d, s[e / KEY_CHANNELS]);
            }
        }
    }
    group_sums(s, p, red, squares);
    keep_packed(v);
}

// out and the checkpoint of a stretch, from the lanes' means and rstds by key.  `v` holds its first COUNT units; the others
// follow as these are done with.
template <int COUNT>
PW_DEVICE void apply(pw::Unit (&v)[COUNT], const Stretch& c, const Place& p, const pw::Constants& k, void* out,
                     unsigned char* codes, unsigned char* exponents, const float (&mean)[KEYS], const float (&rstd)[KEYS],
                     const float (&w)[8], const float (&b)[8]) {
    const unsigned bytes = (unsigned)c.pixels * (C * pw::VALUE_BYTES);
    const pw_rsrc rs_out = pw::buffer(reinterpret_cast<unsigned char*>(out) + c.first * (C * pw::VALUE_BYTES), bytes);
    const pw_rsrc rs_codes = pw::buffer(codes + c.first * C, SPIO_GN_KEPT ? (unsigned)c.pixels * C : 0);
    const pw_rsrc rs_exp = pw::buffer(exponents + c.first * EXP_ROW, SPIO_GN_KEPT ? (unsigned)c.pixels * EXP_ROW : 0);
    float scale[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) scale[e] = rstd[e / KEY_CHANNELS] * (SPIO_GN_HAS_WEIGHT ? w[e] : 1.f);
    // (the codes and exponents of lanes without any are stored behind the end of theirs)
    const unsigned off_codes = p.live ? (unsigned)(p.row * C + p.channel) : pw::OOB;
    const unsigned off_exp = p.live && p.tid % 4 == 0 ? (unsigned)(p.row * EXP_ROW + p.channel / 32) : pw::OOB;
    const unsigned off_bits = p.live ? (unsigned)(p.row * EXP_ROW + BLOCKS + p.channel / 8) : pw::OOB;
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const pw::Unit x = v[u % COUNT];
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = pw::plus(x, e, -mean[e / KEY_CHANNELS], k);
            y[e] = pw::activate(SPIO_GN_HAS_BIAS ? __builtin_fmaf(d, scale[e], b[e]) : d * scale[e]);
        }
        pw::store_unit<pw::STREAM>(rs_out, c.off + u * STEP, pw::pack(y));
        if (SPIO_GN_KEPT) {
            const unsigned ex = pw::block_exponent(x);
            __builtin_amdgcn_raw_buffer_store_b64(pw::encode(x, ex), rs_codes, (int)(off_codes + u * (ROWS * C)), 0, pw::STREAM);
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)ex, rs_exp, (int)(off_exp + u * (ROWS * EXP_ROW)), 0, 0);
        }
        if (kBits) {
            unsigned bits = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) bits |= pw::passes(y[e]) ? 1u << e : 0u;  // (relu of z passes where z does)
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)bits, rs_exp, (int)(off_bits + u * (ROWS * EXP_ROW)), 0, 0);
        }
        if (u + COUNT < UN) v[u % COUNT] = pw::load_unit<pw::STREAM>(c.in, c.off + (u + COUNT) * STEP);
        __builtin_amdgcn_sched_barrier(0);
    }
}

PW_DEVICE float inverse_deviation(float squares, long long pixels) {
    return __builtin_amdgcn_rsqf(squares * (pw::reciprocal((float)(unsigned)pixels * CG)) + SPIO_GN_EPS);
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
    const pw::Constants k;
    const Stretch c = stretch_of(in, p, pixels);
    pw::Unit v[UN];
    load_units<UN, pw::STREAM>(v, c);
    float w[8] = {}, b[8] = {};
    if (SPIO_GN_HAS_WEIGHT) load_vector(w, weight, p);
    if (SPIO_GN_HAS_BIAS) load_vector(b, bias, p);
    moments(v, c, p, k, red, sum, squares);
    float mean[KEYS], rstd[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const int g = group_of(p, i) < GS ? group_of(p, i) : 0;
        mean[i] = mean_of(sum[g], c.pixels);
        rstd[i] = inverse_deviation(squares[g], pixels);
    }
    if (stats)
        for (int g = p.tid; g < GS && p.slice * GS + g < GROUPS; g += THREADS) {
            float* s = stats + ((long long)p.image * GROUPS + p.slice * GS + g) * 2;
            s[0] = mean_of(sum[g], c.pixels);
            s[1] = inverse_deviation(squares[g], pixels);
        }
    apply(v, c, p, k, out, codes, exponents, mean, rstd, w, b);
}

#else

// partials[image][group][stretch] = mean, sum of squared differences
SPIO_GN_KERNEL SPIO_KERNEL_NAME(void*, unsigned char*, unsigned char*, float* __restrict__ partials,
                                const void* __restrict__ in, const float*, const float*, long long pixels, long long) {
    __shared__ float red[RED_FLOATS], sum[GS], squares[GS];
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), stretches);
    const pw::Constants k;
    const Stretch c = stretch_of(in, p, pixels);
    pw::Unit v[UN];
    load_units<UN, 0>(v, c);
    moments(v, c, p, k, red, sum, squares);
    for (int g = p.tid; g < GS && p.slice * GS + g < GROUPS; g += THREADS) {
        float* s = partials + (((long long)p.image * GROUPS + p.slice * GS + g) * stretches + p.stretch) * 2;
        s[0] = mean_of(sum[g], c.pixels);
        s[1] = squares[g];
    }
}

SPIO_GN_KERNEL SPIO_GN_CONCAT(SPIO_KERNEL_NAME, _apply)(
    float* __restrict__ stats, const float* __restrict__ partials, void* __restrict__ out,
    unsigned char* __restrict__ codes, unsigned char* __restrict__ exponents, const void* __restrict__ in,
    const float* __restrict__ weight, const float* __restrict__ bias, long long pixels, long long) {
    __shared__ float means[GS], rstds[GS];
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), stretches);
    const pw::Constants k;
    const Stretch c = stretch_of(in, p, pixels);
    pw::Unit v[DEPTH];
    load_units<DEPTH, pw::STREAM>(v, c);
    float w[8] = {}, b[8] = {};
    if (SPIO_GN_HAS_WEIGHT) load_vector(w, weight, p);
    if (SPIO_GN_HAS_BIAS) load_vector(b, bias, p);

    // The lanes of a wave share a group's stretches; sets of n values with means m and squares q join as
    // n = n1 + n2, m = m1 + (m2 - m1) n2/n, q = q1 + q2 + (m2 - m1)^2 n1 n2/n.  Where one is empty there is no difference:
    // that to its mean of zero would be the other's mean, whose square may overflow.
    constexpr int LANES = group_lanes();
    const int part = p.tid % LANES;
    for (int g = p.tid / LANES; g < GS; g += THREADS / LANES) {
        float n = 0.f, m = 0.f, q = 0.f;
        auto join = [&](float n2, float m2, float q2) {
            const bool empty = n == 0.f;
            const float total = n + n2, share = total > 0.f ? n2 * pw::reciprocal(total) : 0.f;
            const float d = empty || n2 == 0.f ? 0.f : m2 - m;
            q += q2 + d * d * n * share;
            m = empty ? m2 : __builtin_fmaf(d, share, m);
            n = total;
        };
        if (p.slice * GS + g < GROUPS) {
            const float* s = partials + ((long long)p.image * GROUPS + p.slice * GS + g) * stretches * 2;
            for (unsigned first = part; first < stretches; first += LANES * 4) {  // four loads under way
                float m2[4], q2[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned i = first + j * LANES;
                    m2[j] = i < stretches ? s[2 * i] : 0.f;
                    q2[j] = i < stretches ? s[2 * i + 1] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // (images have less than 2^31 pixels.  A conversion of 64 bits would shift by a register, which this
                    // hardware gets wrong where that is a wave's last one: a stretch of 240 values then counted as one.)
                    const unsigned before = (first + j * LANES) * SPAN;
                    const unsigned left = before < (unsigned)pixels ? (unsigned)pixels - before : 0u;
                    join((float)(left < SPAN ? left : SPAN) * CG, m2[j], q2[j]);
                }
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
    for (int i = 0; i < KEYS; ++i) {
        const int g = group_of(p, i) < GS ? group_of(p, i) : 0;
        mean[i] = means[g];
        rstd[i] = rstds[g];
    }
    apply(v, c, p, k, out, codes, exponents, mean, rstd, w, b);
}

#endif
