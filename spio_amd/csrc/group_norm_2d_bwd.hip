// Backward of the group norm with an activation of group_norm_2d.hip (NHWC tensors, gfx950).
//
//   xhat = (in - mean) * rstd          mean and rstd of the forward pass; in as it was, or its 8-bit form (SPIO_GN_KEPT)
//   dz = dout * act'(xhat * weight + bias),  g = dz * weight,  m = pixels * C/G
//   din = rstd * (g - sum_group(g) / m - xhat * sum_group(g * xhat) / m)
//   dweight[c] = sum dz * xhat,  dbias[c] = sum dz          float32, over images and pixels
//
// The group's sums are those of its channels times their weights, so one pair of sums for each image and channel
// serves all three gradients.  Where an image's slice of channels fits the registers of one workgroup (SPIO_GN_SPLIT 0)
// input and gradient are read once, and a second launch adds the images' rows of channel sums: 128n 768c 7x7 without
// activation 7.4 us for 30 MB and 2.9, 32n 192c 28x28 float32 with silu 16.3 us for 59 MB and 3.9.  (Its few workgroups walk all
// rows: 4096n 64c 8x8 takes 20.6 us and 28.0.)
//
// Otherwise the first launch leaves a row of channel sums for every stretch and the pair of each group; the second one
// reads input and gradient again, and its first workgroups add the rows meanwhile (as a launch of its own that takes 3
// us).  128n 96c 56x56 with silu from 8 bits: 27.7 us for 121 MB and 32.8 us for 198 MB (6.0 TB/s).  Both issue vector
// instructions for 81 to 86 % of their time: a value costs 15 or 16 of them in either launch, an exp and a rcp among them,
// which count fourfold.  One launch whose workgroups exchange sums through memory waits more than it saves
// (32n 48c 224x224 148 to 165 us against 125 to 144).  Nothing is atomic: every sum is made in the same order always.
#include "spio_group_norm.h"

#ifndef SPIO_GN_AFFINE
#define SPIO_GN_AFFINE 1  // the sums over images are wanted
#endif

namespace {

using namespace gn;

struct Inputs {  // a unit of the norm's input, as the backward pass has it, and of grad_output
#if SPIO_GN_KEPT
    pw_uint2 code;
    unsigned exponent, bits;
#else
    pw::Unit x;
#endif
    pw::Unit dy;
};

constexpr unsigned STEP = (unsigned)(ROWS * C) * pw::VALUE_BYTES;

// A stretch of an image (all of it where images are whole)
struct Stretch {
    int pixels;         // from its first on
    unsigned off;       // of the lane's first unit; the others follow STEP apart
    unsigned off_codes, off_exp, off_bits;
    long long first;    // pixel of the tensors that the offsets start from
    pw_rsrc in, exponents, dout;
};

PW_DEVICE Stretch stretch_of(const void* in, const unsigned char* exponents, const void* dout, const Place& p,
                             long long pixels) {
    const long long begin = SPIO_GN_SPLIT ? (long long)p.stretch * SPAN : 0;
    const long long left = pixels - begin;
    constexpr int IN_BYTES = SPIO_GN_KEPT ? 1 : pw::VALUE_BYTES;
    Stretch s;
    s.pixels = (int)(left < SPAN ? left : SPAN);
    s.first = p.image * pixels + begin;
    s.off = p.live ? (unsigned)(p.row * C + p.channel) * pw::VALUE_BYTES : pw::OOB;
    s.off_codes = p.live ? (unsigned)(p.row * C + p.channel) : pw::OOB;
    s.off_exp = p.live ? (unsigned)(p.row * EXP_ROW + p.channel / 32) : pw::OOB;
    s.off_bits = p.live ? (unsigned)(p.row * EXP_ROW + BLOCKS + p.channel / 8) : pw::OOB;
    s.in = pw::buffer(reinterpret_cast<const unsigned char*>(in) + s.first * (C * IN_BYTES), (unsigned)s.pixels * (C * IN_BYTES));
    s.exponents = pw::buffer(exponents + s.first * EXP_ROW, SPIO_GN_KEPT ? (unsigned)s.pixels * EXP_ROW : 0);
    s.dout = pw::buffer(reinterpret_cast<const unsigned char*>(dout) + s.first * (C * pw::VALUE_BYTES),
                        (unsigned)s.pixels * (C * pw::VALUE_BYTES));
    return s;
}

template <int POLICY>
PW_DEVICE Inputs load_inputs(const Stretch& s, int u) {
    Inputs in;
#if SPIO_GN_KEPT
    in.code = __builtin_amdgcn_raw_buffer_load_b64(s.in, (int)(s.off_codes + u * (ROWS * C)), 0, POLICY);
    in.exponent = __builtin_amdgcn_raw_buffer_load_b8(s.exponents, (int)(s.off_exp + u * (ROWS * EXP_ROW)), 0, 0);
    if (kBits) in.bits = __builtin_amdgcn_raw_buffer_load_b8(s.exponents, (int)(s.off_bits + u * (ROWS * EXP_ROW)), 0, 0);
#else
    in.x = pw::load_unit<POLICY>(s.in, s.off + u * STEP);
#endif
    in.dy = pw::load_unit<POLICY>(s.dout, s.off + u * STEP);
    return in;
}

// How many of a stretch's units a lane has in registers: all where it works on them twice, else DEPTH, each replaced
// by the next as soon as it is done with: a lane needs no more registers for a longer stretch.
constexpr int HELD = SPIO_GN_SPLIT ? DEPTH : UN;
// ... with dz in place of grad_output: that takes more registers, but an activation's derivative takes more
// instructions than all the rest of the second pass (silu, us: 128n 384c 14x14 16.8 -> 14.7, 64n 128c 28x28 17.3 -> 13.8).
constexpr bool kHoldsDz = !SPIO_GN_SPLIT && SPIO_ACT;

template <int POLICY>
PW_DEVICE void load_first(Inputs (&in)[HELD], const Stretch& s) {
#pragma unroll
    for (int u = 0; u < HELD; ++u) in[u] = load_inputs<POLICY>(s, u);
}
// The next one in place of one that is done with
template <int POLICY>
PW_DEVICE void load_next(Inputs (&in)[HELD], const Stretch& s, int u) {
    if (u + HELD < UN) in[u % HELD] = load_inputs<POLICY>(s, u + HELD);
    __builtin_amdgcn_sched_barrier(0);  // a unit is worked on when it is there, not when all are
}

PW_DEVICE void keep_packed(Inputs (&in)[HELD]) {
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
#if SPIO_GN_KEPT
        asm volatile("" : "+v"(in[u].code), "+v"(in[u].exponent));
#else
        pw::keep_packed(in[u].x);
#endif
        if (!kHoldsDz) pw::keep_packed(in[u].dy);
    }
}

struct Lane {  // a lane's eight channels: z = (x - mean) * scale + bias
    float w[8], scale[8], b[8];
    float mean[KEYS], rstd[KEYS];
    pw::Constants k;
};

PW_DEVICE void load_lane(Lane& l, const float* stats, const float* weight, const float* bias, const Place& p) {
    if (SPIO_GN_HAS_WEIGHT)
        load_vector(l.w, weight, p);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) l.w[e] = 1.f;
    if (SPIO_GN_HAS_BIAS && SPIO_ACT)
        load_vector(l.b, bias, p);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) l.b[e] = 0.f;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const int g = p.slice * GS + group_of(p, i);
        const float* s = stats + ((long long)p.image * GROUPS + (p.live ? g : 0)) * 2;
        l.mean[i] = s[0];
        l.rstd[i] = s[1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) l.scale[e] = l.w[e] * l.rstd[e / KEY_CHANNELS];
}

// x - mean and dz of a unit (what lies behind the last pixel has dy = 0, and with it dz)
PW_DEVICE void centre(float (&d)[8], const Inputs& in, const Lane& l) {
#if SPIO_GN_KEPT
    const float step = pw::block_step(in.exponent);
#endif
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#if SPIO_GN_KEPT
        d[e] = __builtin_fmaf(pw::code(in.code, e), step, -l.mean[e / KEY_CHANNELS]);
#else
        d[e] = pw::plus(in.x, e, -l.mean[e / KEY_CHANNELS], l.k);
#endif
    }
}
PW_DEVICE void work(float (&d)[8], float (&dz)[8], const Inputs& in, const Lane& l) {
    centre(d, in, l);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#if SPIO_GN_KEPT
        if (kBits) {
            dz[e] = in.bits >> e & 1 ? pw::value(in.dy, e) : 0.f;
            continue;
        }
#endif
        const float z = SPIO_GN_HAS_BIAS ? __builtin_fmaf(d[e], l.scale[e], l.b[e]) : d[e] * l.scale[e];
        dz[e] = pw::activate_grad<false>(in.dy, e, z, l.k);
    }
}

// The stretch's sums of dz and of dz * xhat: [which][channel of the slice] in `red`, and in `row`, those of dz * xhat first.
constexpr int WIDTH = SUP * 8;
constexpr int COLUMNS = 2 * WIDTH;
constexpr int PARTS = THREADS / COLUMNS > 1 ? THREADS / COLUMNS : 1;  // threads that share a column
constexpr int RED = SUM_ROWS * COLUMNS > PARTS * COLUMNS ? SUM_ROWS * COLUMNS : PARTS * COLUMNS;

template <int POLICY>
PW_DEVICE void channel_sums(Inputs (&in)[HELD], float (&held)[UN][8], const Stretch& c, const Place& p, const Lane& l,
                            float* red, float* row) {
    float s1[8] = {}, s2[8] = {};
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        float d[8], dz[8];
        work(d, dz, in[u % HELD], l);
        if (kHoldsDz)
#pragma unroll
            for (int e = 0; e < 8; ++e) held[u][e] = dz[e];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s1[e] += dz[e];
            s2[e] = __builtin_fmaf(dz[e], d[e], s2[e]);
            asm volatile("" : "+v"(s1[e]), "+v"(s2[e]));  // (now: all units' sums would be put off behind the last load)
        }
        load_next<POLICY>(in, c, u);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s2[e] *= l.rstd[e / KEY_CHANNELS];
    if (!SPIO_GN_SPLIT) keep_packed(in);
    if (kFold) {
#pragma unroll
        for (int m = SUP; m < 64; m <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s1[e] += lane_xor(s1[e], m);
                s2[e] += lane_xor(s2[e], m);
            }
    }
    if (kFold ? (p.tid & 63) < SUP : p.row < ROWS) {
        float* to = red + (kFold ? p.tid >> 6 : p.row) * COLUMNS + p.sub * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            to[e] = s1[e];
            to[WIDTH + e] = s2[e];
        }
    }
    sync();
    // a column's rows by PARTS threads, then those
    float sum[(COLUMNS + THREADS - 1) / THREADS];
#pragma unroll
    for (int i = 0; i < (COLUMNS + THREADS - 1) / THREADS; ++i) {
        sum[i] = 0.f;
        const int col = PARTS > 1 ? p.tid % COLUMNS : p.tid + i * THREADS;
        const int part = PARTS > 1 ? p.tid / COLUMNS : 0;
        if (col < COLUMNS && part < PARTS)
            for (int r = part; r < SUM_ROWS; r += PARTS) sum[i] += red[r * COLUMNS + col];
    }
    if (PARTS > 1) {
        sync();
        if (p.tid / COLUMNS < PARTS) red[p.tid] = sum[0];
        sync();
        if (p.tid < COLUMNS) {
#pragma unroll
            for (int q = 1; q < PARTS; ++q) sum[0] += red[q * COLUMNS + p.tid];
        }
    }
    sync();
#pragma unroll
    for (int i = 0; i < (COLUMNS + THREADS - 1) / THREADS; ++i) {
        const int col = p.tid + i * THREADS;
        if (col < COLUMNS) {
            red[col] = sum[i];
            const int channel = p.slice * SLICE + col % WIDTH;
            if (SPIO_GN_AFFINE && col % WIDTH < SLICE && channel < C) row[(1 - col / WIDTH) * C + channel] = sum[i];
        }
    }
    sync();
}

// The pairs of sums of the slice's groups, from the channel sums that channel_sums left in `red`.
PW_DEVICE void group_pairs(const Place& p, const float* red, float* pairs, const float* weight) {
    constexpr int LANES = group_lanes();
    const int part = p.tid % LANES;
    for (int g = p.tid / LANES; g < GS; g += THREADS / LANES) {
        float a = 0.f, b = 0.f;
        for (int e = part; e < CG; e += LANES) {
            const int col = g * CG + e;
            const int channel = p.slice * SLICE + col;
            const float w = SPIO_GN_HAS_WEIGHT && channel < C ? weight[channel] : 1.f;
            a = __builtin_fmaf(red[col], w, a);
            b = __builtin_fmaf(red[WIDTH + col], w, b);
        }
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) {
            a += lane_xor(a, m);
            b += lane_xor(b, m);
        }
        if (part == 0) {
            pairs[g] = a;
            pairs[GS + g] = b;
        }
    }
    sync();
}

PW_DEVICE void apply(Inputs (&in)[HELD], const float (&held)[UN][8], const Stretch& c, const Place& p, const Lane& l,
                     void* din, const float* pairs, long long pixels) {
    const pw_rsrc rs = pw::buffer(reinterpret_cast<unsigned char*>(din) + c.first * (C * pw::VALUE_BYTES),
                                  (unsigned)c.pixels * (C * pw::VALUE_BYTES));
    const float count = pw::reciprocal((float)(unsigned)pixels * CG);
    // rstd * (dz * w - m1 - xhat * m2) = dz * scale + c1 + (x - mean) * c2
    float c1[KEYS], c2[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const int g = group_of(p, i) < GS ? group_of(p, i) : 0;
        c1[i] = -l.rstd[i] * (pairs[g] * count);
        c2[i] = -l.rstd[i] * l.rstd[i] * (pairs[GS + g] * count);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        float d[8], dz[8], dx[8];
        if (kHoldsDz) {
            centre(d, in[u % HELD], l);
#pragma unroll
            for (int e = 0; e < 8; ++e) dz[e] = held[u][e];
        } else {
            work(d, dz, in[u % HELD], l);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = e / KEY_CHANNELS;
            dx[e] = __builtin_fmaf(dz[e], l.scale[e], __builtin_fmaf(d[e], c2[i], c1[i]));
        }
        pw::store_unit<pw::STREAM>(rs, c.off + u * STEP, pw::pack(dx));
        load_next<pw::STREAM>(in, c, u);
    }
}

// sums[i] = sum over `rows` rows of rows[row][i], i < 2 * C: workgroup `block` has 32 columns, THREADS / 32 slices of
// rows, which meet in LDS.  There may be as many rows as images and stretches: sixteen at a time are added in a tree of
// 32 bits, and these sums in 64.  (In 32 bits a chain of 8192 equal terms was off by 2^-13.7.)
PW_DEVICE void add_rows(float* sums, const float* table, long long rows, int block, double* red) {
    constexpr int PARTS_OF_ROWS = THREADS / 32;
    const int tid = (int)__builtin_amdgcn_workitem_id_x();
    const int col = block * 32 + tid % 32, part = tid / 32;
    double s = 0.;
    if (col < 2 * C) {
        for (long long r = part; r < rows; r += PARTS_OF_ROWS * 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const long long row = r + i * PARTS_OF_ROWS;
                v[i] = row < rows ? table[row * (2 * C) + col] : 0.f;
            }
#pragma unroll
            for (int step = 8; step; step /= 2)
#pragma unroll
                for (int i = 0; i < step; ++i) v[i] += v[i + step];
            s += (double)v[0];
        }
    }
    red[tid] = s;
    sync();
    if (part == 0 && col < 2 * C) {
        for (int i = 1; i < PARTS_OF_ROWS; ++i) s += red[i * 32 + tid];
        sums[col] = (float)s;
    }
}
constexpr int ADDING = SPIO_GN_AFFINE ? (2 * C + 31) / 32 : 0;  // workgroups that add the rows

}  // namespace

#define SPIO_GN_CONCAT2(a, b) a##b
#define SPIO_GN_CONCAT(a, b) SPIO_GN_CONCAT2(a, b)
#define SPIO_GN_KERNEL extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS)))

#if !SPIO_GN_SPLIT

// rows[image][2][C]: 0 = grad_weight's, 1 = grad_bias's
SPIO_GN_KERNEL SPIO_KERNEL_NAME(float* __restrict__ rows, void* __restrict__ din, const void* __restrict__ in,
                                const unsigned char* __restrict__ exponents, const void* __restrict__ dout,
                                const float* __restrict__ stats, const float* __restrict__ weight,
                                const float* __restrict__ bias, long long pixels, long long) {
    __shared__ float red[RED], pairs[2 * GS];
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), 1);
    const Stretch c = stretch_of(in, exponents, dout, p, pixels);
    Inputs units[HELD];
    load_first<pw::STREAM>(units, c);
    float dz[UN][8];
    Lane l;
    load_lane(l, stats, weight, bias, p);
    channel_sums<pw::STREAM>(units, dz, c, p, l, red, rows + (long long)p.image * (2 * C));
    group_pairs(p, red, pairs, weight);
    apply(units, dz, c, p, l, din, pairs, pixels);
}

#if SPIO_GN_AFFINE
SPIO_GN_KERNEL SPIO_GN_CONCAT(SPIO_KERNEL_NAME, _reduce)(float* __restrict__ sums, const float* __restrict__ rows,
                                                         long long images) {
    __shared__ double red[THREADS];
    add_rows(sums, rows, images, (int)__builtin_amdgcn_workgroup_id_x(), red);
}
#endif

#else

// rows[image][stretch][2][C], then pairs[image][2][group][stretch]
SPIO_GN_KERNEL SPIO_KERNEL_NAME(float* __restrict__ rows, void*, const void* __restrict__ in,
                                const unsigned char* __restrict__ exponents, const void* __restrict__ dout,
                                const float* __restrict__ stats, const float* __restrict__ weight,
                                const float* __restrict__ bias, long long pixels, long long images) {
    __shared__ float red[RED], pairs[2 * GS];
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    const Place p = place(__builtin_amdgcn_workgroup_id_x(), stretches);
    const Stretch c = stretch_of(in, exponents, dout, p, pixels);
    Inputs units[HELD];
    load_first<0>(units, c);
    float dz[UN][8];
    Lane l;
    load_lane(l, stats, weight, bias, p);
    channel_sums<0>(units, dz, c, p, l, red, rows + ((long long)p.image * stretches + p.stretch) * (2 * C));
    group_pairs(p, red, pairs, weight);
    float* out = rows + (SPIO_GN_AFFINE ? images * stretches * (2 * C) : 0);
    for (int i = p.tid; i < 2 * GS; i += THREADS) {
        const int g = p.slice * GS + i % GS;
        if (g < GROUPS) out[(((long long)p.image * 2 + i / GS) * GROUPS + g) * stretches + p.stretch] = pairs[i];
    }
}

SPIO_GN_KERNEL SPIO_GN_CONCAT(SPIO_KERNEL_NAME, _apply)(
    float* __restrict__ sums, const float* __restrict__ rows, void* __restrict__ din, const void* __restrict__ in,
    const unsigned char* __restrict__ exponents, const void* __restrict__ dout, const float* __restrict__ stats,
    const float* __restrict__ weight, const float* __restrict__ bias, long long pixels, long long images) {
    __shared__ union {
        float pairs[2 * GS];
        double rows[THREADS];
    } lds;
    float* const pairs = lds.pairs;
    const unsigned stretches = (unsigned)((pixels + SPAN - 1) / SPAN);
    const unsigned block = __builtin_amdgcn_workgroup_id_x();
    if (block < ADDING) {
        add_rows(sums, rows, images * stretches, (int)block, lds.rows);
        return;
    }
    const Place p = place(block - ADDING, stretches);
    const Stretch c = stretch_of(in, exponents, dout, p, pixels);
    Inputs units[HELD];
    load_first<pw::STREAM>(units, c);
    float dz[UN][8];
    Lane l;
    load_lane(l, stats, weight, bias, p);
    const float* parts = rows + (SPIO_GN_AFFINE ? images * stretches * (2 * C) : 0);
    constexpr int LANES = group_lanes();
    const int part = p.tid % LANES;
    for (int g = p.tid / LANES; g < GS; g += THREADS / LANES) {
        float a = 0.f, b = 0.f;
        if (p.slice * GS + g < GROUPS) {
            const float* s = parts + ((long long)p.image * 2 * GROUPS + p.slice * GS + g) * stretches;
            for (unsigned first = part; first < stretches; first += LANES * 4) {  // four loads under way
                float a4[4], b4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned i = first + j * LANES;
                    a4[j] = i < stretches ? s[i] : 0.f;
                    b4[j] = i < stretches ? s[(long long)GROUPS * stretches + i] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a += a4[j];
                    b += b4[j];
                }
            }
        }
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) {
            a += lane_xor(a, m);
            b += lane_xor(b, m);
        }
        if (part == 0) {
            pairs[g] = a;
            pairs[GS + g] = b;
        }
    }
    sync();
    apply(units, dz, c, p, l, din, pairs, pixels);
}

#endif
