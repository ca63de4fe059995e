// Causal convolution along the tokens of tokens-by-channels tensors, each channel with its own filter of W taps (gfx950):
//
//   z[t] = bias + sum_i weight[i] x[t - W + 1 + i],  y[t] = act(z[t])          (SPIO_ACT: none or silu)
//   dz[t] = dy[t] act'(z[t]),  dx[t] = sum_i weight[i] dz[t + W - 1 - i],  dweight[i] = sum_t dz[t] x[t - W + 1 + i]
//
//   SPIO_MODE 0  forward    before the first token: `before`, or zeros; the last W - 1 inputs go to `after`
//   SPIO_MODE 1  backward   z is computed again; sums over tokens as partial sums, a row for every slice of tokens
//   SPIO_MODE 2  sums       the partial sums added up
//   SPIO_MODE 3  step       one token of every sequence
//
// A lane has eight neighbouring channels (16 bytes of a 16-bit type) and walks along a slice of tokens with the last
// inputs, and backward the last dz, in registers, so that every tensor is read once but for the W - 1 tokens beside a
// slice.  Neighbouring lanes have neighbouring channels, then the next slice.  HBM-bound: 2 + 2 bytes a value forward,
// 2 + 2 + 2 backward for 16-bit types.  8n 2048l 2048c, four taps and silu in bfloat16: forward 28 us (5.0 TB/s), backward 44
// (5.4 TB/s; vector instructions issue in 79 % of it), sums 5; a prompt of 2051 tokens of 1536 channels 6.7, a token 2.2, which
// is what a launch takes.
#include "spio_tokens.h"

#ifndef SPIO_MODE
#error "SPIO_MODE, SPIO_WIDTH, SPIO_WDTYPE are required"
#endif

namespace {

using tk::value_t;
constexpr int W = SPIO_WIDTH, K = W - 1;
constexpr int U = SPIO_UNROLL;  // tokens requested at once

#if SPIO_WDTYPE == 0
typedef _Float16 weight_t;
#elif SPIO_WDTYPE == 1
typedef __bf16 weight_t;
#else
typedef float weight_t;
#endif

// Filters and biases of eight channels: they start on 16 bytes and are W + 1 units of eight values
__device__ inline void unit_of(const void* from, long long unit, float (&v)[8]) {
    const pw_uint4* p = (const pw_uint4*)((const weight_t*)from + unit * 8);
    typedef weight_t weight4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const weight4 w = ((const weight4*)p)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = (float)w[e];
    }
}
__device__ inline void filters(const SpioConv1dArgs& a, long long channel, float (&w)[W][8], float (&bias)[8]) {
    float all[W][8];
#pragma unroll
    for (int i = 0; i < W; ++i) unit_of(a.weight, channel / 8 * W + i, all[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bias[e] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i][e] = all[(e * W + i) / 8][(e * W + i) % 8];
    }
    if (a.bias) unit_of(a.bias, channel / 8, bias);
}

// The place of a lane: eight channels of a slice of a sequence
struct Place {
    long long sequence, channel, first, last, slice;
    bool live;
};
__device__ inline Place place(const SpioConv1dArgs& a) {
    Place p;
    const unsigned units = (unsigned)(a.channels / 8), slices = (unsigned)((a.tokens + a.slice - 1) / a.slice);
    const unsigned id = __builtin_amdgcn_workgroup_id_x() * 256 + __builtin_amdgcn_workitem_id_x();  // (fewer than 2^32)
    const unsigned rest = id / units;
    p.channel = id % units * 8;
    p.slice = rest % slices;
    p.sequence = rest / slices;
    p.live = p.sequence < a.sequences;
    p.first = p.slice * a.slice;
    p.last = p.first + a.slice < a.tokens ? p.first + a.slice : a.tokens;
    return p;
}
// Inputs of token t, which may be one before the first
__device__ inline void input_before(const SpioConv1dArgs& a, const Place& p, long long t, float (&v)[8]) {
    if (t >= 0) {
        tk::values(tk::load((const value_t*)a.x + (p.sequence * a.tokens + t) * a.x_row + p.channel), v);
    } else if (a.before) {
        tk::values(tk::load((const value_t*)a.before + (p.sequence * K + K + t) * a.channels + p.channel), v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
}

}  // namespace

#if SPIO_MODE == 0

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const SpioConv1dArgs a) {
    const Place p = place(a);
    if (!p.live) return;
    float w[W][8], bias[8], x[K + U][8];
    filters(a, p.channel, w, bias);
#pragma unroll
    for (int i = 0; i < K; ++i) input_before(a, p, p.first - K + i, x[i]);
    const value_t* in = (const value_t*)a.x + p.sequence * a.tokens * a.x_row + p.channel;
    value_t* out = (value_t*)a.out + p.sequence * a.tokens * a.channels + p.channel;
    pw::Unit next[U];
#pragma unroll
    for (int t = 0; t < U; ++t) next[t] = tk::load(in + (p.first + t < p.last ? p.first + t : p.last - 1) * a.x_row);
    long long token = p.first;
    for (; token < p.last; token += U) {
#pragma unroll
        for (int t = 0; t < U; ++t) tk::values(next[t], x[K + t]);
        if (token + U < p.last) {
#pragma unroll
            for (int t = 0; t < U; ++t) {
                const long long at = token + U + t;
                next[t] = tk::load(in + (at < p.last ? at : p.last - 1) * a.x_row);
            }
        }
#pragma unroll
        for (int t = 0; t < U; ++t) {
            if (token + t >= p.last) break;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float z = bias[e];
#pragma unroll
                for (int i = 0; i < W; ++i) z = __builtin_fmaf(w[i][e], x[t + i][e], z);
                y[e] = pw::activate(z);
            }
            tk::store<true>(out + (token + t) * a.channels, pw::pack(y));
            // the inputs before the token behind the last
            if (a.after && token + t + 1 == a.tokens) {
#pragma unroll
                for (int i = 0; i < K; ++i)
                    tk::store<false>((value_t*)a.after + (p.sequence * K + i) * a.channels + p.channel, pw::pack(x[t + 1 + i]));
            }
        }
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = x[U + i][e];
    }
}

#elif SPIO_MODE == 1

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const SpioConv1dArgs a) {
    const Place p = place(a);
    if (!p.live) return;
    float w[W][8], bias[8], x[K + U][8], dz[K + U][8], dw[W][8], db[8];
    filters(a, p.channel, w, bias);
#pragma unroll
    for (int i = 0; i < K; ++i) input_before(a, p, p.first - K + i, x[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) dw[i][e] = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) dz[i][e] = 0.f;
    }
    const value_t* in = (const value_t*)a.x + p.sequence * a.tokens * a.x_row + p.channel;
    const value_t* dy = (const value_t*)a.dy + p.sequence * a.tokens * a.channels + p.channel;
    value_t* dx = (value_t*)a.dx + p.sequence * a.tokens * a.channels + p.channel;
    // dx of a token needs dz of the K tokens behind it: those behind the slice are computed here, too
    const long long last = p.last + K, read = last < a.tokens ? last : a.tokens;
    pw::Unit next_x[U], next_dy[U];
    auto request = [&](long long token) {
#pragma unroll
        for (int t = 0; t < U; ++t) {
            const long long at = token + t < read ? token + t : read - 1;
            next_x[t] = tk::load(in + at * a.x_row);
            next_dy[t] = tk::load(dy + at * a.channels);
        }
    };
    request(p.first);
    for (long long token = p.first; token < last; token += U) {
        float g[U][8];
#pragma unroll
        for (int t = 0; t < U; ++t) {
            tk::values(next_x[t], x[K + t]);
            tk::values(next_dy[t], g[t]);
        }
        if (token + U < read) request(token + U);
#pragma unroll
        for (int t = 0; t < U; ++t) {
            const long long at = token + t;
            if (at >= last) break;
            const bool there = at < a.tokens, own = at < p.last;
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = g[t][e];
                if (SPIO_ACT == 2) {
                    float z = bias[e];
#pragma unroll
                    for (int i = 0; i < W; ++i) z = __builtin_fmaf(w[i][e], x[t + i][e], z);
                    const float s = pw::sigmoid(z);
                    v *= __builtin_fmaf(s, __builtin_fmaf(-z, s, z), s);  // s + s z (1 - s)
                }
                v = there ? v : 0.f;
                dz[K + t][e] = v;
                if (own) {
                    db[e] += v;
#pragma unroll
                    for (int i = 0; i < W; ++i) dw[i][e] = __builtin_fmaf(v, x[t + i][e], dw[i][e]);
                }
                float r = 0.f;
#pragma unroll
                for (int i = 0; i < W; ++i) r = __builtin_fmaf(w[i][e], dz[K + t - i][e], r);
                d[e] = r;
            }
            if (at - K >= p.first) tk::store<true>(dx + (at - K) * a.channels, pw::pack(d));
        }
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = x[U + i][e], dz[i][e] = dz[U + i][e];
    }
    const long long slices = (a.tokens + a.slice - 1) / a.slice;
    float* sums = a.partials + (p.sequence * slices + p.slice) * (W + 1) * a.channels + p.channel;
#pragma unroll
    for (int i = 0; i <= W; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[i * a.channels + e] = i < W ? dw[i % W][e] : db[e];
}

#elif SPIO_MODE == 2

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const SpioConv1dArgs a) {
    const long long rows = a.sequences * ((a.tokens + a.slice - 1) / a.slice);
    tk::column_sums({a.partials, rows, a.channels, W, 1, a.dweight, a.dbias, nullptr}, __builtin_amdgcn_workgroup_id_x());
}

#else

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64))) SPIO_KERNEL_NAME(const SpioConv1dArgs a) {
    const unsigned units = (unsigned)(a.channels / 8);
    const unsigned id = __builtin_amdgcn_workgroup_id_x() * 64 + __builtin_amdgcn_workitem_id_x();
    const long long sequence = id / units, channel = id % units * 8;
    if (sequence >= a.sequences) return;
    float w[W][8], bias[8], x[W][8], y[8];
    pw::Unit unit[W];
#pragma unroll
    for (int i = 0; i < W; ++i)
        unit[i] = i < K ? tk::load((const value_t*)a.before + (sequence * K + i) * a.channels + channel)
                        : tk::load((const value_t*)a.x + sequence * a.x_row + channel);
    filters(a, channel, w, bias);
#pragma unroll
    for (int i = 0; i < W; ++i) tk::values(unit[i], x[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float z = bias[e];
#pragma unroll
        for (int i = 0; i < W; ++i) z = __builtin_fmaf(w[i][e], x[i][e], z);
        y[e] = pw::activate(z);
    }
    tk::store<false>((value_t*)a.out + sequence * a.channels + channel, pw::pack(y));
#pragma unroll
    for (int i = 0; i < K; ++i) tk::store<false>((value_t*)a.after + (sequence * K + i) * a.channels + channel, unit[i + 1]);
}

#endif
