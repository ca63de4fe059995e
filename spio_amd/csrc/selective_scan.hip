// Selective scan of a state-space layer over tokens-by-channels tensors (gfx950).  For every sequence and channel, with
// states h[0..N) in float32:
//
//   dl    = softplus(delta[t] + bias)           (or the sum itself)
//   h[s]  = exp(dl A[s]) h[s] + dl u[t] B[t][s]
//   y     = sum_s C[t][s] h[s] + D u[t];        out[t] = y silu(gate[t])
//
// and its gradients, g[s] = dL/dh[s] going from the last token to the first:
//
//   dy = dout silu(gate),  dgate = dout y silu'(gate),  g[t][s] = C[t][s] dy[t] + exp(dl[t+1] A[s]) g[t+1][s]
//   du = dl sum_s g B + D dy;   ddl = u sum_s g B + sum_s A g exp(dl A) h[t-1];   dA = sum g exp(dl A) h[t-1] dl
//   dB = sum_channels g dl u,   dC = sum_channels dy h,   dD = sum dy u,   ddelta = ddl softplus' = dbias's terms
//
//   SPIO_MODE 0  ends      what a chunk of tokens adds to the states, and the sum of its dl
//   SPIO_MODE 1  out       outputs, from the states before a chunk
//   SPIO_MODE 2  ends back what a chunk adds to exp(dl A) g at its first token
//   SPIO_MODE 3  back      gradients; sums over channels and over tokens as partial sums
//   SPIO_MODE 4  sums      the partial sums added up
//   SPIO_MODE 5  step      one token of every sequence: states read and written once
//   SPIO_MODE 6  join      the ends of chunks made the states before them; 7: the same from the last chunk to the first
//
// Modes 0 to 2: a lane is a channel and holds its N states, a wave is 64 channels and a chunk of a sequence (mode 3: two
// channels and half of their states).  So nothing crosses lanes but the sums over channels of dB and dC, and B and C are the
// same for a wave: it converts tiles of T tokens of them to float32 in LDS, and reads them back as broadcasts.  A state's
// decay over a chunk is exp(A sum dl), so that a chunk is joined by one product: where sequences and channels alone do not
// fill the device a sequence is cut into chunks, at the price of a first pass (modes 0 and 2) and a join.
//
// What bounds it are vector instructions, for each state and token forward a product, an exponential (which takes a SIMD as
// long as two others), a product and two multiply-adds, backward those and eight more, and one or two exponentials.  4n
// 2048l 2048c with 16 states, gate and softplus in bfloat16, each sequence in 32 chunks of 64 tokens (us traced, and the share of the
// time in which vector instructions issue): ends 70 (98 %), join 11, outputs with kept states 94 (83 %, and 427 MB at 4.6
// TB/s, of which 268 are kept states: memory as much as instructions), ends back 68 (96 %), join 11, gradients 231 (84 %), sums
// 11; the tensors of all of these would move in 46.  Without chunks, 128n 196l 768c: outputs 151 (53 %), gradients 315 (74 %),
// 1536 waves on 1024 SIMDs; a prompt of 1n 4099l 1536c in 74 chunks 30 (74 %) + 12 + 38 (72 %).
#include "spio_tokens.h"

#ifndef SPIO_MODE
#error "SPIO_MODE, SPIO_STATES, SPIO_T, SPIO_HELD, SPIO_WAVES, SPIO_GATE, SPIO_SOFTPLUS, SPIO_KEEP are required"
#endif

namespace {

constexpr int N = SPIO_STATES;
constexpr int T = SPIO_T;                  // tokens of a tile, and between kept states where there are such
constexpr int NP = (N + 3) / 4 * 4;        // states of a row in LDS, zeros behind the last one
constexpr int M = 2 * N;                   // a token's B and C
constexpr int STAGED = (T * N + 63) / 64;  // of a tile's B, a lane's, and of its C
constexpr bool GATE = SPIO_GATE, SOFTPLUS = SPIO_SOFTPLUS, KEEP = SPIO_KEEP;
constexpr int HELD = SPIO_HELD;            // last tokens of a tile whose decays the backward pass holds, the others are taken again

typedef SpioScanArgs Args;
using tk::LN2;
using tk::LOG2E;
using tk::barrier;
using tk::exp2_;
using tk::from;
using tk::value_t;

// log(1 + exp(x)).  exp(-|x|) = e is at most 1, and log(1 + e) = 2 artanh(e / (2 + e)), whose series
// needs seven terms at a third: exact to the last places where e is small, too.
__device__ inline float softplus(float x) {
    const float e = exp2_(__builtin_fabsf(x) * -LOG2E);
    const float s = e * pw::reciprocal(2.f + e), q = s * s;
    float r = 2.f / 13;
    r = __builtin_fmaf(r, q, 2.f / 11);
    r = __builtin_fmaf(r, q, 2.f / 9);
    r = __builtin_fmaf(r, q, 2.f / 7);
    r = __builtin_fmaf(r, q, 2.f / 5);
    r = __builtin_fmaf(r, q, 2.f / 3);
    r = __builtin_fmaf(r, q, 2.f);
    return __builtin_fmaf(r, s, x > 0.f ? x : x == x ? 0.f : x);
}

// ---- where a wave is, and what it reads a tile ahead ----

struct Place {
    long long sequence;
    int block, chunk, chunks;
    int first, last;  // tokens of the chunk: [first, last)
    int channel, loaded;
    bool live;
};
__device__ inline Place place(const Args& a) {
    Place p;
    const unsigned blocks = (unsigned)((a.channels + 63) / 64);
    p.chunks = (int)((a.tokens + a.chunk - 1) / a.chunk);
    unsigned id = __builtin_amdgcn_workgroup_id_x();
    p.block = (int)(id % blocks);
    id /= blocks;
    p.chunk = (int)(id % (unsigned)p.chunks);
    p.sequence = id / (unsigned)p.chunks;
    p.first = p.chunk * (int)a.chunk;
    const int end = p.first + (int)a.chunk;
    p.last = end < (int)a.tokens ? end : (int)a.tokens;
    p.channel = p.block * 64 + (int)__builtin_amdgcn_workitem_id_x();
    p.live = p.channel < (int)a.channels;
    p.loaded = p.live ? p.channel : (int)a.channels - 1;  // lanes without a channel read the last one's
    return p;
}

// The value that many bytes behind an address that all lanes have
__device__ inline float at(const float* base, unsigned bytes) { return *(const float*)((const char*)base + bytes); }

// Memory from an address on that all lanes have.  Stores of lanes behind `bytes` are dropped; loads stay before the end by
// themselves (WHOLE).
constexpr unsigned WHOLE = 0x7ffffff0u;
constexpr unsigned SIZE = sizeof(value_t);
__device__ inline value_t load(pw_rsrc rs, unsigned lane_bytes, unsigned bytes) {
#if SPIO_DTYPE == 2
    return pw::as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (int)lane_bytes, (int)bytes, 0));
#else
    return __builtin_bit_cast(value_t, __builtin_amdgcn_raw_buffer_load_b16(rs, (int)lane_bytes, (int)bytes, 0));
#endif
}
// (What may be behind the end is so by the lane's offset: the scalar one is not relied upon there.)
__device__ inline void store(pw_rsrc rs, unsigned lane_bytes, value_t v) {
#if SPIO_DTYPE == 2
    __builtin_amdgcn_raw_buffer_store_b32(pw::as_bits(v), rs, (int)lane_bytes, 0, 0);
#else
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rs, (int)lane_bytes, 0, 0);
#endif
}
__device__ inline void store_float(pw_rsrc rs, unsigned lane_bytes, float v) {
    __builtin_amdgcn_raw_buffer_store_b32(pw::as_bits(v), rs, (int)lane_bytes, 0, 0);
}
// The rows of a tile of an array [tokens][channels] to be stored to, as far as there are tokens
__device__ inline pw_rsrc rows_to(void* to, const Args& a, const Place& p, int token) {
    const int count = p.last - token < T ? p.last - token : T;
    return pw::buffer((value_t*)to + (p.sequence * a.tokens + token) * a.channels, (unsigned)count * (unsigned)a.channels * SIZE);
}

// The tile of tokens [token, token + T), those from `last` on in the place of which the last one is read.
struct Tile {
    value_t u[T], delta[T], gate[T], dout[T], B[STAGED], C[STAGED];
};
__device__ inline void request_channels(value_t (&v)[T], const void* from, long long stride, long long row0, const Place& p, int token) {
    const pw_rsrc rs = pw::buffer((const value_t*)from + (row0 + token) * stride, WHOLE);
    const int left = p.last - 1 - token;
#pragma unroll
    for (int t = 0; t < T; ++t) v[t] = load(rs, (unsigned)p.loaded * SIZE, (unsigned)(t < left ? t : left) * (unsigned)stride * SIZE);
}
__device__ inline void request_rows(value_t (&v)[STAGED], const void* from, long long stride, long long row0, const Place& p, int token) {
    const int lane = (int)__builtin_amdgcn_workitem_id_x();
    const pw_rsrc rs = pw::buffer((const value_t*)from + (row0 + token) * stride, WHOLE);
    const int left = p.last - 1 - token;
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
        const int e = i * 64 + lane, t = e / N < left ? e / N : left;
        v[i] = load(rs, (unsigned)(t * (int)stride + e % N) * SIZE, 0);
    }
}
template <bool U, bool DOUT, bool B, bool C>
__device__ inline void request(Tile& tile, const Args& a, const Place& p, int token) {
    const long long row0 = p.sequence * a.tokens;
    if (U) request_channels(tile.u, a.u, a.u_row, row0, p, token);
    request_channels(tile.delta, a.delta, a.delta_row, row0, p, token);
    if (C && GATE) request_channels(tile.gate, a.gate, a.gate_row, row0, p, token);
    if (DOUT) request_channels(tile.dout, a.dout, a.channels, row0, p, token);
    if (B) request_rows(tile.B, a.B, a.b_row, row0, p, token);
    if (C) request_rows(tile.C, a.C, a.c_row, row0, p, token);
}
// B and C of the tile in LDS, [T][2][NP]; zeros from token `count` on, so that nothing that is not finite is multiplied there
template <bool B, bool C>
__device__ inline void stage(const Tile& tile, int count, float* lds) {
    const int lane = (int)__builtin_amdgcn_workitem_id_x();
    barrier();
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
        const int e = i * 64 + lane, t = e / N, s = e % N;
        if (e >= T * N) break;
        if (B) lds[t * 2 * NP + s] = t < count ? (float)tile.B[i] : 0.f;
        if (C) lds[(t * 2 + 1) * NP + s] = t < count ? (float)tile.C[i] : 0.f;
    }
    if (N % 2 && lane < 2 * T) lds[lane * NP + N] = 0.f;  // (read where the states are halved)
    barrier();
}
__device__ inline void row_of(const float* lds, int t, int which, float (&v)[NP]) {
    typedef float float4_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < NP / 4; ++i) {
        const float4_t q = ((const float4_t*)(lds + (t * 2 + which) * NP))[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = q[j];
    }
}

// The states of a half of the wave only, (N + 1) / 2 each; zeros behind the last one
template <int H>
__device__ inline void half_row(const float* lds, int t, int which, int half, float (&v)[H]) {
    const float* row = lds + (t * 2 + which) * NP + half * H;
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = row[i];
}

// A rate as the exponent of 2 that it is; finite from below, so that a time step of zero (a token behind the last one) decays
// nothing at a rate of minus infinity, either
__device__ inline float rate(float A) {
    const float r = A * LOG2E;
    return r < -3.4e38f ? -3.4e38f : r;
}
__device__ inline void rates(const Args& a, const Place& p, float (&A2)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) A2[s] = rate(a.A[(long long)p.loaded * N + s]);
}
__device__ inline float time_step(float raw) { return SOFTPLUS ? softplus(raw) : raw; }

}  // namespace

#if SPIO_MODE == 0 || SPIO_MODE == 1

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64))) SPIO_KERNEL_NAME(const Args a) {
    __shared__ __attribute__((aligned(16))) float lds[T * 2 * NP];
    constexpr bool OUT = SPIO_MODE == 1;
    const Place p = place(a);
    if (!OUT && p.chunk + 1 == p.chunks) return;  // nothing comes behind the last chunk
    Tile tile;
    request<true, false, true, OUT>(tile, a, p, p.first);
    float A2[N], h[N];
    rates(a, p, A2);
    const float bias = a.bias ? a.bias[p.loaded] : 0.f;
    const float D = OUT && a.D ? a.D[p.loaded] : 0.f;
#pragma unroll
    for (int s = 0; s < N; ++s) h[s] = 0.f;
    if (OUT && p.chunks > 1) {
        const float* start = a.ends + (p.sequence * p.chunks + p.chunk) * (N + 1) * a.channels;
#pragma unroll
        for (int s = 0; s < N; ++s) h[s] = at(start + s * a.channels, (unsigned)p.loaded * 4u);
    } else if (OUT && a.before) {
#pragma unroll
        for (int s = 0; s < N; ++s) h[s] = a.before[(p.sequence * a.channels + p.loaded) * N + s];
    }
    float sum = 0.f;
    const long long tiles = (a.tokens + T - 1) / T;
    const unsigned lane_bytes = p.live ? (unsigned)p.channel * SIZE : pw::OOB;
    for (int token = p.first; token < p.last; token += T) {
        stage<true, OUT>(tile, p.last - token, lds);
        float u[T], dl[T], gate[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            u[t] = (float)tile.u[t];
            dl[t] = time_step((float)tile.delta[t] + bias);
            if (token + t >= p.last) u[t] = dl[t] = 0.f;  // (decays by 1, adds nothing)
            gate[t] = OUT && GATE ? (float)tile.gate[t] : 0.f;
            if (!OUT) sum += dl[t];
        }
        if (token + T < p.last) request<true, false, true, OUT>(tile, a, p, token + T);
        if (OUT && KEEP) {
            const pw_rsrc kept = pw::buffer(a.kept + (p.sequence * tiles + token / T) * N * a.channels, N * (unsigned)a.channels * 4);
#pragma unroll
            for (int s = 0; s < N; ++s) {
                const int row = s * (int)a.channels * 4;
                __builtin_amdgcn_raw_buffer_store_b32(pw::as_bits(h[s]), kept, (int)(p.live ? (unsigned)p.channel * 4 : pw::OOB), row, 0);
            }
        }
        const pw_rsrc out = rows_to(a.out, a, p, token);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float B[NP], C[NP];
            row_of(lds, t, 0, B);
            if (OUT) row_of(lds, t, 1, C);
            const float x = dl[t] * u[t];
            float y = D * u[t];
#pragma unroll
            for (int s = 0; s < N; ++s) {
                h[s] = __builtin_fmaf(exp2_(dl[t] * A2[s]), h[s], x * B[s]);
                if (OUT) y = __builtin_fmaf(C[s], h[s], y);
            }
            if (OUT) {
                if (GATE) y *= gate[t] * pw::sigmoid(gate[t]);
                store(out, lane_bytes + (unsigned)t * (unsigned)a.channels * SIZE, (value_t)y);
            }
        }
    }
    if (!p.live) return;
    if (!OUT) {
        float* e = a.ends + (p.sequence * p.chunks + p.chunk) * (N + 1) * a.channels + p.channel;
#pragma unroll
        for (int s = 0; s < N; ++s) e[s * a.channels] = h[s];
        e[N * a.channels] = sum;
    } else if (a.after && p.chunk + 1 == p.chunks) {
#pragma unroll
        for (int s = 0; s < N; ++s) a.after[(p.sequence * a.channels + p.channel) * N + s] = h[s];
    }
}

#elif SPIO_MODE == 2

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64))) SPIO_KERNEL_NAME(const Args a) {
    __shared__ __attribute__((aligned(16))) float lds[T * 2 * NP];
    const Place p = place(a);
    if (p.chunk == 0) return;  // nothing comes before the first chunk
    Tile tile;
    int token = p.first + (p.last - p.first - 1) / T * T;
    request<false, true, false, true>(tile, a, p, token);
    float A2[N], r[N], sum = 0.f;
    rates(a, p, A2);
    const float bias = a.bias ? a.bias[p.loaded] : 0.f;
#pragma unroll
    for (int s = 0; s < N; ++s) r[s] = 0.f;
    for (; token >= p.first; token -= T) {
        stage<false, true>(tile, p.last - token, lds);
        float dy[T], dl[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float gate = GATE ? (float)tile.gate[t] : 0.f;
            dy[t] = (float)tile.dout[t] * (GATE ? gate * pw::sigmoid(gate) : 1.f);
            dl[t] = time_step((float)tile.delta[t] + bias);
            if (token + t >= p.last) dy[t] = dl[t] = 0.f;
            sum += dl[t];
        }
        if (token > p.first) request<false, true, false, true>(tile, a, p, token - T);
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
            float C[NP];
            row_of(lds, t, 1, C);
#pragma unroll
            for (int s = 0; s < N; ++s) r[s] = exp2_(dl[t] * A2[s]) * __builtin_fmaf(C[s], dy[t], r[s]);
        }
    }
    if (!p.live) return;
    float* e = a.ends + (p.sequence * p.chunks + p.chunk) * (N + 1) * a.channels + p.channel;
#pragma unroll
    for (int s = 0; s < N; ++s) e[s * a.channels] = r[s];
    e[N * a.channels] = sum;
}

#elif SPIO_MODE == 3

namespace {

// Sums over a wave's lanes of m values a lane, in steps that halve both: of a pair of values a lane keeps the one that its
// bit names and adds the half that another lane has of it.  After six steps a lane holds the sum of one value
// (sum_index), where there are fewer than 64 values the same as other lanes.
template <int STEP>
__device__ inline float halves(float a, float b, int lane) {
    if (STEP < 2) {
        // lanes or rows of lanes exchanged: a's lower halves with b's in the first, the upper ones in the second
        const auto r = STEP == 0 ? __builtin_amdgcn_permlane32_swap(pw::as_bits(a), pw::as_bits(b), false, false)
                                 : __builtin_amdgcn_permlane16_swap(pw::as_bits(a), pw::as_bits(b), false, false);
        return pw::as_float(r[0]) + pw::as_float(r[1]);
    }
    const bool upper = lane & 32 >> STEP;
    const float mine = upper ? b : a, other = upper ? a : b;
    // row_ror:8, row_half_mirror, quad_perm [2,3,0,1] and [1,0,3,2]
    constexpr int CTRL = STEP == 2 ? 0x128 : STEP == 3 ? 0x141 : STEP == 4 ? 0x4E : 0xB1;
    return mine + from<CTRL>(other);
}
template <int STEP, int m>
struct Sum {
    static constexpr int half = (m + 1) / 2;
    static __device__ inline float of(const float (&v)[m], int lane) {
        float r[half];
#pragma unroll
        for (int i = 0; i < half; ++i) r[i] = halves<STEP>(v[i], m == 1 ? v[i] : i + half < m ? v[i + half] : 0.f, lane);
        return Sum<STEP + 1, half>::of(r, lane);
    }
    // the value that a lane holds; -1: none, or one that another lane has as well
    static __device__ inline int index(int lane) {
        const int i = Sum<STEP + 1, half>::index(lane);
        const int bit = lane & 32 >> STEP ? 1 : 0;
        const int at = m == 1 ? (bit ? -1 : i) : i + bit * half;
        return i < 0 || at >= m ? -1 : at;
    }
};
template <int m>
struct Sum<6, m> {
    static_assert(m == 1, "at most 64 values");
    static __device__ inline float of(const float (&v)[1], int) { return v[0]; }
    static __device__ inline int index(int) { return 0; }
};

}  // namespace

// A lane has two channels, 32 apart, and half of their states: the sums over channels of dB and dC so begin within a lane and
// cross 32 others, half as many steps as with a channel a lane, and a lane needs half of B and C.  What goes by channel (time
// steps, gradients of the inputs) is done with a channel a lane, and passes through LDS one way, through an exchange of
// halves of the wave with which the sums over states end the other way.
extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64), amdgpu_waves_per_eu(SPIO_WAVES)))
SPIO_KERNEL_NAME(const Args a) {
    __shared__ __attribute__((aligned(16))) float lds[T * 2 * NP];
    enum { DL, X, DY, U, SLOPE, DGATE, OWN };
    __shared__ float own[T][OWN][64];  // of every token of the tile, by channel
    constexpr int H = (N + 1) / 2;     // states of a lane
    const int lane = (int)__builtin_amdgcn_workitem_id_x(), half = lane / 32, j = lane % 32;
    const Place p = place(a);
    const int blocks = (int)((a.channels + 63) / 64);
    const long long tiles = (a.tokens + T - 1) / T;
    Tile tile;
    int token = p.first + (p.last - p.first - 1) / T * T;
    request<true, true, true, true>(tile, a, p, token);
    int channel[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        channel[c] = p.block * 64 + c * 32 + j;
        channel[c] = channel[c] < (int)a.channels ? channel[c] : (int)a.channels - 1;
    }
    // (a state behind the last one, where they are odd: rate, B and C of zero)
    auto state = [&](int i) { return half * H + i < N ? half * H + i : N - 1; };
    auto there = [&](int i) { return half * H + i < N; };
    // Rows of states [N][channels]: bytes from row i to the lane's state i of a channel.  What is not there, a channel or a state
    // behind the last one (of the upper half, where they are odd), is behind the end by the lane's offset alone: zeros are loaded
    // there, stores dropped.  (The device counts the scalar offset of row i against the end as well, but the builtin does not promise
    // that.)
    unsigned offset[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int at = p.block * 64 + c * 32 + j;
        offset[c] = at < (int)a.channels ? (unsigned)(half * H * (int)a.channels + at) * 4u : pw::OOB;
    }
    const int row_bytes = (int)a.channels * 4;
    auto states = [&](const float* rows) { return pw::buffer(rows, N * (unsigned)row_bytes); };
    auto offset_of = [&](int c, int i) { return (int)(N % 2 && i == H - 1 && half ? pw::OOB : offset[c]); };
    auto load_state = [&](pw_rsrc rs, int c, int i) {
        return pw::as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, offset_of(c, i), i * row_bytes, 0));
    };
    float A2[2][H], r[2][H], dA[2][H];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < H; ++i) {
            A2[c][i] = there(i) ? rate(a.A[(long long)channel[c] * N + state(i)]) : 0.f;
            r[c][i] = dA[c][i] = 0.f;
        }
    if (p.chunks > 1) {  // what the chunks behind this one add
        const pw_rsrc start = states(a.ends + (p.sequence * p.chunks + p.chunk) * (N + 1) * a.channels);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < H; ++i) r[c][i] = load_state(start, c, i);
    }
    const float bias = a.bias ? a.bias[p.loaded] : 0.f;
    const float D = a.D ? a.D[p.loaded] : 0.f;
    const unsigned lane_bytes = p.live ? (unsigned)p.channel * SIZE : pw::OOB;
    float dD = 0.f, dbias = 0.f;
    // which of its half's sums a lane ends with
    const int value = Sum<1, 2 * H>::index(j), sum_state = half * H + value % H;
    const unsigned sum_bytes = value < 0 || sum_state >= N ? pw::OOB : (unsigned)(p.block * M + value / H * N + sum_state) * 4u;
    float next[2][H];  // states before the tile that comes next
    auto request_states = [&](int token) {
        const pw_rsrc kept = states(a.kept + (p.sequence * tiles + token / T) * N * a.channels);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < H; ++i) next[c][i] = load_state(kept, c, i);
    };
    request_states(token);
    for (; token >= p.first; token -= T) {
        float before[2][H], h[T][2][H], decay[HELD ? HELD : 1][2][H];  // states before the tile and behind its tokens
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < H; ++i) before[c][i] = next[c][i];
        stage<true, true>(tile, p.last - token, lds);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const bool counts = token + t < p.last && p.live;
            const float raw = counts ? (float)tile.delta[t] + bias : 0.f;
            const float dout = counts ? (float)tile.dout[t] : 0.f;
            const float u = counts ? (float)tile.u[t] : 0.f;
            float dl = time_step(raw);
            asm("" : "+v"(dl));  // (not a branch around it)
            dl = counts ? dl : 0.f;
            own[t][DL][lane] = dl;
            own[t][X][lane] = dl * u;
            own[t][U][lane] = u;
            own[t][SLOPE][lane] = SOFTPLUS ? pw::sigmoid(raw) : 1.f;
            if (GATE) {
                const float gate = counts ? (float)tile.gate[t] : 0.f, s = pw::sigmoid(gate), v = gate * s;
                own[t][DY][lane] = dout * v;
                own[t][DGATE][lane] = dout * __builtin_fmaf(v, 1.f - s, s);
            } else {
                own[t][DY][lane] = dout;
            }
        }
        barrier();
        const pw_rsrc to_du = rows_to(a.du, a, p, token), to_ddelta = rows_to(a.ddelta, a, p, token),
                      to_dgate = rows_to(a.dgate, a, p, token);
        const int count = p.last - token < T ? p.last - token : T;
        const pw_rsrc token_sums = pw::buffer(a.token_sums + (p.sequence * a.tokens + token) * blocks * M,
                                              (unsigned)count * (unsigned)blocks * M * 4u);
        if (token > p.first) request<true, true, true, true>(tile, a, p, token - T);
        float y[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float B[H], C[H], part[2];
            half_row(lds, t, 0, half, B);
            half_row(lds, t, 1, half, C);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float dl = own[t][DL][c * 32 + j], x = own[t][X][c * 32 + j];
                part[c] = 0.f;
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const float d = exp2_(dl * A2[c][i]);
                    if (t >= T - HELD) decay[t - (T - HELD)][c][i] = d;
                    h[t][c][i] = __builtin_fmaf(d, t ? h[t ? t - 1 : 0][c][i] : before[c][i], x * B[i]);
                    part[c] = __builtin_fmaf(C[i], h[t][c][i], part[c]);
                }
            }
            y[t] = halves<0>(part[0], part[1], lane);
        }
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
            // (once the registers of the last token are free)
            if (t == (T > 1 ? T - 2 : 0) && token > p.first) request_states(token - T);
            float B[H], C[H], sums[2 * H], gB[2] = {}, gq[2] = {};
            half_row(lds, t, 0, half, B);
            half_row(lds, t, 1, half, C);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float x = own[t][X][c * 32 + j], dy = own[t][DY][c * 32 + j];
                float dl = own[t][DL][c * 32 + j];
                if (t < T - HELD) asm("" : "+v"(dl));  // (or the exponentials would be held)
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const float g = __builtin_fmaf(C[i], dy, r[c][i]);
                    sums[i] = c ? __builtin_fmaf(x, g, sums[i]) : x * g;
                    sums[H + i] = c ? __builtin_fmaf(dy, h[t][c][i], sums[H + i]) : dy * h[t][c][i];
                    gB[c] = __builtin_fmaf(g, B[i], gB[c]);
                    r[c][i] = (t >= T - HELD ? decay[t >= T - HELD ? t - (T - HELD) : 0][c][i] : exp2_(dl * A2[c][i])) * g;
                    const float w = r[c][i] * (t ? h[t ? t - 1 : 0][c][i] : before[c][i]);
                    dA[c][i] = __builtin_fmaf(w, dl, dA[c][i]);
                    gq[c] = __builtin_fmaf(w, A2[c][i], gq[c]);
                }
            }
            const float total = Sum<1, 2 * H>::of(sums, lane);
            const float all_gB = halves<0>(gB[0], gB[1], lane), all_gq = halves<0>(gq[0], gq[1], lane);
            const float u = own[t][U][lane], dy = own[t][DY][lane];
            const float du = __builtin_fmaf(all_gB, own[t][DL][lane], D * dy);
            const float ddelta = __builtin_fmaf(all_gB, u, all_gq * LN2) * own[t][SLOPE][lane];
            dD = __builtin_fmaf(dy, u, dD);
            dbias += ddelta;  // (of a token that is not there all are zero)
            const unsigned row = (unsigned)t * (unsigned)a.channels * SIZE;
            store_float(token_sums, sum_bytes + (unsigned)t * (unsigned)blocks * M * 4u, total);
            store(to_du, lane_bytes + row, (value_t)du);
            store(to_ddelta, lane_bytes + row, (value_t)ddelta);
            if (GATE) store(to_dgate, lane_bytes + row, (value_t)(own[t][DGATE][lane] * __builtin_fmaf(D, u, y[t])));
        }
    }
    float* sums = a.channel_sums + (p.sequence * p.chunks + p.chunk) * (N + 2) * a.channels;
    const pw_rsrc to_dA = states(sums);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < H; ++i)
            __builtin_amdgcn_raw_buffer_store_b32(pw::as_bits(dA[c][i]), to_dA, offset_of(c, i), i * row_bytes, 0);
    if (!p.live) return;
    sums[N * a.channels + p.channel] = dD;
    sums[(N + 1) * a.channels + p.channel] = dbias;
}

#elif SPIO_MODE == 4

// The first workgroups add up 256 sums over blocks of channels each, the rest those over chunks.
extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const Args a) {
    const int tid = (int)__builtin_amdgcn_workitem_id_x();
    const long long rows = a.sequences * a.tokens;
    const long long row_groups = (rows * M + 255) / 256;
    const long long group = __builtin_amdgcn_workgroup_id_x();
    if (group < row_groups) {
        const long long at = group * 256 + tid;
        if (at >= rows * M) return;
        const int blocks = (int)((a.channels + 63) / 64);
        const long long row = at / M;
        const int s = (int)(at % M);
        const float* from = a.token_sums + row * blocks * M + s;
        float sum = 0.f;
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) sum += from[(long long)b * M];
        if (s < N)
            ((value_t*)a.dB)[row * N + s] = (value_t)sum;
        else
            ((value_t*)a.dC)[row * N + s - N] = (value_t)sum;
        return;
    }
    const long long chunks = (a.tokens + a.chunk - 1) / a.chunk;
    tk::column_sums({a.channel_sums, a.sequences * chunks, a.channels, N, 2, a.dA, a.dD, a.dbias}, group - row_groups);
}

#elif SPIO_MODE == 6 || SPIO_MODE == 7

// A lane is a state of a channel, and goes from chunk to chunk, v = exp(A sum dl) v + end, leaving v in the place of the
// end.  The ends of JOINED chunks are requested at once: waiting for memory is all that it does (4n 2048l 2048c, 32 chunks, with 4, 8,
// 16 and 32 at once 8.9, 8.7, 10.7 and 26 us; 1n 4099l 1536c, 74 chunks, 11.0, 10.9, 14.5 and 28).
extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64))) SPIO_KERNEL_NAME(const Args a) {
    constexpr bool BACK = SPIO_MODE == 7;
    constexpr int JOINED = 8;
    const unsigned blocks = (unsigned)((a.channels + 63) / 64);
    const unsigned id = __builtin_amdgcn_workgroup_id_x();
    const long long channel = id % blocks * 64 + __builtin_amdgcn_workitem_id_x();
    const int s = (int)(id / blocks % N);
    const long long sequence = id / blocks / N;
    const int chunks = (int)((a.tokens + a.chunk - 1) / a.chunk);
    if (channel >= a.channels) return;
    const float A2 = rate(a.A[channel * N + s]);
    float v = !BACK && a.before ? a.before[(sequence * a.channels + channel) * N + s] : 0.f;
    float* ends = a.ends + sequence * chunks * (N + 1) * a.channels + channel;
    for (int first = 0; first < chunks; first += JOINED) {
        float end[JOINED], sum[JOINED];
#pragma unroll
        for (int k = 0; k < JOINED; ++k) {
            const int i = first + k < chunks ? first + k : chunks - 1;
            const float* e = ends + (BACK ? chunks - 1 - i : i) * (N + 1) * a.channels;
            end[k] = e[s * a.channels];
            sum[k] = e[N * a.channels];
        }
#pragma unroll
        for (int k = 0; k < JOINED; ++k) {
            const int i = first + k;
            if (i >= chunks) break;
            ends[((BACK ? chunks - 1 - i : i) * (N + 1) + s) * a.channels] = v;
            // The factor's whole powers of two go into v first: by itself it may be infinite, or zero, where its product with
            // a small, or a large, v is not.  (They are bounded, as v's are; nothing stays nothing at an infinite factor.)
            const float power = sum[k] * A2;
            const int whole = (int)__builtin_amdgcn_fmed3f(power, -400.f, 400.f);
            v = v == 0.f ? end[k] : __builtin_fmaf(exp2_(power - (float)whole), __builtin_ldexpf(v, whole), end[k]);
        }
    }
}

#else

// (64n 1536c 16 states 5.1 us: 2.2 a launch takes, 13.6 MB in the rest)
// One token: a lane has four states of a channel, so that a wave's loads of states are whole lines; the lanes of a channel
// (a power of two) add their parts of y.
extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const Args a) {
    constexpr int LANES = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8;
    typedef float float4_t __attribute__((ext_vector_type(4)));
    const long long id = (long long)__builtin_amdgcn_workgroup_id_x() * 256 + __builtin_amdgcn_workitem_id_x();
    const int part = (int)(id % LANES);
    const long long at = id / LANES, last = a.sequences * a.channels - 1;
    const long long item = at <= last ? at : last;
    const long long sequence = item / a.channels;
    const int c = (int)(item % a.channels);
    float h[4], A2[4], B[4], C[4];
    const float* before = a.before + item * N;
    if (N % 4 == 0 && part * 4 < N) {
        const float4_t v = *(const float4_t*)(before + part * 4);
        const float4_t w = *(const float4_t*)(a.A + (long long)c * N + part * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = v[i], A2[i] = rate(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = part * 4 + i < N;
            h[i] = there ? before[part * 4 + i] : 0.f;
            A2[i] = there ? rate(a.A[(long long)c * N + part * 4 + i]) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool there = part * 4 + i < N;
        B[i] = there ? (float)((const value_t*)a.B)[sequence * a.b_row + part * 4 + i] : 0.f;
        C[i] = there ? (float)((const value_t*)a.C)[sequence * a.c_row + part * 4 + i] : 0.f;
    }
    const float u = (float)((const value_t*)a.u)[sequence * a.u_row + c];
    const float gate = GATE ? (float)((const value_t*)a.gate)[sequence * a.gate_row + c] : 0.f;
    const float dl = time_step((float)((const value_t*)a.delta)[sequence * a.delta_row + c] + (a.bias ? a.bias[c] : 0.f));
    const float x = dl * u;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = __builtin_fmaf(exp2_(dl * A2[i]), h[i], x * B[i]);
        y = __builtin_fmaf(C[i], h[i], y);
    }
    if (LANES >= 2) y += from<0xB1>(y);   // quad_perm [1,0,3,2]
    if (LANES >= 4) y += from<0x4E>(y);   // quad_perm [2,3,0,1]
    if (LANES >= 8) y += from<0x141>(y);  // row_half_mirror
    if (at > last) return;
    if (part == 0) {
        y = __builtin_fmaf(a.D ? a.D[c] : 0.f, u, y);
        if (GATE) y *= gate * pw::sigmoid(gate);
        ((value_t*)a.out)[item] = (value_t)y;
    }
    float* after = a.after + item * N;
    if (N % 4 == 0) {
        if (part * 4 < N) *(float4_t*)(after + part * 4) = float4_t{h[0], h[1], h[2], h[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (part * 4 + i < N) after[part * 4 + i] = h[i];
    }
}

#endif
