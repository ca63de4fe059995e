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
//   SPIO_MODE 1  out       outputs, from the states before a chunk: those of the ends before it joined
//   SPIO_MODE 2  ends back what a chunk adds to exp(dl A) g at its first token
//   SPIO_MODE 3  back      gradients; sums over channels and over tokens as partial sums
//   SPIO_MODE 4  sums      the partial sums added up
//   SPIO_MODE 5  step      one token of every sequence: states read and written once
//
// Modes 0 to 3: a lane is a channel and holds its N states, a wave is 64 channels and a chunk of a sequence.  So nothing
// crosses lanes but the sums over channels of dB and dC, and B and C are the same for a wave: it converts tiles of T
// tokens of them to float32 in LDS, and reads them back as broadcasts.  A state's decay over a chunk is
// exp(A sum dl), so that a chunk is joined by one product: where the channels alone do not fill the device a
// sequence is cut into chunks, at the price of the first pass (mode 0 and 2).
//
// What bounds it are vector instructions: a product, an exponential (four times as long as the others), a product and
// two multiply-adds for each state and token; the tensors move in a third of that time.
#include "spio_tokens.h"

#ifndef SPIO_MODE
#error "SPIO_MODE, SPIO_STATES are required"
#endif

namespace {

constexpr int N = SPIO_STATES;
constexpr int T = SPIO_T;                       // tokens of a tile, and between kept states
constexpr int NP = (N + 3) / 4 * 4;        // states of a row in LDS
constexpr int M = 2 * N;                   // a token's B and C
constexpr int STAGED = (T * M + 63) / 64;  // of those of a tile, a lane's
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

// The tile of tokens [token, token + T), those from `last` on in the place of which the last one is read.
struct Tile {
    value_t u[T], delta[T], gate[T], dout[T], bc[STAGED];
};
template <bool U, bool DOUT, bool B, bool C>
__device__ inline void request(Tile& tile, const Args& a, const Place& p, int token) {
    const long long row0 = p.sequence * a.tokens;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const int at = token + t < p.last ? token + t : p.last - 1;
        const long long row = row0 + at;
        if (U) tile.u[t] = ((const value_t*)a.u + row * a.u_row)[p.loaded];
        tile.delta[t] = ((const value_t*)a.delta + row * a.delta_row)[p.loaded];
        if (C && a.gate) tile.gate[t] = ((const value_t*)a.gate + row * a.gate_row)[p.loaded];
        if (DOUT) tile.dout[t] = ((const value_t*)a.dout + row * a.channels)[p.loaded];
    }
    const int lane = (int)__builtin_amdgcn_workitem_id_x();
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
        int e = i * 64 + lane;
        e = e < T * M ? e : T * M - 1;
        const int t = e / M, s = e % M;
        const int at = token + t < p.last ? token + t : p.last - 1;
        const bool is_c = s >= N;
        if (is_c ? !C : !B) continue;
        const value_t* from = is_c ? (const value_t*)a.C + (row0 + at) * a.c_row + (s - N) : (const value_t*)a.B + (row0 + at) * a.b_row + s;
        tile.bc[i] = *from;
    }
}
// B and C of the tile in LDS, [T][2][NP]
__device__ inline void stage(const Tile& tile, float* lds) {
    const int lane = (int)__builtin_amdgcn_workitem_id_x();
    barrier();
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
        const int e = i * 64 + lane, t = e / M, s = e % M;
        if (e < T * M) lds[(t * 2 + (s >= N)) * NP + (s >= N ? s - N : s)] = (float)tile.bc[i];
    }
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

// A of a channel as the exponents of 2 that its rates are
__device__ inline void rates(const Args& a, const Place& p, float (&A2)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) A2[s] = a.A[(long long)p.loaded * N + s] * LOG2E;
}
__device__ inline float time_step(const Args& a, float delta, float bias) {
    const float raw = delta + bias;
    return a.softplus ? softplus(raw) : raw;
}

// What precedes the chunk in the order of the scan, joined: chunk by chunk from the far end, v = exp(A sum dl) v + end
__device__ inline void join(const Args& a, const Place& p, const float (&A2)[N], float (&v)[N], bool back) {
    const long long row = a.channels;
    const float* ends = a.ends + p.sequence * p.chunks * (N + 1) * row + p.loaded;
    const int count = back ? p.chunks - 1 - p.chunk : p.chunk;
    for (int i = 0; i < count; ++i) {
        const float* e = ends + (long long)(back ? p.chunks - 1 - i : i) * (N + 1) * row;
        const float sum = e[N * row];
#pragma unroll
        for (int s = 0; s < N; ++s) v[s] = __builtin_fmaf(exp2_(sum * A2[s]), v[s], e[s * row]);
    }
}

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
    for (int s = 0; s < N; ++s) h[s] = OUT && a.before ? a.before[(p.sequence * a.channels + p.loaded) * N + s] : 0.f;
    if (OUT && p.chunk) join(a, p, A2, h, false);
    float sum = 0.f;
    const long long tiles = (a.tokens + T - 1) / T;
    for (int token = p.first; token < p.last; token += T) {
        stage(tile, lds);
        float u[T], dl[T], gate[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            u[t] = (float)tile.u[t];
            dl[t] = time_step(a, (float)tile.delta[t], bias);
            if (token + t >= p.last) u[t] = dl[t] = 0.f;  // (decays by 1, adds nothing)
            gate[t] = OUT && a.gate ? (float)tile.gate[t] : 0.f;
            if (!OUT) sum += dl[t];
        }
        if (token + T < p.last) request<true, false, true, OUT>(tile, a, p, token + T);
        if (OUT && a.kept && p.live) {
            float* kept = a.kept + ((p.sequence * tiles + token / T) * N) * a.channels + p.channel;
#pragma unroll
            for (int s = 0; s < N; ++s) kept[s * a.channels] = h[s];
        }
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
            if (OUT && token + t < p.last && p.live) {
                if (a.gate) y *= gate[t] * pw::sigmoid(gate[t]);
                ((value_t*)a.out + (p.sequence * a.tokens + token + t) * a.channels)[p.channel] = (value_t)y;
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
        stage(tile, lds);
        float dy[T], dl[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float gate = a.gate ? (float)tile.gate[t] : 0.f;
            dy[t] = (float)tile.dout[t] * (a.gate ? gate * pw::sigmoid(gate) : 1.f);
            dl[t] = time_step(a, (float)tile.delta[t], bias);
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

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64, 64), amdgpu_waves_per_eu(SPIO_WAVES))) SPIO_KERNEL_NAME(const Args a) {
    __shared__ __attribute__((aligned(16))) float lds[T * 2 * NP];
    enum { U, DL, SLOPE, DY, DGATE, OWN };
    __shared__ float own[T][OWN][64];  // what a lane has of every token of the tile, out of the registers' way
    const int lane = (int)__builtin_amdgcn_workitem_id_x();
    const Place p = place(a);
    const int blocks = (int)((a.channels + 63) / 64);
    const long long tiles = (a.tokens + T - 1) / T;
    Tile tile;
    int token = p.first + (p.last - p.first - 1) / T * T;
    request<true, true, true, true>(tile, a, p, token);
    float A2[N], r[N], dA[N];
    rates(a, p, A2);
    const float bias = a.bias ? a.bias[p.loaded] : 0.f;
    const float D = a.D ? a.D[p.loaded] : 0.f;
    float dD = 0.f, dbias = 0.f;
#pragma unroll
    for (int s = 0; s < N; ++s) r[s] = dA[s] = 0.f;
    if (p.chunk + 1 < p.chunks) join(a, p, A2, r, true);
    const int mine = Sum<0, M>::index(lane);
    for (; token >= p.first; token -= T) {
        float h[N], q[T][N];  // q: exp(dl A) h of the token before
        const float* kept = a.kept + ((p.sequence * tiles + token / T) * N) * a.channels + p.loaded;
#pragma unroll
        for (int s = 0; s < N; ++s) h[s] = kept[s * a.channels];
        stage(tile, lds);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const bool there = token + t < p.last && p.live;
            const float raw = (float)tile.delta[t] + bias;
            const float dout = there ? (float)tile.dout[t] : 0.f;
            own[t][U][lane] = there ? (float)tile.u[t] : 0.f;
            own[t][DL][lane] = there ? time_step(a, (float)tile.delta[t], bias) : 0.f;
            own[t][SLOPE][lane] = a.softplus ? pw::sigmoid(raw) : 1.f;
            if (a.gate) {
                const float gate = (float)tile.gate[t], s = pw::sigmoid(gate), v = gate * s;
                own[t][DY][lane] = dout * v;
                own[t][DGATE][lane] = dout * __builtin_fmaf(v, 1.f - s, s);
            } else {
                own[t][DY][lane] = dout;
            }
        }
        if (token > p.first) request<true, true, true, true>(tile, a, p, token - T);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            float B[NP], C[NP];
            row_of(lds, t, 0, B);
            row_of(lds, t, 1, C);
            const float u = own[t][U][lane], dl = own[t][DL][lane], x = dl * u;
            float y = D * u;
#pragma unroll
            for (int s = 0; s < N; ++s) {
                q[t][s] = exp2_(dl * A2[s]) * h[s];
                h[s] = __builtin_fmaf(x, B[s], q[t][s]);
                y = __builtin_fmaf(C[s], h[s], y);
            }
            if (a.gate) own[t][DGATE][lane] *= y;
        }
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
            __builtin_amdgcn_sched_barrier(0);
            float B[NP], C[NP], sums[N];
            row_of(lds, t, 0, B);
            row_of(lds, t, 1, C);
            const float u = own[t][U][lane], dy = own[t][DY][lane];
            float dl = own[t][DL][lane];
            asm("" : "+v"(dl));  // (its exponentials are taken again: those of the way forth would take T * N registers)
            const float x = dl * u;
            float gB = 0.f, gq = 0.f;
#pragma unroll
            for (int s = 0; s < N; ++s) {
                const float g = __builtin_fmaf(C[s], dy, r[s]);
                sums[s] = halves<0>(x * g, dy * __builtin_fmaf(x, B[s], q[t][s]), lane);
                gB = __builtin_fmaf(g, B[s], gB);
                const float w = g * q[t][s];
                dA[s] = __builtin_fmaf(w, dl, dA[s]);
                gq = __builtin_fmaf(w, A2[s], gq);
                r[s] = exp2_(dl * A2[s]) * g;
            }
            const float total = Sum<1, N>::of(sums, lane);
            const float du = __builtin_fmaf(gB, dl, D * dy);
            const float ddelta = __builtin_fmaf(gB, u, gq * LN2) * own[t][SLOPE][lane];
            if (token + t < p.last) {
                dD = __builtin_fmaf(dy, u, dD);
                dbias += ddelta;
                const long long row = p.sequence * a.tokens + token + t;
                if (mine >= 0) a.token_sums[(row * blocks + p.block) * M + mine] = total;
                if (p.live) {
                    ((value_t*)a.du + row * a.channels)[p.channel] = (value_t)du;
                    ((value_t*)a.ddelta + row * a.channels)[p.channel] = (value_t)ddelta;
                    if (a.gate) ((value_t*)a.dgate + row * a.channels)[p.channel] = (value_t)own[t][DGATE][lane];
                }
            }
        }
    }
    if (!p.live) return;
    float* sums = a.channel_sums + (p.sequence * p.chunks + p.chunk) * (N + 2) * a.channels + p.channel;
#pragma unroll
    for (int s = 0; s < N; ++s) sums[s * a.channels] = dA[s];
    sums[N * a.channels] = dD;
    sums[(N + 1) * a.channels] = dbias;
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
    tk::column_sums({a.channel_sums, a.sums, a.sequences * chunks, a.channels, N, 2}, group - row_groups);
}

#else

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
        for (int i = 0; i < 4; ++i) h[i] = v[i], A2[i] = w[i] * LOG2E;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = part * 4 + i < N;
            h[i] = there ? before[part * 4 + i] : 0.f;
            A2[i] = there ? a.A[(long long)c * N + part * 4 + i] * LOG2E : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool there = part * 4 + i < N;
        B[i] = there ? (float)((const value_t*)a.B)[sequence * a.b_row + part * 4 + i] : 0.f;
        C[i] = there ? (float)((const value_t*)a.C)[sequence * a.c_row + part * 4 + i] : 0.f;
    }
    const float u = (float)((const value_t*)a.u)[sequence * a.u_row + c];
    const float gate = a.gate ? (float)((const value_t*)a.gate)[sequence * a.gate_row + c] : 0.f;
    const float dl = time_step(a, (float)((const value_t*)a.delta)[sequence * a.delta_row + c], a.bias ? a.bias[c] : 0.f);
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
        if (a.gate) y *= gate * pw::sigmoid(gate);
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
