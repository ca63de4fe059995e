// Rotation of the heads of queries and keys by their positions, with or without a norm of every head before it (gfx950):
//
//   xhat = x rsqrt(mean(x^2) + eps),  n = xhat weight                       (SPIO_NORM; else n = x)
//   angle = position frequency[i];  a pair (n1, n2) of channels becomes
//   (n1 cos - n2 sin, n2 cos + n1 sin) scale,                               channels behind the pairs stay as they are
//
// Pair i is channels (2i, 2i + 1) (SPIO_INTERLEAVED) or (i, pairs + i).  Backward, the gradients are turned by the
// negative angle, then
//
//   g = dn weight,  dx = rstd (g - xhat mean(g xhat)),  dweight = sum dn xhat
//
//   SPIO_MODE 0  forward
//   SPIO_MODE 1  backward   sums over tokens and heads as partial sums, a row for every workgroup
//   SPIO_MODE 2  sums       the partial sums added up
//
// A lane has two units of eight channels of a head, those of eight pairs where these are rotated; LANES neighbouring lanes
// are a head, and a group of them has the same head numbers modulo `parts` of a token.  So cosines and sines are computed
// once for all of these, and the sums of a norm cross lanes of a row only.  Angles are taken in turns in float64 (a
// position of six digits leaves float32 no digits behind the turns), of which the fraction is exact in float32.
// HBM-bound: 2 + 2 bytes a value forward, 2 + 2 + 2 backward with norms for 16-bit types.  4n 2048l, 24 and 8 heads of 128
// channels with norms in bfloat16: forward 32 us (4.2 TB/s), backward 44 (4.6 TB/s; vector instructions issue in half of it), sums 4;
// 16385 tokens of 32 and 8 heads 73 (4.6 TB/s); 2n 4097l, 16 and 16 heads of 80 channels without, 29 and 30 (3.0 TB/s), twice what a
// copy takes: there is one item for each group of lanes, so that all of them read, turn and write at about the same time.  Traced, of
// two sets of tensors in turn; back to back over five sets 37, 48, 73 and 28.  It waits for memory, most for what it reads:
// without angles the passes took as long, without stores one of 36 us took 26.
#include "spio_tokens.h"

#ifndef SPIO_MODE
#error "SPIO_MODE, SPIO_HEAD, SPIO_NORM, SPIO_INTERLEAVED, SPIO_HEADS are required"
#endif

namespace {

using tk::value_t;
constexpr int D = SPIO_HEAD, UNITS = D / 8;
constexpr int PAIRED = (UNITS + 1) / 2;  // lanes of a head that have channels
// (a norm's sums cross a power of two of lanes)
constexpr int LANES = !SPIO_NORM ? PAIRED : PAIRED <= 1 ? 1 : PAIRED <= 2 ? 2 : PAIRED <= 4 ? 4 : PAIRED <= 8 ? 8 : 16;
constexpr int GROUPS = 256 / LANES;      // of a workgroup
constexpr int U = SPIO_HEADS;            // heads requested at once
constexpr bool BACK = SPIO_MODE == 1;
constexpr bool FULL = UNITS == 2 * LANES;  // no lane is without channels
// Whether the first heads of both tensors are requested before a token's angles are computed, or of k behind those of q: a
// backward pass with norms has no registers for that (4n 2048l 24q 8k 128d 51 us, else 48)
constexpr bool AHEAD = !(BACK && SPIO_NORM);
static_assert(D % 8 == 0 && D <= 256, "heads of up to 256 channels, whole units");

// cos and sin of a fraction of a turn in [-1/2, 1/2]: the nearest quarter turn, and the Taylor series of what is left, at
// most pi / 4 (next terms 2e-10 and 2e-9)
__device__ inline void cos_sin(float turn, float& c, float& s) {
    const float quarter = __builtin_rintf(turn * 4.f);
    const float x = __builtin_fmaf(quarter, -0.25f, turn) * 6.28318531f, q = x * x;
    float sine = 2.75573192e-6f, cosine = -2.75573192e-7f;
    sine = __builtin_fmaf(sine, q, -1.98412698e-4f);
    sine = __builtin_fmaf(sine, q, 8.33333333e-3f);
    sine = __builtin_fmaf(sine, q, -0.166666667f);
    sine = __builtin_fmaf(sine * q, x, x);
    cosine = __builtin_fmaf(cosine, q, 2.48015873e-5f);
    cosine = __builtin_fmaf(cosine, q, -1.38888889e-3f);
    cosine = __builtin_fmaf(cosine, q, 4.16666667e-2f);
    cosine = __builtin_fmaf(cosine, q, -0.5f);
    cosine = __builtin_fmaf(cosine, q, 1.f);
    const int k = (int)quarter;
    const float even = k & 1 ? sine : cosine, odd = k & 1 ? cosine : sine;
    c = (k + 1) & 2 ? -even : even;
    s = k & 2 ? -odd : odd;
}

// The two units of a lane (-1: none), and the first of the pairs in each of them that neighbours make (SPIO_INTERLEAVED:
// four), or of the eight pairs that both make
struct Place {
    int unit[2], pair[2], pairs;
    bool rotated;  // (SPIO_INTERLEAVED: the pairs before `pairs` are)
};
__device__ inline Place place(int lane, int pairs) {
    Place p;
    const int half = pairs / 8;
    p.pairs = pairs;
    p.rotated = SPIO_INTERLEAVED || lane < half;
    p.unit[0] = SPIO_INTERLEAVED ? 2 * lane : lane < half ? lane : half + lane;
    p.unit[1] = SPIO_INTERLEAVED ? 2 * lane + 1 : lane < half ? half + lane : PAIRED + lane;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        p.pair[i] = SPIO_INTERLEAVED ? 4 * p.unit[i] : 8 * lane + 4 * i;
        if (lane >= PAIRED || p.unit[i] >= UNITS) p.unit[i] = -1;
    }
    return p;
}
__device__ inline int pair_of(const Place& p, int i) { return p.pair[i / 4] + i % 4; }

// (v[0], v[1]) turned by the angles.  A pair behind the rotated ones (PART: there are such) is left alone: its sine of zero
// times an infinity is none.
template <bool PART>
__device__ inline void rotate_pairs(float (&v)[2][8], const float (&c)[8], const float (&s)[8], const Place& p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float& a = SPIO_INTERLEAVED ? v[i / 4][i % 4 * 2] : v[0][i];
        float& b = SPIO_INTERLEAVED ? v[i / 4][i % 4 * 2 + 1] : v[1][i];
        const bool there = !PART || pair_of(p, i) < p.pairs;
        const float turned = a * c[i] - b * s[i], other = __builtin_fmaf(a, s[i], b * c[i]);
        a = there ? turned : a;
        b = there ? other : b;
    }
}
__device__ inline void rotate(float (&v)[2][8], const float (&c)[8], const float (&s)[8], const Place& p) {
    if (SPIO_INTERLEAVED && 2 * p.pairs < D)
        rotate_pairs<true>(v, c, s, p);
    else if (p.rotated)
        rotate_pairs<false>(v, c, s, p);
}

struct Rows {
    const value_t *x, *dy;
    value_t* out;
    long long row, head;  // of x
    int heads;
};

// U heads of a token as they are in memory: `head`, head + parts, ...; those behind the last one in the place of which that
// is read, and the first unit in the place of none.  No branch is in the way, so that a wait is for what is needed alone.
struct Batch {
    pw::Unit x[U][2], dy[U][2];
};
__device__ inline void request(Batch& b, const Rows& r, const Place& p, long long token, int head, int parts) {
    const value_t* x = r.x + token * r.row;
    const value_t* dy = r.dy + token * r.heads * D;
#pragma unroll
    for (int h = 0; h < U; ++h) {
        const int last = r.heads ? r.heads - 1 : 0, at = head + h * parts < last ? head + h * parts : last;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int unit = FULL || p.unit[i] >= 0 ? p.unit[i] : 0;
            b.x[h][i] = b.dy[h][i] = pw::Unit{};
            if (SPIO_NORM || !BACK) b.x[h][i] = tk::load(x + at * r.head + unit * 8);
            if (BACK) b.dy[h][i] = tk::load(dy + at * D + unit * 8);
        }
    }
}
__device__ inline void work_on(const Batch& b, const Rows& r, const Place& p, long long token, int head, int parts,
                               const float (&c)[8], const float (&s)[8], const float (&w)[2][8], float eps, float (&dw)[2][8]) {
#pragma unroll
    for (int h = 0; h < U; ++h) {
        const bool there = head + h * parts < r.heads;
        float v[2][8], g[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            tk::values(b.x[h][i], v[i]);
            tk::values(b.dy[h][i], g[i]);
            if (SPIO_NORM && !FULL && p.unit[i] < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = g[i][e] = 0.f;
            }
        }
        if (SPIO_NORM) {
            float squares = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(v[i][e], v[i][e], squares);
            squares = tk::sum_of<LANES>(squares);
            const float rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(squares, 1.f / D, eps));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= rstd;
            if (BACK) {
                rotate(g, c, s, p);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (there) dw[i][e] = __builtin_fmaf(g[i][e], v[i][e], dw[i][e]);
                        g[i][e] *= w[i][e];
                        dot = __builtin_fmaf(g[i][e], v[i][e], dot);
                    }
                dot = tk::sum_of<LANES>(dot) * (1.f / D);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[i][e] = rstd * __builtin_fmaf(-dot, v[i][e], g[i][e]);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] *= w[i][e];
                rotate(v, c, s, p);
            }
        } else if (BACK) {
            rotate(g, c, s, p);
        } else {
            rotate(v, c, s, p);
        }
        value_t* out = r.out + (token * r.heads + head + h * parts) * D;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            // (past the caches: 2n 4097l 16q 16k 80d 28 us, else 34)
            if (there && (FULL || p.unit[i] >= 0)) tk::store<true>(out + p.unit[i] * 8, pw::pack(BACK ? g[i] : v[i]));
    }
}

// What was requested before is not moved behind what follows
__device__ inline void pinned() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// The heads `part`, `part + parts`, ... of a token, of which the first batch has been requested.  The next one is requested before
// the present one is worked on (behind the last one that is read again): its wait would be for the stores before it, too.
__device__ inline void heads_of(Batch& b, const Rows& r, const Place& p, long long token, int part, int parts,
                                const float (&c)[8], const float (&s)[8], const float (&w)[2][8], float eps, float (&dw)[2][8]) {
    for (int head = part; head < r.heads; head += parts * U) {
        Batch next;
        request(next, r, p, token, head + parts * U, parts);
        pinned();
        work_on(b, r, p, token, head, parts, c, s, w, eps, dw);
        b = next;
    }
}

__device__ inline void weights(const float* from, const Place& p, float (&w)[2][8]) {
    typedef float float4_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const bool there = FULL || p.unit[i] >= 0;
            const float4_t v = from ? *(const float4_t*)(from + (there ? p.unit[i] : 0) * 8 + e) : float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k) w[i][e + k] = there ? v[k] : 0.f;
        }
}

}  // namespace

#if SPIO_MODE < 2

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const SpioRotaryArgs a) {
    const int tid = (int)__builtin_amdgcn_workitem_id_x(), lane = tid % LANES, group = tid / LANES;
    if (group >= GROUPS) return;  // (not with norms)
    const int pairs = (int)a.pairs, parts = (int)a.parts, wide = (int)a.wide_positions;
    const Place p = place(lane, pairs);
    const float eps = __builtin_fmaxf((float)a.eps, 1.17549435e-38f);  // (less counts as the smallest normal number)
    Rows q = {(const value_t*)a.q, (const value_t*)a.dq, (value_t*)a.q_out, a.q_row, a.q_head, (int)a.q_heads};
    Rows k = {(const value_t*)a.k, (const value_t*)a.dk, (value_t*)a.k_out, a.k_row, a.k_head, (int)a.k_heads};
    if (!q.heads) q.x = k.x, q.dy = k.dy, q.row = k.row;
    if (!k.heads) k.x = q.x, k.dy = q.dy, k.row = q.row;
    float wq[2][8], wk[2][8], dwq[2][8] = {}, dwk[2][8] = {};
    weights(SPIO_NORM ? a.q_weight : nullptr, p, wq);
    weights(SPIO_NORM ? a.k_weight : nullptr, p, wk);
    // (those of lanes and pairs that are not rotated are not used; nothing here waits for what is loaded, or the heads would
    // be requested later)
    double frequency[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) frequency[i] = a.frequencies[pair_of(p, i) < pairs ? pair_of(p, i) : 0];
    const unsigned groups = __builtin_amdgcn_grid_size_x() / 256 * GROUPS, items = (unsigned)(a.tokens * parts);  // (fewer than 2^31)
    // (a group's lanes stay together: they cross lanes for the norm)
    for (unsigned item = __builtin_amdgcn_workgroup_id_x() * GROUPS + group; item < items; item += groups) {
        const unsigned token = item / (unsigned)parts;
        const int part = (int)(item % (unsigned)parts);
        const unsigned at = token < (unsigned)a.position_tokens ? token : token % (unsigned)a.position_tokens;
        // (requested before the heads: loads come back in their order.  Of an int64 the halves apart, of an int32 the one)
        const int* slot = (const int*)a.positions + (unsigned long long)at * (unsigned)(1 + wide);
        const int low = slot[0], high = slot[wide];
        Batch q_heads, k_heads;
        request(q_heads, q, p, token, part, parts);
        if (AHEAD) request(k_heads, k, p, token, part, parts);
        pinned();
        const double position = wide ? __builtin_fma((double)high, 4294967296., (double)(unsigned)low) : (double)low;
        const double turned = position * 0.15915494309189535;  // by a frequency of one
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double turns = turned * frequency[i];
            cos_sin((float)(turns - __builtin_rint(turns)), c[i], s[i]);
            c[i] *= (float)a.scale, s[i] *= BACK ? -(float)a.scale : (float)a.scale;
        }
        heads_of(q_heads, q, p, token, part, parts, c, s, wq, eps, dwq);
        if (!AHEAD) request(k_heads, k, p, token, part, parts);
        heads_of(k_heads, k, p, token, part, parts, c, s, wk, eps, dwk);
    }
#if SPIO_MODE == 1 && SPIO_NORM
    // the groups of a workgroup, one after the other
    __shared__ float sums[GROUPS][D];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        tk::barrier();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (p.unit[i] >= 0) sums[group][p.unit[i] * 8 + e] = which ? dwk[i][e] : dwq[i][e];
        tk::barrier();
        for (int d = tid; d < D; d += 256) {
            float sum = 0.f;
#pragma unroll 8
            for (int g = 0; g < GROUPS; ++g) sum += sums[g][d];
            a.partials[((long long)__builtin_amdgcn_workgroup_id_x() * 2 + which) * D + d] = sum;
        }
    }
#endif
}

#else

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256))) SPIO_KERNEL_NAME(const SpioRotaryArgs a) {
    // (`parts` has the rows)
    tk::column_sums({a.partials, a.parts, D, 0, 2, nullptr, a.dq_weight, a.dk_weight}, __builtin_amdgcn_workgroup_id_x());
}

#endif
