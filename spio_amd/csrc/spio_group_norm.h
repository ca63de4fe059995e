// Geometry of the group norm kernels over channels-last tensors, and the sums over a workgroup (gfx950).
//
//   SPIO_GN_C, SPIO_GN_GROUPS   channels, groups
//   SPIO_GN_SLICE               channels that a workgroup works on: whole groups and whole blocks of 32 channels,
//                               or all of them; the last slice may have fewer
//   SPIO_GN_THREADS, SPIO_GN_UNITS   threads of a workgroup; units of eight channels that a lane holds
//   SPIO_GN_ROWS                pixels whose units the threads have at a time
//   SPIO_GN_EPS, SPIO_GN_HAS_WEIGHT, SPIO_GN_HAS_BIAS
//   SPIO_GN_KEPT                the input in the 8-bit form is written (forward) or read (backward)
//   SPIO_GN_SPLIT               images are cut into stretches of pixels, one workgroup each
//
// A workgroup's pixels form rows of ROWS: lane t has unit t % SUP of the pixels t / SUP + k * ROWS, the same eight channels
// of all of them, and loads of neighbouring lanes are neighbours in memory.
//
// The 8-bit form's blocks are up to 32 channels of one pixel; its exponents lie in rows of ceil(C / 32) bytes.  With
// relu a byte for every eight channels follows them in the row: bit e, whether the gradient of that output passes.  (Its
// derivative jumps at zero: the kept input is on the other side of it where the output is less than half a step.)
#ifndef SPIO_GROUP_NORM_H
#define SPIO_GROUP_NORM_H

#include "spio_pointwise.h"

#ifndef SPIO_GN_C
#error "SPIO_GN_C, SPIO_GN_GROUPS, SPIO_GN_SLICE, SPIO_GN_THREADS, SPIO_GN_UNITS are required"
#endif
#ifndef SPIO_GN_HAS_WEIGHT
#define SPIO_GN_HAS_WEIGHT 1
#endif
#ifndef SPIO_GN_HAS_BIAS
#define SPIO_GN_HAS_BIAS 1
#endif
#ifndef SPIO_GN_KEPT
#define SPIO_GN_KEPT 0
#endif
#ifndef SPIO_GN_SPLIT
#define SPIO_GN_SPLIT 0
#endif
#ifndef SPIO_GN_EPS
#define SPIO_GN_EPS 1e-5f
#endif

namespace gn {

constexpr int C = SPIO_GN_C;
constexpr int GROUPS = SPIO_GN_GROUPS;
constexpr int SLICE = SPIO_GN_SLICE;
constexpr int THREADS = SPIO_GN_THREADS;
constexpr int UN = SPIO_GN_UNITS;
constexpr int CG = C / GROUPS;                  // channels of a group
constexpr int SLICES = (C + SLICE - 1) / SLICE;
constexpr int GS = SLICE / CG;                  // groups of a slice
constexpr int SU = SLICE / 8;                   // units of a pixel's slice
// a block of the 8-bit form is four neighbouring lanes of one wave
constexpr int SUP = SPIO_GN_KEPT ? (SU + 3) / 4 * 4 : SU;
constexpr int ROWS = SPIO_GN_ROWS;
constexpr int SPAN = ROWS * UN;                 // pixels that a workgroup holds
constexpr int WAVES = THREADS / 64;
constexpr int BLOCKS = (C + 31) / 32;           // exponents of a pixel
constexpr bool kBits = SPIO_GN_KEPT && SPIO_ACT == 1;
constexpr int EXP_ROW = BLOCKS + (kBits ? C / 8 : 0);
static_assert(C % 8 == 0 && C % GROUPS == 0 && SLICE % 8 == 0 && SLICE % CG == 0 && SLICE <= C, "bad geometry");
static_assert(SLICE == C || SLICE % 32 == 0, "a block lies in one slice");
// Units that a lane has under way where it does not hold on to them (with 4, 6 or 8 of them 32n 48c 224x224 and 128n 96c
// 56x56 take as long or longer: what more units hide, fewer waves beside each other lose)
#ifndef SPIO_GN_DEPTH
#define SPIO_GN_DEPTH 3
#endif
constexpr int DEPTH = SPIO_GN_DEPTH < UN ? SPIO_GN_DEPTH : UN;
static_assert(THREADS % 64 == 0 && ROWS >= 1 && ROWS <= THREADS / SUP, "bad geometry");

// A lane's eight channels as the groups divide them: KEYS values for it, KEY_CHANNELS channels each, all of one group.
constexpr int KEYS = CG % 8 == 0 ? 1 : 8 % CG == 0 ? 8 / CG : 8;
constexpr int KEY_CHANNELS = 8 / KEYS;
constexpr int GROUP_KEYS = CG / KEY_CHANNELS;   // of a group

// Lanes of a wave that have the same channels add up by an exchange if their number is a power of two.
constexpr bool kFold = SUP <= 64 && (SUP & (SUP - 1)) == 0;
static_assert(!kFold || ROWS == THREADS / SUP, "lanes without a pixel are not folded in");
constexpr int SUM_ROWS = kFold ? WAVES : ROWS;  // what then is left to add

struct Place {
    int tid, sub, row;   // thread, unit in the slice, first pixel
    int image, slice, stretch;
    int channel;         // the first of the lane's eight
    bool live;           // it has channels and pixels
};

PW_DEVICE float lane_xor(float v, int mask) {
    const int lane = (int)__builtin_amdgcn_workitem_id_x() & 63;
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((lane ^ mask) << 2, __builtin_bit_cast(int, v)));
}
PW_DEVICE void sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// Workgroup `block` of `stretches` stretches an image: neighbours are slices of the same pixels, then stretches, then images.
// (Slices that are not whole lines share some.  Workgroups are dealt to the XCDs in turn, so neighbours have different
// L2s and meet in the memory-side cache; what that costs is in the rule that chooses the slices.)
PW_DEVICE Place place(unsigned block, unsigned stretches) {
    Place p;
    p.tid = (int)__builtin_amdgcn_workitem_id_x();
    p.sub = p.tid % SUP;
    p.row = p.tid / SUP;
    p.slice = SLICES == 1 ? 0 : (int)(block % SLICES);
    const unsigned rest = block / SLICES;
    p.stretch = SPIO_GN_SPLIT ? (int)(rest % stretches) : 0;
    p.image = (int)(SPIO_GN_SPLIT ? rest / stretches : rest);
    p.channel = p.slice * SLICE + p.sub * 8;
    p.live = p.row < ROWS && p.sub < SU && p.channel < C;
    return p;
}

// Sums over the workgroup of a lane's values for its KEYS keys: `sums[group of the slice]`, in the same order
// always.  Lanes that are not live have zeros.  `red` may be used again after the next barrier.
// (rows an odd number of 16 bytes apart: lanes that read one column of several rows meet different banks)
constexpr int RED_PITCH = ((SUP * KEYS + 3) / 4 | 1) * 4;
constexpr int RED_FLOATS = SUM_ROWS * RED_PITCH;
constexpr int group_lanes() {
    int lanes = 64;
    while (lanes > 1 && lanes * GS > THREADS) lanes /= 2;
    return lanes;
}
constexpr int key_lanes() {
    int lanes = 1;
    while (2 * lanes <= GROUP_KEYS && group_lanes() / lanes > SUM_ROWS) lanes *= 2;
    return lanes;
}
PW_DEVICE void group_sums(float (&v)[KEYS], const Place& p, float* red, float* sums) {
    if (kFold) {
#pragma unroll
        for (int m = SUP; m < 64; m <<= 1)
#pragma unroll
            for (int k = 0; k < KEYS; ++k) v[k] += lane_xor(v[k], m);
        if ((p.tid & 63) < SUP)
#pragma unroll
            for (int k = 0; k < KEYS; ++k) red[(p.tid >> 6) * RED_PITCH + p.sub * KEYS + k] = v[k];
    } else if (p.row < ROWS) {
#pragma unroll
        for (int k = 0; k < KEYS; ++k) red[p.row * RED_PITCH + p.sub * KEYS + k] = v[k];
    }
    sync();
    // the lanes of a group share its rows, and its keys where these are fewer
    constexpr int LANES = group_lanes();
    constexpr int BY_KEY = key_lanes();
    constexpr int BY_ROW = LANES / BY_KEY;
    const int part = p.tid % LANES;
    for (int g = p.tid / LANES; g < GS; g += THREADS / LANES) {
        float s = 0.f;
        for (int r = part / BY_KEY; r < SUM_ROWS; r += BY_ROW) {
            const float* from = red + r * RED_PITCH + g * GROUP_KEYS + part % BY_KEY;
#pragma unroll 8
            for (int e = 0; e < GROUP_KEYS; e += BY_KEY)
                if (GROUP_KEYS % BY_KEY == 0 || e + part % BY_KEY < GROUP_KEYS) s += from[e];
        }
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) s += lane_xor(s, m);
        if (part == 0) sums[g] = s;
    }
    sync();
}
// Key k of a lane belongs to this group of the slice.
PW_DEVICE int group_of(const Place& p, int k) { return (p.sub * KEYS + k) / GROUP_KEYS; }

// Eight values of a float32 [C] vector from `channel` on.
PW_DEVICE void load_vector(float (&v)[8], const float* vector, const Place& p) {
    const pw_rsrc rs = pw::buffer(vector, C * 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const pw_uint4 q = __builtin_amdgcn_raw_buffer_load_b128(rs, p.live ? (p.channel + 4 * h) * 4 : (int)pw::OOB, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = pw::as_float(q[e]);
    }
}

}  // namespace gn

#endif
