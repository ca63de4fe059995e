// What the kernels of element-wise work and of channels-last norms share (gfx950): units of eight values in one
// of three types, activations, and the 8-bit form that a tensor is kept in between its two passes.
//
//   SPIO_DTYPE  0 float16, 1 bfloat16, 2 float32: the tensors' type; all arithmetic is in float32
//   SPIO_ACT    0 none, 1 relu, 2 silu, 3 gelu (the one of the normal distribution, not tanh's)
//
// 8-bit form.  A block is up to 32 neighbouring values; it is held as one signed byte a value (its code) and one
// byte for the block (its exponent, biased by 127):
//   E     = the smallest exponent with max|x| < 127.5 * 2^(E-6), at least 7-127; byte E+127
//   code  = x / 2^(E-6) to the nearest integer, ties to even: -127..127
//   value = code * 2^(E-6)
// A step is a power of two, so that quotient, product and the rounding are exact in float32 and a block is off by
// half a step at most: 1/127.5 of its largest value, or 2^-127 where that is more.  (Values of more than 127.5 steps of the
// largest exponent are held as 127.)  Byte 255 marks a block that held an infinity or a NaN;
// all of it comes back as NaN.
#ifndef SPIO_POINTWISE_H
#define SPIO_POINTWISE_H

#ifndef SPIO_DTYPE
#error "SPIO_DTYPE is required"
#endif
#ifndef SPIO_ACT
#define SPIO_ACT 0
#endif

typedef unsigned int pw_uint2 __attribute__((ext_vector_type(2)));
typedef unsigned int pw_uint4 __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t pw_rsrc;

namespace pw {

#define PW_DEVICE __device__ inline __attribute__((always_inline))

constexpr int VALUE_BYTES = SPIO_DTYPE == 2 ? 4 : 2;
constexpr int QUADS = SPIO_DTYPE == 2 ? 2 : 1;  // 16-byte words of a unit
constexpr int UNIT_BYTES = 16 * QUADS;
constexpr unsigned OOB = 0x80000000u;           // an offset behind the end of every descriptor
constexpr int STREAM = 2;                       // cache policy of what is read or written once

PW_DEVICE float as_float(unsigned u) { return __builtin_bit_cast(float, u); }
PW_DEVICE unsigned as_bits(float f) { return __builtin_bit_cast(unsigned, f); }

// Bytes [base, base + bytes) as a buffer: loads behind its end give zeros, stores there are dropped.
PW_DEVICE pw_rsrc buffer(const void* base, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

struct Unit {
    pw_uint4 q[QUADS];
};

template <int POLICY>
PW_DEVICE Unit load_unit(pw_rsrc rs, unsigned off) {
    Unit u;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) u.q[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + 16 * i), 0, POLICY);
    return u;
}
// (The offset is in a vector register and the scalar one stays constant: 16-byte stores with a scalar offset can
// store their data registers as they are after a following write.)
template <int POLICY>
PW_DEVICE void store_unit(pw_rsrc rs, unsigned off, const Unit& u) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) __builtin_amdgcn_raw_buffer_store_b128(u.q[i], rs, (int)(off + 16 * i), 0, POLICY);
}

// What is done with a unit behind this starts from its registers again: values converted ahead of it would take two to
// four times as many in between.
PW_DEVICE void keep_packed(Unit& u) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) asm volatile("" : "+v"(u.q[i]));
}

typedef _Float16 pw_half2 __attribute__((ext_vector_type(2)));
typedef _Float16 pw_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 pw_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pw_float2 __attribute__((ext_vector_type(2)));

PW_DEVICE float value(const Unit& u, int e) {
    if (SPIO_DTYPE == 2) return as_float(u.q[e / 4 % QUADS][e % 4]);
    if (SPIO_DTYPE == 1) return as_float(e % 2 ? u.q[0][e / 2] & 0xffff0000u : u.q[0][e / 2] << 16);
    return (float)__builtin_bit_cast(pw_half8, u.q[0])[e];
}
// The vector units are what most of these kernels wait for, so instructions count: a float16 value enters a
// mixed-precision multiply-add instead of being converted, in products with a 1 and sums with a -0 that the compiler
// does not know for such.
struct Constants {
    float one = 1.f, zero = -0.f;
    PW_DEVICE Constants() { asm("" : "+s"(one), "+s"(zero)); }
};
PW_DEVICE float plus(const Unit& u, int e, float c, const Constants& k) {  // value + c
    return SPIO_DTYPE == 0 ? __builtin_fmaf(value(u, e), k.one, c) : value(u, e) + c;
}
PW_DEVICE float times(const Unit& u, int e, float f, const Constants& k) {  // value * f
    return SPIO_DTYPE == 0 ? __builtin_fmaf(value(u, e), f, k.zero) : value(u, e) * f;
}

// Rounds to nearest, ties to even.
PW_DEVICE Unit pack(const float (&v)[8]) {
    Unit u;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const pw_float2 pair = {v[e], v[e + 1]};
        if (SPIO_DTYPE == 2) {
            u.q[e / 4 % QUADS][e % 4] = as_bits(v[e]);
            u.q[e / 4 % QUADS][e % 4 + 1] = as_bits(v[e + 1]);
        } else if (SPIO_DTYPE == 1) {
            u.q[0][e / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector(pair, pw_bf16x2));
        } else {
            u.q[0][e / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector(pair, pw_half2));
        }
    }
    return u;
}

// 1 / v to the last place or nearly
PW_DEVICE float reciprocal(float v) {
    const float r = __builtin_amdgcn_rcpf(v);
    return __builtin_fmaf(__builtin_fmaf(-v, r, 1.f), r, r);
}

// s / n for a count n with r = reciprocal(n), exact where s is a multiple of n: the mean of n equal values is that value, and
// they have no difference to it (s * r may be a step off, which is a whole deviation where there is no other).
PW_DEVICE float quotient(float s, float n, float r) {
    const float q = s * r;
    return __builtin_fmaf(__builtin_fmaf(-q, n, s), r, q);
}

// ---- activations ----

// 1 / (1 + exp(-z)); the hardware's exponential and reciprocal are within a unit in the last place.
PW_DEVICE float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

// The normal distribution at z: exp(-z^2 / 2) and the upper tail at |z|, which is that times R(|z|); R falls smoothly from
// a half like 1/|z|: a polynomial in t = 1 / (1 + p|z|), fitted to its values (scipy's erfcx) at Chebyshev points of t for
// |z| <= 14 by reweighted least squares.  Relative error of the tail 1.5e-7, or 4.6e-6 with two degrees less, which is for
// single results in 16 bits: sums of many show it (grad_bias of 16n 24c 144x144 was off by 1.6e-6 of its norm for 4e-7).
template <bool SHORT>
PW_DEVICE void normal(float z, float& e, float& tail) {
    const float a = __builtin_fabsf(z);
    e = __builtin_amdgcn_exp2f(a * a * -0.721347520f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, SHORT ? 0.31f : 0.3f, 1.f));
    float r;
    if (SHORT) {
        r = -0.07392936f;
        r = __builtin_fmaf(r, t, 0.18045098f);
        r = __builtin_fmaf(r, t, 0.01574401f);
        r = __builtin_fmaf(r, t, 0.13343013f);
        r = __builtin_fmaf(r, t, 0.1204412f);
        r = __builtin_fmaf(r, t, 0.12386071f);
    } else {
        r = 0.03567488f;
        r = __builtin_fmaf(r, t, -0.1572035f);
        r = __builtin_fmaf(r, t, 0.2063542f);
        r = __builtin_fmaf(r, t, -0.05368425f);
        r = __builtin_fmaf(r, t, 0.12856192f);
        r = __builtin_fmaf(r, t, 0.09991341f);
        r = __builtin_fmaf(r, t, 0.12075397f);
        r = __builtin_fmaf(r, t, 0.1196293f);
    }
    tail = e * (r * t);
}

PW_DEVICE float activate(float z) {
    if (SPIO_ACT == 1) return z < 0.f ? 0.f : z;  // (NaN stays)
    if (SPIO_ACT == 2) return z * sigmoid(z);
    if (SPIO_ACT == 3) {
        float e, tail;
        normal<SPIO_DTYPE != 2>(z, e, tail);
        return z * (z < 0.f ? tail : 1.f - tail);
    }
    return z;
}

// Whether relu's gradient at z is the output's (as torch has it: at NaN it is)
PW_DEVICE bool passes(float z) { return !(z <= 0.f); }

// value e of dy times the activation's derivative at z (SHORT as in normal)
template <bool SHORT>
PW_DEVICE float activate_grad(const Unit& dy, int e, float z, const Constants& k) {
    if (SPIO_ACT == 1) return passes(z) ? value(dy, e) : 0.f;
    if (SPIO_ACT == 2) {
        const float s = sigmoid(z);
        return times(dy, e, __builtin_fmaf(s, __builtin_fmaf(-z, s, z), s), k);  // s + s z (1 - s)
    }
    if (SPIO_ACT == 3) {
        float density, tail;
        normal<SHORT>(z, density, tail);
        return times(dy, e, __builtin_fmaf(z, density * 0.398942280f, z < 0.f ? tail : 1.f - tail), k);
    }
    return value(dy, e);
}

// ---- 8-bit form ----

// Bits of the largest magnitude of a unit, in the order of the tensors' type (a NaN's are the largest).
PW_DEVICE unsigned largest(const Unit& u) {
    if (SPIO_DTYPE == 2) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < QUADS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned w = u.q[i][j] & 0x7fffffffu;
                m = m > w ? m : w;
            }
        return m;
    }
    typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
    ushort2_t m = __builtin_bit_cast(ushort2_t, u.q[0][0] & 0x7fff7fffu);
#pragma unroll
    for (int j = 1; j < 4; ++j)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, u.q[0][j] & 0x7fff7fffu));
    return m[0] > m[1] ? m[0] : m[1];
}
template <int CTRL>
PW_DEVICE unsigned dpp_max(unsigned v) {
    const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
    return v > other ? v : other;
}
// The exponent byte of the block that four neighbouring lanes hold a unit of each.
PW_DEVICE unsigned block_exponent(const Unit& u) {
    unsigned m = largest(u);
    m = dpp_max<0xB1>(m);  // quad_perm [1,0,3,2]
    m = dpp_max<0x4E>(m);  // quad_perm [2,3,0,1]
    if (SPIO_DTYPE == 1) m <<= 16;
    if (SPIO_DTYPE == 0) m = as_bits((float)__builtin_bit_cast(_Float16, (unsigned short)m));
    // adding a 128th of a unit carries into the exponent where the mantissa is 127.5/64 or more
    const unsigned e = (m + 0x10000u) >> 23;
    const unsigned in_range = e < 7 ? 7 : e > 254 ? 254 : e;
    return m >= 0x7f800000u ? 255 : in_range;
}
// The codes of a unit, by a product and a sum whose low byte is the integer (1.5 * 2^23 has a unit of one there).
PW_DEVICE pw_uint2 encode(Unit u, unsigned exponent) {
    const float inverse = as_float((260u - exponent) << 23);
    if (SPIO_DTYPE != 0 && __builtin_amdgcn_ballot_w64(exponent == 254)) {
        // values behind 127 steps of the largest exponent are held as that
        constexpr float limit = 0x1.fcp127f;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_fmed3f(value(u, e), -limit, limit);
        u = pack(x);
    }
    unsigned r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = as_bits(__builtin_fmaf(value(u, e), inverse, 12582912.f));
    pw_uint2 codes;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        // bytes 0 and 4 of two registers, then bytes 0, 1, 4, 5
        const unsigned lo = __builtin_amdgcn_perm(r[4 * h + 1], r[4 * h], 0x0c0c0400u);
        const unsigned hi = __builtin_amdgcn_perm(r[4 * h + 3], r[4 * h + 2], 0x0c0c0400u);
        codes[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
    return codes;
}
// The step of an exponent byte; NaN for that of a block without a value.
PW_DEVICE float block_step(unsigned exponent) {
    const unsigned e = exponent < 7 ? 7 : exponent;
    unsigned bits = exponent == 255 ? 0x7fc00000u : (e - 6) << 23;
    asm("" : "+v"(bits));  // (the choice would be made of every value's product instead)
    return as_float(bits);
}
PW_DEVICE float code(const pw_uint2& codes, int e) { return (float)(signed char)(codes[e / 4] >> 8 * (e % 4)); }

}  // namespace pw

#endif
