// Element-wise work on dense tensors with an 8-bit checkpoint (gfx950):
//
//   SPIO_MODE 0  forward    y = act(x), and x in the 8-bit form (SPIO_KEEP)      (y, codes, exponents, x, n)
//   SPIO_MODE 1  backward   dx = dy * act'(x as it was kept)                     (dx, codes, exponents, dy, n)
//                (relu keeps a bit a value in place of the codes, whether its gradient passes: its derivative jumps at
//                zero, where half a step of the 8-bit form would lose it whole; there are no exponents)
//   SPIO_MODE 2  pack       x in the 8-bit form                                  (codes, exponents, x, n)
//   SPIO_MODE 3  unpack     the values that codes and exponents stand for        (x, codes, exponents, n)
//
// A block of the 8-bit form is 32 neighbours in memory, the last one what is left (spio_pointwise.h).
//
// HBM-bound: 2 + 2 + 1 bytes a value forward, 2 + 1 + 2 backward for 16-bit types.  A lane holds units of eight
// values, so that loads are 16 bytes and four neighbouring lanes hold a block: its largest magnitude is two
// steps through the data-parallel-primitive operand path, nothing meets in LDS.  A workgroup has one stretch of
// THREADS * UNROLL units, all requested before the first is worked on: 256 * 2, which beats larger ones by up to a tenth.
// 128n 384c 56x56 with gelu, 776 MB each way, forward 140-148 us (5.2-5.5 TB/s) and backward 138 by themselves, 246 one after
// the other, where the checkpoint comes from the memory-side cache; vector instructions take as long (23 and 22 a value)
// and run beside the loads.  With relu, 636 MB each way, 98 and 97 us (6.5 TB/s), 194 one after the other.  128n 64c 56x56,
// 78 MB each way: pack 13.1-15.0 us (5.2-5.9 TB/s), unpack 13.2-15.8.
#include "spio_pointwise.h"

#ifndef SPIO_MODE
#error "SPIO_MODE, SPIO_THREADS, SPIO_UNROLL are required"
#endif
#ifndef SPIO_KEEP
#define SPIO_KEEP 0
#endif

namespace {

constexpr int THREADS = SPIO_THREADS;
constexpr int UN = SPIO_UNROLL;
constexpr bool kReadsValues = SPIO_MODE != 3;
constexpr bool kBits = SPIO_ACT == 1 && SPIO_MODE < 2;  // a byte a unit, bit e that of its value e
constexpr bool kReadsCodes = (SPIO_MODE == 1 && !kBits) || SPIO_MODE == 3;
constexpr bool kWritesCodes = SPIO_MODE == 2 || (SPIO_MODE == 0 && SPIO_KEEP && !kBits);
constexpr bool kReadsBits = SPIO_MODE == 1 && kBits, kWritesBits = SPIO_MODE == 0 && SPIO_KEEP && kBits;
constexpr bool kWritesValues = SPIO_MODE != 2;

#if SPIO_DTYPE == 2
typedef unsigned value_t;
#else
typedef unsigned short value_t;
#endif

// The largest float16 values round up to 64 steps of 1024, which is none: they come back as the largest (and NaN as NaN).
PW_DEVICE float finite(float v) {
    if (SPIO_DTYPE != 0) return v;
    v = v > 65504.f ? 65504.f : v;
    return v < -65504.f ? -65504.f : v;
}

// Values [0, count) of a last unit that is not whole.
PW_DEVICE pw::Unit load_part(const value_t* p, int count) {
    pw::Unit u = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < count) {
            const unsigned w = p[e];
            if (SPIO_DTYPE == 2)
                u.q[e / 4 % pw::QUADS][e % 4] = w;
            else
                u.q[0][e / 2] |= w << (e % 2 * 16);
        }
    return u;
}
PW_DEVICE void store_part(value_t* p, const pw::Unit& u, int count) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < count)
            p[e] = (value_t)(SPIO_DTYPE == 2 ? u.q[e / 4 % pw::QUADS][e % 4] : u.q[0][e / 2] >> (e % 2 * 16));
}

}  // namespace

extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS)))
SPIO_KERNEL_NAME(
#if SPIO_MODE == 2
    unsigned char* __restrict__ codes, unsigned char* __restrict__ exponents, const value_t* __restrict__ in,
#elif SPIO_MODE == 3
    value_t* __restrict__ out, unsigned char* __restrict__ codes, unsigned char* __restrict__ exponents,
#else
    value_t* __restrict__ out, unsigned char* __restrict__ codes, unsigned char* __restrict__ exponents,
    const value_t* __restrict__ in,
#endif
    long long n) {
#if SPIO_MODE == 2
    value_t* out = nullptr;
#elif SPIO_MODE == 3
    const value_t* in = nullptr;
#endif
    const int tid = (int)__builtin_amdgcn_workitem_id_x();
    const long long first = (long long)__builtin_amdgcn_workgroup_id_x() * (THREADS * UN);  // unit
    const long long left = n - first * 8;  // values from there on, at least one
    const int values = (int)(left < THREADS * UN * 8 ? left : THREADS * UN * 8);
    const int whole = values / 8, part = values % 8;
    const pw_rsrc rs_in = pw::buffer(in + first * 8, kReadsValues ? whole * pw::UNIT_BYTES : 0);
    const pw_rsrc rs_out = pw::buffer(out + first * 8, kWritesValues ? whole * pw::UNIT_BYTES : 0);
    const pw_rsrc rs_codes = pw::buffer(codes + first * 8, kReadsCodes || kWritesCodes ? whole * 8 : 0);
    const pw_rsrc rs_exp = pw::buffer(exponents + first / 4, kReadsCodes || kWritesCodes ? (values + 31) / 32 : 0);
    const pw_rsrc rs_bits = pw::buffer(codes + first, kReadsBits || kWritesBits ? (values + 7) / 8 : 0);

    const pw::Constants constants;
    pw::Unit v[UN];
    pw_uint2 c[UN];
    unsigned ex[UN], bits[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int unit = u * THREADS + tid;
        if (kReadsValues) v[u] = pw::load_unit<pw::STREAM>(rs_in, unit * pw::UNIT_BYTES);
        if (kReadsCodes) {
            c[u] = __builtin_amdgcn_raw_buffer_load_b64(rs_codes, unit * 8, 0, pw::STREAM);
            ex[u] = __builtin_amdgcn_raw_buffer_load_b8(rs_exp, unit / 4, 0, 0);
        }
        if (kReadsBits) bits[u] = __builtin_amdgcn_raw_buffer_load_b8(rs_bits, unit, 0, 0);
    }
    if (part) {  // the last unit of the tensor
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int unit = u * THREADS + tid;
            if (unit != whole) continue;
            if (kReadsValues) v[u] = load_part(in + (first + unit) * 8, part);
            if (kReadsCodes) {
                c[u] = pw_uint2{0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < part) c[u][e / 4] |= (unsigned)codes[(first + unit) * 8 + e] << (e % 4 * 8);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int unit = u * THREADS + tid;
        if (kWritesCodes) {
            ex[u] = pw::block_exponent(v[u]);
            c[u] = pw::encode(v[u], ex[u]);
            __builtin_amdgcn_raw_buffer_store_b64(c[u], rs_codes, unit * 8, 0, pw::STREAM);
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)ex[u], rs_exp, tid % 4 == 0 ? unit / 4 : (int)pw::OOB, 0, 0);
        }
        if (kWritesBits) {
            bits[u] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) bits[u] |= pw::passes(pw::value(v[u], e)) ? 1u << e : 0u;
            __builtin_amdgcn_raw_buffer_store_b8((unsigned char)bits[u], rs_bits, unit, 0, 0);
        }
        if (kWritesValues) {
            float y[8];
            const float step = kReadsCodes ? pw::block_step(ex[u]) : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (kReadsBits)
                    y[e] = bits[u] >> e & 1 ? pw::value(v[u], e) : 0.f;
                else if (SPIO_MODE == 1)
                    y[e] = pw::activate_grad<SPIO_DTYPE != 2>(v[u], e, pw::code(c[u], e) * step, constants);
                else if (SPIO_MODE == 3)
                    y[e] = finite(pw::code(c[u], e) * step);
                else
                    y[e] = pw::activate(pw::value(v[u], e));
            }
            v[u] = pw::pack(y);
            pw::store_unit<pw::STREAM>(rs_out, unit * pw::UNIT_BYTES, v[u]);
        }
    }
    if (part) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int unit = u * THREADS + tid;
            if (unit != whole) continue;
            if (kWritesValues) store_part(out + (first + unit) * 8, v[u], part);
            if (kWritesCodes) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < part) codes[(first + unit) * 8 + e] = (unsigned char)(c[u][e / 4] >> (e % 4 * 8));
            }
        }
    }
}
