// What the kernels over an 8-bit KV cache in blocks share (include/leafhip.h:
// lh_kv_batch, lh_kv8): which requests of a batch a kernel may follow, and the
// codes' arithmetic.
#pragma once
#include "device_common.h"
#include "kernels.h"

namespace leafhip {

// A request's rows of the step, [start, start + rows), of `length` keys; rows
// is 0 where the arrays, which may come from anywhere, name rows or keys that
// the batch has no room for.
struct Kv8Request {
    int start, rows, length;
};
__device__ __forceinline__ Kv8Request kv8_request(const KvBatchView& b, int r) {
    Kv8Request q{b.starts[r], b.rows[r], b.lengths[r]};
    const bool fits = q.rows > 0 && q.rows <= b.max_rows && q.start >= 0 && q.start <= b.tokens - q.rows &&
                      q.length >= q.rows && q.length <= (long long)b.width << b.block_shift;
    if (!fits) q.rows = 0;
    return q;
}

__device__ __forceinline__ bool finite_f32(float v) { return __builtin_fabsf(v) < INFINITY; }

// x / scale to the nearest whole number, ties to even, for |x| <= 127 scale
// (1 + 2^-24): x * (1 / scale) rounds to it or, next to a border, to a
// neighbour; x - q * scale is exact (a multiple of the smaller ulp, less than
// scale), and decides.  (Of a NaN any code.)
__device__ __forceinline__ int nearest_i8(float x, float scale, float inverse) {
    float q = __builtin_rintf(x * inverse);
    const float rest = fmaf(-q, scale, x), twice = 2.0f * __builtin_fabsf(rest);
    if (twice > scale || (twice == scale && ((int)q & 1))) q += __builtin_copysignf(1.0f, rest);
    return (int)q;
}

// The smallest power of two, from 2^-40, times which 448 is at least `most`.
__device__ __forceinline__ float e4m3_scale(float most) {
    const uint32_t bits = __float_as_uint(most);
    // 448 = 1.75 * 2^8
    const int exponent = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)max(exponent, 127 - 40) << 23);
}

// The reciprocal of a power of two from 2^-126 to 2^126.
__device__ __forceinline__ float inverse_of_power(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }

// Two f32 values of at most 448 to e4m3, ties to even, in the low two bytes.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
}

}  // namespace leafhip
