// Values to the codes of an 8-bit cache: what the kernels that write one share.
#pragma once
#include "kv8.hpp"

namespace ptoamd {

// Eight values in units of their scale -> eight codes.  int8: nearest, ties to even, clamped.  E4M3: the hardware's conversion, which
// rounds every value inside +-448 to the nearest code, ties to even; values are clamped to that first.
template <int CODE>
__device__ __forceinline__ uint2 kv8_codes(const float* x)
{
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (CODE == PTOAMD_I8) {
            w[h] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[h] |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(rintf(x[4 * h + i]), -127.0f, 127.0f) & 0xFFu) << (8 * i);
        } else {
            float c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                c[i] = __builtin_amdgcn_fmed3f(x[4 * h + i], -448.0f, 448.0f);
            int pk = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
            w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], pk, true);
        }
    }
    return make_uint2(w[0], w[1]);
}

template <int CODE>
constexpr float KV8_PER_LARGEST = CODE == PTOAMD_I8 ? 1.0f / 127.0f : 1.0f / 448.0f;  // a page's scale over its largest magnitude

// A page's scale once values have come into it whose largest magnitude has these bits.  (Bits, so that an infinity or a NaN among them is the largest.)
template <int CODE>
__device__ __forceinline__ float kv8_grown_scale(float old, uint32_t largest)
{
    float now = u2f(largest) * KV8_PER_LARGEST<CODE>;
    now = old > now ? old : now;
    now = now < 0x1p-126f ? 0.0f : now;
    return largest >= 0x7F800000u || old != old ? NAN : now;
}
// Eight codes in a unit that is 1 / `by` of theirs.
template <int CODE>
__device__ __forceinline__ uint2 kv8_scaled_codes(uint2 w, float by)
{
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = kv8_value<CODE>(((i < 4 ? w.x : w.y) >> (8 * (i % 4))) & 0xFFu) * by;
    return kv8_codes<CODE>(x);
}

}  // namespace ptoamd
