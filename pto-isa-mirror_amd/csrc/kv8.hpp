// A cache of keys and values held in 8 bits, as the kernels see it: pages, the spans of sequences, codes.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ptoamd.h"
#include "device_types.hpp"

namespace ptoamd {

struct Kv8Side {
    uint8_t* codes;
    float* scales;
    int64_t page, head, token;  // strides in bytes
};
struct Kv8 {
    Kv8Side k, v;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* cu_tokens;  // null: max_tokens for every sequence
    int pages, kv_heads, page_shift, head_dim, max_pages, tokens, max_tokens;

    // the new tokens of a sequence, whatever cu_tokens holds: rows first .. first + count - 1, inside the operands
    __device__ __forceinline__ int first_token(int seq) const { return cu_tokens ? min(max(cu_tokens[seq], 0), tokens) : seq * max_tokens; }
    __device__ __forceinline__ int token_count(int seq, int first) const
    {
        return cu_tokens ? min(max(cu_tokens[seq + 1], first) - first, min(max_tokens, tokens - first)) : max_tokens;
    }
    __device__ __forceinline__ int length(int seq) const { return min(max(lengths[seq], 0), max_pages << page_shift); }
    // a page of a sequence, or -1 where the table names none
    __device__ __forceinline__ int page_of(int seq, int block) const
    {
        const int p = table[(int64_t)seq * max_pages + block];
        return (unsigned)p < (unsigned)pages ? p : -1;
    }
};

// The value a code stands for, in units of its scale.
template <int CODE>
__device__ __forceinline__ float kv8_value(uint32_t code)
{
    return CODE == PTOAMD_I8 ? (float)(int8_t)code : e4m3_to_f32(code);
}

int kv8_from(const char* what, const ptoamd_kv8_cache* c, int tokens, const int32_t* cu_tokens, int max_tokens, Kv8* out);

}  // namespace ptoamd
