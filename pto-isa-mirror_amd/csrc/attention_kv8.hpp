// Attention over a cache held in 8 bits: what its kernels share.
#pragma once
#include <stddef.h>

#include "common_host.hpp"
#include "kv8.hpp"
#include "kv8_places.hpp"
#include "lds_dma.hpp"

namespace ptoamd {

struct AttentionArgs {
    Kv8 cache;
    const uint8_t* q;
    uint8_t* out;
    float* lse;
    int64_t q_token, q_head, out_token, out_head;  // bytes
    int heads, group;                              // query heads, and those that share a key head
    int causal, window;
    float scale;
    int wide;  // rows of q and out allow 16-byte accesses
    // The keys of a row in parts, where splits > 1 (at most so many): every part leaves its sums of a row (unscaled) and the row's reference and
    // sum, [split][token][head]; a second kernel joins them in the order of the parts.
    // Few rows, row_tiles of 16 a workgroup: parts of `chunk` tokens, each a workgroup's.  Many: `cuts`, of the rows in row_tiles tiles a sequence (Cuts).
    int splits, chunk, row_tiles, sequences;
    int* cuts;
    float* part_out;
    float2* part_sum;
};

// Many rows, keys in parts: all (key head, tile of rows, tile of keys) that there are, in this order, in equal stretches, one for a workgroup a CU.
// What the host does not know, how long the sequences are, is counted by each workgroup at its start.  A tile of rows counts for as many tiles
// of keys more, before its first, as its start and end cost: 448 keys' (12 to 14 us; 64 keys take 2).
struct Cuts {
    static constexpr int MOST = 256;                                       // tiles of rows of all sequences
    static constexpr int HEAD = 0, STRETCH = 1, FIRST = 2, SIZE = MOST + 3;  // tiles of keys: a key head's, a workgroup's, those before a tile of rows
    static constexpr size_t BYTES = 2048;
    static_assert(SIZE * sizeof(int) <= BYTES, "the join finds them at the workspace's start");
};
// The heads that the few and many kernels are built for; a smaller head takes the next of them: lanes beyond its elements read its first ones again,
// which the queries' zeros there take out of the scores, and whose results are not stored.  0: only the generic kernel.
constexpr int built_head(int head_dim) { return head_dim % 16 != 0 || head_dim > 256 ? 0 : head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
constexpr int many_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }  // a tile's
constexpr int MANY_KEYS = 64, MANY_START = 448 / MANY_KEYS;

// The waves of a few-rows workgroup of so many tiles of 16 rows: eight where two fit a SIMD's registers (heads up to 128 elements, one tile), else four.
constexpr int few_waves(int head_dim, int row_tiles) { return head_dim <= 128 && row_tiles == 1 ? 8 : 4; }
int launch_attention_few(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
int launch_attention_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
int launch_attention_join(const AttentionArgs& a, bool f16, int sequences, hipStream_t stream);
int prepare_attention_kernels();  // the launch attributes of all of them, for the current device

// Wave-uniform reads of what no kernel writes (tables, lengths, scales) through the scalar cache.
template <typename T>
__device__ __forceinline__ T load_uniform(const T* p)
{
    typedef const __attribute__((address_space(4))) T* constant_ptr;
    return *(constant_ptr)(uintptr_t)p;
}

// A field of the arguments (a kernel's only parameter), read from memory where it is asked for: what only the end of a kernel needs would else
// sit in scalar registers all through its loop.
struct ArgumentsAgain {
    uint64_t at;
    __device__ __forceinline__ ArgumentsAgain() : at((uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr()) { asm volatile("" : "+s"(at)); }
    template <typename T>
    __device__ __forceinline__ T field(size_t offset) const
    {
        return *(const __attribute__((address_space(4))) T*)(at + offset);
    }
    template <typename T>
    __device__ __forceinline__ T* global(size_t offset) const  // (through an integer the compiler no longer knows what memory)
    {
        return (T*)(__attribute__((address_space(1))) T*)(uintptr_t)field<uint64_t>(offset);
    }
    __device__ __forceinline__ const AttentionArgs* all() const
    {
        return (const AttentionArgs*)(const __attribute__((address_space(4))) AttentionArgs*)at;
    }
};
#define ARGUMENT(again, name) (again).template field<decltype(AttentionArgs::name)>(offsetof(AttentionArgs, name))

// A sequence's place in the call: its rows of q, its length, the keys that any of its queries sees (aligned down to 32 tokens at the start).
struct Span {
    int first, count, length, begin;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int seq)
{
    const Kv8& c = a.cache;
    Span s;
    s.first = seq * c.max_tokens;
    s.count = c.max_tokens;
    if (c.cu_tokens != nullptr) {
        s.first = min(max(load_uniform(c.cu_tokens + seq), 0), c.tokens);
        s.count = min(max(load_uniform(c.cu_tokens + seq + 1), s.first) - s.first, min(c.max_tokens, c.tokens - s.first));
    }
    s.length = min(max(load_uniform(c.lengths + seq), 0), c.max_pages << c.page_shift);
    s.begin = first_key(s.length - s.count, a.window) & ~31;
    return s;
}
// Whether a sequence's keys are in several parts, which are joined; else its workgroups write what the call returns.
__device__ __forceinline__ bool several_parts(const AttentionArgs& a, const Span& s) { return a.splits > 1 && s.length - s.begin > a.chunk; }
// The keys that a query at `place` of a sequence of `length` tokens sees: [x, y).
__device__ __forceinline__ int2 visible_keys(const AttentionArgs& a, int place, int length)
{
    return keys_of(place, length, a.causal, a.window);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two codes side by side in a dword's low (HIGH false) or high half -> two f16.  Every int8 and every E4M3 value is one.
// int8: with its sign bit turned a code is c + 128; under a high byte of 0x64 that is the f16 1024 + 128 + c, exactly.  (`w` then comes turned
// from kv8_turn.)
template <int CODE>
__device__ __forceinline__ uint32_t kv8_turn(uint32_t w) { return CODE == PTOAMD_I8 ? w ^ 0x80808080u : w; }
template <int CODE, bool HIGH>
__device__ __forceinline__ uint32_t kv8_pair_to_f16(uint32_t w)
{
    if (CODE == PTOAMD_I8) {
        const f16x2 biased = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(w, 0x64646464u, HIGH ? 0x00070006u : 0x00050004u));
        const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        return __builtin_bit_cast(uint32_t, biased - bias);
    }
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HIGH));
}
// Two dwords' bytes number B side by side, as f16: B of `even` low, B of `odd` high.
// int8: the turned code c + 128 alone is the f16 (c + 128) 2^-24, a subnormal one, exactly, and the matrix instructions take it as that: one
// permutation of bytes.  The 128 goes with products of a constant (UNBIAS), the 2^24 into what the sums are scaled with.  E4M3: two codes side by
// side are converted together.
constexpr uint32_t UNBIAS = 0x80808080u;  // two f16 of -128 2^-24
template <int CODE>
constexpr float KV8_UNIT = CODE == PTOAMD_I8 ? 16777216.0f : 1.0f;
// (dwords of int8 come turned)
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t even, uint32_t odd, int b)
{
    return __builtin_amdgcn_perm(odd, even, 0x0C000C00u | (uint32_t)b | (uint32_t)(4 + b) << 16);
}
// Two codes side by side, of keys whose products start at UNBIAS's: int8 comes turned and stays c + 128, as above.
template <int CODE, bool HIGH>
__device__ __forceinline__ uint32_t kv8_key_pair(uint32_t w)
{
    return CODE == PTOAMD_I8 ? __builtin_amdgcn_perm(w, w, HIGH ? 0x0C030C02u : 0x0C010C00u) : kv8_pair_to_f16<CODE, HIGH>(w);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Eight elements of a row of q, as they lie there.
__device__ __forceinline__ uint4 load_row8(const uint8_t* p, bool wide)
{
    if (wide)
        return *reinterpret_cast<const uint4*>(p);
    const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void widen_row8(uint4 raw, float* x)
{
    struct V { T e[8]; };
    const V v = __builtin_bit_cast(V, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = (float)v.e[i];
}
// Eight results.  (The packed dwords are what both ways store: given elements, the compiler makes one of the two, then of the narrow stores.)
template <typename T>
__device__ __forceinline__ void store_row8(uint8_t* p, bool wide, const float* x)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = sizeof(T) == 2 && __is_same(T, _Float16) ? pack_f16(x[2 * i], x[2 * i + 1]) : f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
    if (wide) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        uint16_t* e = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[2 * i] = (uint16_t)w[i];
            e[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
    }
}

// A row of queries is multiplied as f16, scaled by the power of two that brings its largest element into [1, 2): what that takes off an
// element of bf16 or f16 is below 2^-25 of the largest.  The factor that undoes it; NaN for a row that holds an infinity or a NaN.
struct RowScale {
    float down, up;
};
template <typename T>
__device__ __forceinline__ RowScale row_scale(uint32_t largest)
{
    const uint32_t bits = f2u((float)__builtin_bit_cast(T, (uint16_t)largest));
    if (bits >= 0x7F800000u)
        return RowScale{1.0f, NAN};
    const uint32_t e = min(max(bits >> 23, 1u), 253u);
    return RowScale{u2f((254u - e) << 23), u2f(e << 23)};
}

// The largest magnitude among a lane's elements of its row, as the bits of its 16-bit type without the sign (in order, an infinity above every
// number and a NaN above that).
template <int STEPS>
__device__ __forceinline__ uint32_t largest_of(const uint4* q)
{
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 largest = {0, 0};
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
        const uint32_t w[4] = {q[st].x, q[st].y, q[st].z, q[st].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    }
    return max((uint32_t)largest[0], (uint32_t)largest[1]);
}
template <typename T, int STEPS>
__device__ __forceinline__ void scale_to_f16(uint4* q, float by)
{
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
        float x[8];
        widen_row8<T>(q[st], x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] *= by;
        q[st] = make_uint4(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
    }
}

// A softmax reference starts here: finite, so that a row that has seen no key yet subtracts nothing undefined.
constexpr float NO_REFERENCE = -3.0e38f;
// Weights are 2^(score - reference), rounded to f16.  A reference is set so that the largest weight is 2^11, and follows only when one
// would pass 2^15: f16 keeps all its bits down to 2^-25 of the largest weight and loses what is below 2^-36 of it, and the sums are scaled
// again in few of the tiles.  (f16, as the products of both sides' types have one rate, and codes are f16 exactly.  Error of results against 64 bits, root
// mean square relative to theirs, beside f32 weights: of f16 results 2.4e-4 for 2.1e-4, 48 ragged sequences; of bf16 ones 1.7e-3 either way.)
constexpr float SET_TO = 11.0f, MOST = 15.0f;
// The scale of a page's values as a weight: its logarithm goes into the weight, its inverse back out of the sum.  A scale below 2^-64 counts
// as 0: the page's codes are then taken as 0, and 2^-64 stands for it here.
constexpr float LEAST_SCALE = 0x1p-64f;
struct ValueScale {
    float log2, inverse;
};
__device__ __forceinline__ ValueScale value_scale(float s)
{
    const float at_least = s < LEAST_SCALE ? LEAST_SCALE : s;  // (NaN stays)
    return ValueScale{__builtin_amdgcn_logf(at_least), __builtin_amdgcn_rcpf(at_least)};
}

}  // namespace ptoamd
