// Attention over a cache held in 8 bits: what its kernels share.
#pragma once
#include <stddef.h>

#include "common_host.hpp"
#include "drafted.hpp"
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
    // Few rows, row_tiles of 16 a workgroup: parts of `chunk` tokens, each a workgroup's.  Many: `cuts`, of the rows in row_tiles tiles of tile_rows a
    // sequence (Cuts).
    int splits, chunk, row_tiles, tile_rows, sequences;
    int* cuts;
    float* part_out;
    float2* part_sum;
    // of drafted tokens, in place of `causal`: rows of tree_words 32-bit words (seen_keys)
    const uint32_t* tree;
    int tree_words;
    int longest;  // few rows: 0, or sequences are taken in the order of span_in_turn
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
constexpr int MANY_KEYS = 64;
// What a tile of rows' start and end cost, in tiles of keys: those of half as many rows take half the time.
constexpr int many_start(int head_dim, int tile_rows) { return 448 / MANY_KEYS * (many_rows(head_dim) / tile_rows); }

// The waves of a few-rows workgroup of so many tiles of 16 rows: eight where two fit a SIMD's registers (heads up to 128 elements, one tile), else four.
// Of drafted tokens, four only of heads of 128 with three tiles or more and of 256 with two: what the others' registers lack they leave in LDS.  us, four waves
// / eight: 32 x 4 tokens over 8192 keys, 64 / 8 heads of 128, 134 / 119; of 64, 16 x 4 48 / 37, 16 x 6 59 / 45, 40 x 30 ragged up to 4001 35 / 24; 16 / 2 of
// 256, 48 x 2 over 4000 keys 41 / 41, over any number up to 4001 40 / 34.
constexpr int few_waves(int head_dim, int row_tiles, bool tree = false)
{
    return (head_dim <= 128 && row_tiles == 1) || (tree && (head_dim == 256 ? row_tiles == 1 : row_tiles == 2 || head_dim == 64)) ? 8 : 4;
}
constexpr bool few_queries_in_lds(int head_dim, int row_tiles, bool tree) { return tree && ((head_dim == 64 && row_tiles == 2) || head_dim == 256); }
int launch_attention_few(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
int launch_attention_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
// (of drafted tokens)
int launch_attention_tree_few(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
int launch_attention_tree_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream);
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
// That of the nth sequence in the order of their lengths, the longer first: by steps of half an octave below `longest`, those of a step in their order, the
// shortest last.  A wave looks at up to 64 sequences, a lane at one; of more every second, third, ... is in one order, and the orders take turns.
__device__ __forceinline__ Span span_in_turn(const AttentionArgs& a, int nth, int* nth_seq)
{
    const Kv8& c = a.cache;
    const int orders = (a.sequences + 63) / 64, order = nth % orders, lane = threadIdx.x % 64, seq = order + lane * orders;
    const bool there = seq < a.sequences;
    const int at = there ? seq : 0, length = min(max(c.lengths[at], 0), c.max_pages << c.page_shift);
    int first = at * c.max_tokens, count = c.max_tokens;
    if (c.cu_tokens != nullptr) {
        const int from = c.cu_tokens[at], to = c.cu_tokens[at + 1];
        first = min(max(from, 0), c.tokens);
        count = min(max(to, first) - first, min(c.max_tokens, c.tokens - first));
    }
    const int step = max((int)(f2u((float)a.longest) - f2u((float)max(length, 1))) >> 22, 0);
    constexpr int STEPS = 8;  // (the last has all that are shorter)
    nth /= orders;
    uint64_t its = 0;
    for (int i = 0; i <= STEPS; ++i) {
        its = __ballot(there && (i < STEPS ? step == i : step >= STEPS));
        const int n = __popcll(its);
        if (nth < n)
            break;
        nth -= n;
    }
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(its >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)its, 0));
    const int found = __builtin_ctzll(__ballot((its >> lane & 1) != 0 && before == nth));
    Span s;
    s.first = __builtin_amdgcn_readlane(first, found);
    s.count = __builtin_amdgcn_readlane(count, found);
    s.length = __builtin_amdgcn_readlane(length, found);
    s.begin = first_key(s.length - s.count, a.window) & ~31;
    *nth_seq = order + found * orders;
    return s;
}
// Whether a sequence's keys are in several parts, which are joined; else its workgroups write what the call returns.
__device__ __forceinline__ bool several_parts(const AttentionArgs& a, const Span& s) { return a.splits > 1 && s.length - s.begin > a.chunk; }
// The keys that a query at `place` of a sequence of `length` tokens sees: [x, y).
__device__ __forceinline__ int2 visible_keys(const AttentionArgs& a, int place, int length)
{
    return keys_of(place, length, a.causal, a.window);
}

// The keys that any of a sequence's new tokens first .. last sees: [x, y).  TREE: a token stands behind those that it sees, none to all that are drafted.
template <bool TREE>
__device__ __forceinline__ int2 keys_of_any(const AttentionArgs& a, const Span& s, int first, int last)
{
    const int place0 = s.length - s.count;
    if (TREE)
        return make_int2(first_key(place0, a.window), s.length);
    return make_int2(visible_keys(a, place0 + first, s.length).x, visible_keys(a, place0 + last, s.length).y);
}
// Those that every one of them sees.
template <bool TREE>
__device__ __forceinline__ int2 keys_of_every(const AttentionArgs& a, const Span& s, int first, int last)
{
    const int place0 = s.length - s.count;
    if (TREE)
        return make_int2(first_key(s.length - 1, a.window), place0);
    return make_int2(visible_keys(a, place0 + last, s.length).x, visible_keys(a, place0 + first, s.length).y);
}
// Words of a drafted token's row, its bits behind the sequence's last token cleared.
__device__ __forceinline__ uint32_t drafted_word(const AttentionArgs& a, const Span& s, int token, int word)
{
    return own_word(a.tree + (int64_t)(s.first + token) * a.tree_words, a.tree_words, word, s.count);
}
// The first of the older keys that a token sees, whose `words` words lie in LDS.  (No row: none of them.)
__device__ __forceinline__ int first_of_drafted(const AttentionArgs& a, const Span& s, const uint32_t* row, int words, bool valid, int token)
{
    if (!valid)
        return 0x7FFFFFFF;
    return first_of_older(row, words, s.count, token, s.length - s.count, a.window);
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
