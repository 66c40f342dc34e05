// The append to an 8-bit cache with the rotation of positions on the way, and the rotation of the queries beside it.
#include "common_host.hpp"
#include "drafted.hpp"
#include "kv8.hpp"
#include "kv8_codes.hpp"
#include "kv8_places.hpp"

namespace ptoamd {

struct AppendRopeArgs {
    Kv8 cache;
    const uint8_t* src[2];                         // k, v
    int64_t token[2], head[2];                     // strides in bytes
    const uint8_t* q;
    uint8_t* q_out;
    int64_t q_token, q_head, out_token, out_head;  // bytes
    const float* table;
    const int32_t* positions;
    const uint32_t* tree;
    int tree_words;                                // of 32 bits
    int table_rows, half, heads, interleaved;
    int blocks;                                    // most pages that a sequence's new tokens touch
    unsigned append_groups, wide;                  // workgroups of the append; those that a token's queries take

    // the position that the nth new token of a sequence, row `row` of the operands, is turned by; `start` is its first new token's place
    __device__ __forceinline__ int position(int row, int nth, int count, int start) const
    {
        if (positions != nullptr)
            return positions[row];
        return start + (tree != nullptr ? others_seen(tree + (int64_t)row * tree_words, tree_words, count, nth) : nth);
    }
};

// The order of a head's elements in 16s, a thread's unit: 8 elements and the 8 that they are paired with, so that a pair is one thread's.  HALVES: i and
// i + half; NEIGHBOURS: 2 i and 2 i + 1.  ANY is for rotations that are not made of 16s, and for operands off 16 bytes: elements one by one.
enum RopeOrder { HALVES, NEIGHBOURS, ANY };
struct Chunks {
    int lo, hi;  // the unit's two runs of 8 elements; the same one twice where only 8 are left
};
template <RopeOrder ORDER>
__device__ __forceinline__ Chunks chunks_of(int u, int half, int dim)
{
    const int lo = ORDER == HALVES && 8 * u < half ? 8 * u : 16 * u, hi = ORDER == HALVES && 8 * u < half ? 8 * u + half : 16 * u + 8;
    return Chunks{lo, hi < dim ? hi : lo};
}

// A unit of a row, turned.  (A position that the table does not have: NaN.)
template <typename T, RopeOrder ORDER>
__device__ __forceinline__ void load_turned(const AppendRopeArgs& a, const T* row, int position, int u, int dim, float* x)
{
    const bool known = (unsigned)position < (unsigned)a.table_rows;
    const float* turn = a.table + (int64_t)(known ? position : 0) * 2 * a.half;
    const float unknown = known ? 0.0f : NAN;
    if constexpr (ORDER == ANY) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int e = min(16 * u + j, dim - 1);
            x[j] = (float)row[e];
            if (e < 2 * a.half) {
                const int pair = a.interleaved ? e / 2 : e < a.half ? e : e - a.half;
                const bool second = a.interleaved ? e % 2 != 0 : e >= a.half;
                const int other = a.interleaved ? e ^ 1 : second ? e - a.half : e + a.half;
                const float c = turn[pair] + unknown, s = turn[a.half + pair] + unknown, y = (float)row[other];
                x[j] = second ? y * s + x[j] * c : x[j] * c - y * s;
            }
        }
    } else {
        const Chunks at = chunks_of<ORDER>(u, a.half, dim);
        load8<T, true>(row + at.lo, x);
        load8<T, true>(row + at.hi, x + 8);
        if (8 * u < a.half) {
            float c[8], s[8];
            load8<float, true>(turn + 8 * u, c);
            load8<float, true>(turn + a.half + 8 * u, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = ORDER == HALVES ? j : 2 * j, q = ORDER == HALVES ? j + 8 : 2 * j + 1;
                const float first = x[p], second = x[q], cosine = c[j] + unknown, sine = s[j] + unknown;
                x[p] = first * cosine - second * sine;
                x[q] = first * sine + second * cosine;
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x)
{
    struct alignas(16) V { T e[16 / sizeof(T)]; };
    V v[8 * sizeof(T) / 16];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i * sizeof(T) / 16].e[i % (16 / sizeof(T))] = (T)x[i];
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
        reinterpret_cast<V*>(p)[i] = v[i];
}

// Queries: a thread has a unit of one token's head.  (ANY: a pair, or one element behind the pairs, so that the result may lie where the operand does.)
template <typename T, RopeOrder ORDER, int THREADS>
__device__ __forceinline__ void turn_queries(const AppendRopeArgs& a, unsigned group)
{
    const Kv8& c = a.cache;
    const unsigned row_group = group / a.wide;
    const int seq = row_group / (unsigned)c.max_tokens, nth = row_group - (unsigned)seq * c.max_tokens;
    const int first = c.first_token(seq), count = c.token_count(seq, first);
    const int units = ORDER == ANY ? c.head_dim - a.half : (c.head_dim + 15) / 16;
    const int unit = (group - row_group * a.wide) * THREADS + threadIdx.x, head = unit / units, u = unit - head * units;
    if (nth >= count || head >= a.heads)
        return;
    const int position = a.position(first + nth, nth, count, max(c.lengths[seq], 0) - count);
    const T* x = reinterpret_cast<const T*>(a.q + (int64_t)(first + nth) * a.q_token + (int64_t)head * a.q_head);
    T* out = reinterpret_cast<T*>(a.q_out + (int64_t)(first + nth) * a.out_token + (int64_t)head * a.out_head);
    if constexpr (ORDER == ANY) {
        if (u >= a.half) {
            out[u + a.half] = x[u + a.half];
            return;
        }
        const bool known = (unsigned)position < (unsigned)a.table_rows;
        const float* turn = a.table + (int64_t)(known ? position : 0) * 2 * a.half;
        const float cosine = known ? turn[u] : NAN, sine = known ? turn[a.half + u] : NAN;
        const int i = a.interleaved ? 2 * u : u, j = a.interleaved ? 2 * u + 1 : u + a.half;
        const float p = (float)x[i], q = (float)x[j];
        out[i] = (T)(p * cosine - q * sine);
        out[j] = (T)(p * sine + q * cosine);
    } else {
        float y[16];
        load_turned<T, ORDER>(a, x, position, u, c.head_dim, y);
        const Chunks at = chunks_of<ORDER>(u, a.half, c.head_dim);
        store8(out + at.lo, y);
        store8(out + at.hi, y + 8);
    }
}

// The first workgroups append, one a page of a sequence, head and side (keys or values): the append of kvcache.hip, with keys turned as they are read.  The
// others turn queries.  Products and sums in f32; a key is rounded once, to its code.
template <typename T, int CODE, RopeOrder ORDER, int THREADS>
__global__ void __launch_bounds__(THREADS) kvcache_append_rope_kernel(AppendRopeArgs a)
{
    const Kv8& c = a.cache;
    if (blockIdx.x >= a.append_groups) {
        turn_queries<T, ORDER, THREADS>(a, blockIdx.x - a.append_groups);
        return;
    }
    const bool values = blockIdx.x % 2 != 0;
    const unsigned page_head = blockIdx.x / 2, nth_page = page_head / (unsigned)c.kv_heads;
    const int head = page_head - nth_page * c.kv_heads, seq = nth_page / (unsigned)a.blocks, nth = nth_page - seq * (unsigned)a.blocks;
    const Kv8Side side = values ? c.v : c.k;
    const int first = c.first_token(seq), count = c.token_count(seq, first), length = c.length(seq);
    const int start = max(c.lengths[seq], 0) - count;  // place of the first new token; those before 0 or behind the table have none
    if (start >= length)
        return;
    const int block = (max(start, 0) >> c.page_shift) + nth;
    const int lo = max(max(start, 0), block << c.page_shift), hi = min(length, (block + 1) << c.page_shift);
    if (lo >= hi)
        return;
    const int page = c.page_of(seq, block);
    if (page < 0)
        return;
    const int older = lo - (block << c.page_shift), fresh = hi - lo;
    const int per_token = (c.head_dim + 15) / 16, units = fresh * per_token;
    const uint8_t* src = a.src[values] + (int64_t)head * a.head[values];
    auto load = [&](int token, int u, float* x) __attribute__((always_inline)) {  // of the page's new tokens
        const int row_at = first + lo - start + token;
        const T* row = reinterpret_cast<const T*>(src + (int64_t)row_at * a.token[values]);
        if (values) {
            const Chunks at = chunks_of<ANY>(u, 0, c.head_dim);
            load8<T, ORDER != ANY>(row + at.lo, x);
            load8<T, ORDER != ANY>(row + at.hi, x + 8);
        } else {
            load_turned<T, ORDER>(a, row, a.position(row_at, lo - start + token, count, start), u, c.head_dim, x);
        }
    };
    uint32_t largest = 0;
    for (int u = threadIdx.x; u < units; u += THREADS) {
        float x[16];
        load(u / per_token, u % per_token, x);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            largest = max(largest, f2u(x[i]) & 0x7FFFFFFFu);
    }
    __shared__ uint32_t wave_largest[THREADS / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        largest = max(largest, (uint32_t)__shfl_xor((int)largest, d));
    if (threadIdx.x % 64 == 0)
        wave_largest[threadIdx.x / 64] = largest;
    float* scale = side.scales + (int64_t)page * c.kv_heads + head;
    const float before = older > 0 ? *scale : 0.0f;
    __syncthreads();  // (the scale has been read by all before one writes it)
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w)
        largest = max(largest, wave_largest[w]);
    float after = u2f(largest) * KV8_PER_LARGEST<CODE>;
    after = before > after ? before : after;
    after = after < 0x1p-126f ? 0.0f : after;
    if (largest >= 0x7F800000u || before != before)
        after = NAN;
    if (threadIdx.x == 0)
        *scale = after;
    uint8_t* dst = side.codes + (int64_t)page * side.page + (int64_t)head * side.head;
    if (before < after) {  // the older tokens' codes in the new unit
        const float ratio = before / after;
        const int chunks = c.head_dim / 8;
        for (int u = threadIdx.x; u < older * chunks; u += THREADS) {
            uint2* p = reinterpret_cast<uint2*>(dst + (int64_t)(u / chunks) * side.token + (u % chunks) * 8);
            const uint2 w = *p;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = kv8_value<CODE>(((i < 4 ? w.x : w.y) >> (8 * (i % 4))) & 0xFFu) * ratio;
            *p = kv8_codes<CODE>(x);
        }
    }
    const float inverse = after > 0.0f ? 1.0f / after : 0.0f;
    for (int u = threadIdx.x; u < units; u += THREADS) {
        const int token = u / per_token;
        float x[16];
        load(token, u % per_token, x);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = inverse > 0.0f ? x[i] * inverse : 0.0f;  // (a NaN scale: codes of zero)
        const Chunks at = values ? chunks_of<ANY>(u % per_token, 0, c.head_dim) : chunks_of<ORDER>(u % per_token, a.half, c.head_dim);
        uint8_t* to = dst + (int64_t)(older + token) * side.token;
        *reinterpret_cast<uint2*>(to + at.lo) = kv8_codes<CODE>(x);
        if (at.hi != at.lo)
            *reinterpret_cast<uint2*>(to + at.hi) = kv8_codes<CODE>(x + 8);
    }
}

template <typename T, int CODE, RopeOrder ORDER, int THREADS>
static int launch_append_rope(AppendRopeArgs a, int sequences, hipStream_t stream)
{
    const long units = (long)a.heads * (ORDER == ANY ? a.cache.head_dim - a.half : (a.cache.head_dim + 15) / 16);
    const long wide = (units + THREADS - 1) / THREADS, append = 2L * sequences * a.blocks * a.cache.kv_heads;
    const long groups = append + (long)sequences * a.cache.max_tokens * wide;
    PTOAMD_REQUIRE(groups <= 0x7FFFFFFF, PTOAMD_E_UNSUPPORTED, "ptoamd_kvcache_append_rope: %d sequences of %d tokens are too many for one launch", sequences,
                   a.cache.max_tokens);
    a.append_groups = (unsigned)append;
    a.wide = (unsigned)(wide > 0 ? wide : 1);
    hipLaunchKernelGGL((kvcache_append_rope_kernel<T, CODE, ORDER, THREADS>), dim3((unsigned)groups), dim3(THREADS), 0, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("kvcache_append_rope");
    return PTOAMD_OK;
}
// Threads by the bytes that a page's new tokens have of a head, as in kvcache.hip.
template <typename T, int CODE, RopeOrder ORDER>
static int choose_threads(const AppendRopeArgs& a, int sequences, hipStream_t stream)
{
    const int page = 1 << a.cache.page_shift;
    const long bytes = (long)(a.cache.max_tokens < page ? a.cache.max_tokens : page) * a.cache.head_dim * sizeof(T);
    if (bytes <= 8192)
        return launch_append_rope<T, CODE, ORDER, 128>(a, sequences, stream);
    return bytes <= 16384 ? launch_append_rope<T, CODE, ORDER, 256>(a, sequences, stream) : launch_append_rope<T, CODE, ORDER, 512>(a, sequences, stream);
}
template <typename T, int CODE>
static int choose_order(const AppendRopeArgs& a, int sequences, hipStream_t stream)
{
    uint64_t bits = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.q_out | (uint64_t)(uintptr_t)a.table | (uint64_t)a.q_token | (uint64_t)a.q_head |
                    (uint64_t)a.out_token | (uint64_t)a.out_head;
    for (int i = 0; i < 2; ++i)
        bits |= (uint64_t)(uintptr_t)a.src[i] | (uint64_t)a.token[i] | (uint64_t)a.head[i];
    if (a.half % 8 != 0 || bits % 16 != 0)
        return choose_threads<T, CODE, ANY>(a, sequences, stream);
    return a.interleaved ? choose_threads<T, CODE, NEIGHBOURS>(a, sequences, stream) : choose_threads<T, CODE, HALVES>(a, sequences, stream);
}
template <typename T>
static int choose_code(const AppendRopeArgs& a, int code, int sequences, hipStream_t stream)
{
    return code == PTOAMD_I8 ? choose_order<T, PTOAMD_I8>(a, sequences, stream) : choose_order<T, PTOAMD_E4M3>(a, sequences, stream);
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

int ptoamd_kvcache_append_rope(const ptoamd_kv8_cache* cache, void* q_out, const void* q, int heads, const void* k, const void* v, int type, int tokens,
                               const int32_t* cu_tokens, int max_tokens, const float* table, int table_rows, int rot_dim, int interleaved,
                               const int32_t* positions, const uint64_t* tree, int tree_words, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t q_out_token_stride, int64_t q_out_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                               int64_t v_token_stride, int64_t v_head_stride, void* stream)
{
    const char* what = "ptoamd_kvcache_append_rope";
    AppendRopeArgs a{};
    const int rc = kv8_from(what, cache, tokens, cu_tokens, max_tokens, &a.cache);
    if (rc != PTOAMD_OK)
        return rc;
    TraceScope trace("KVCACHE_APPEND_ROPE", "vector", tokens, heads + cache->kv_heads, cache->head_dim);
    trace.in(q, tokens, (long)heads * cache->head_dim, "ND", type).in(k, tokens, (long)cache->kv_heads * cache->head_dim, "ND", type)
        .in(v, tokens, (long)cache->kv_heads * cache->head_dim, "ND", type).in(table, table_rows, rot_dim, "ND", PTOAMD_F32)
        .out(q_out, tokens, (long)heads * cache->head_dim, "ND", type)
        .out(cache->k, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type)
        .out(cache->v, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type);
    PTOAMD_REQUIRE(type == PTOAMD_F32 || type == PTOAMD_F16 || type == PTOAMD_BF16, PTOAMD_E_UNSUPPORTED, "%s: queries, keys and values must be f32, f16 or bf16",
                   what);
    PTOAMD_REQUIRE(cache->head_dim % 8 == 0 && cache->head_dim <= 512, PTOAMD_E_UNSUPPORTED, "%s: head_dim must be a multiple of 8 and at most 512 (%d)", what,
                   cache->head_dim);
    PTOAMD_REQUIRE(heads >= 0 && table_rows > 0, PTOAMD_E_INVALID, "%s: table_rows must be positive, heads not negative (%d, %d)", what, table_rows, heads);
    PTOAMD_REQUIRE((long)heads * cache->head_dim <= 1 << 24, PTOAMD_E_UNSUPPORTED, "%s: %d heads of %d elements are too many", what, heads, cache->head_dim);
    PTOAMD_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= cache->head_dim, PTOAMD_E_INVALID, "%s: rot_dim must be even and at most head_dim (%d of %d)",
                   what, rot_dim, cache->head_dim);
    PTOAMD_REQUIRE(positions == nullptr || tree == nullptr, PTOAMD_E_INVALID, "%s: a token's position is given or follows from the tree, not both", what);
    if (tokens == 0 || max_tokens == 0)
        return PTOAMD_OK;
    PTOAMD_REQUIRE(k && v && table && (heads == 0 || (q && q_out)), PTOAMD_E_INVALID, "%s: null operand", what);
    PTOAMD_REQUIRE(tree == nullptr || a.cache.max_tokens <= PTOAMD_MOST_DRAFTED, PTOAMD_E_UNSUPPORTED, "%s: at most %d tokens of a sequence are drafted (%d)",
                   what, PTOAMD_MOST_DRAFTED, a.cache.max_tokens);
    PTOAMD_REQUIRE(tree == nullptr || (tree_words > 0 && tree_words <= PTOAMD_MOST_DRAFTED / 64 && 64 * tree_words >= a.cache.max_tokens), PTOAMD_E_INVALID,
                   "%s: rows of %d words for %d tokens: one for every 64 is needed, at most %d", what, tree_words, a.cache.max_tokens, PTOAMD_MOST_DRAFTED / 64);
    const int size = type == PTOAMD_F32 ? 4 : 2;
    PTOAMD_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (heads > 0 ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0)) % size == 0 &&
                       (reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(positions)) % 4 == 0 && reinterpret_cast<uintptr_t>(tree) % 8 == 0,
                   PTOAMD_E_ALIGNMENT, "%s: operands must be aligned to their elements", what);
    PTOAMD_REQUIRE(heads == 0 || q_out != q || (q_token_stride == q_out_token_stride && q_head_stride == q_out_head_stride), PTOAMD_E_INVALID,
                   "%s: in place, q_out must have the strides of q", what);
    a.src[0] = static_cast<const uint8_t*>(k);
    a.src[1] = static_cast<const uint8_t*>(v);
    a.token[0] = k_token_stride * size;
    a.token[1] = v_token_stride * size;
    a.head[0] = k_head_stride * size;
    a.head[1] = v_head_stride * size;
    if (heads > 0) {
        a.q = static_cast<const uint8_t*>(q);
        a.q_out = static_cast<uint8_t*>(q_out);
        a.q_token = q_token_stride * size;
        a.q_head = q_head_stride * size;
        a.out_token = q_out_token_stride * size;
        a.out_head = q_out_head_stride * size;
    }
    a.table = table;
    a.positions = positions;
    a.tree = reinterpret_cast<const uint32_t*>(tree);
    a.tree_words = 2 * tree_words;
    a.table_rows = table_rows;
    a.half = rot_dim / 2;
    a.heads = heads;
    a.interleaved = interleaved != 0;
    a.blocks = pages_of(a.cache.max_tokens, a.cache.page_shift);
    hipStream_t s = as_stream(stream);
    switch (type) {
        case PTOAMD_F32: return choose_code<float>(a, cache->code_type, cache->sequences, s);
        case PTOAMD_F16: return choose_code<_Float16>(a, cache->code_type, cache->sequences, s);
        default: return choose_code<__bf16>(a, cache->code_type, cache->sequences, s);
    }
}

}  // extern "C"
