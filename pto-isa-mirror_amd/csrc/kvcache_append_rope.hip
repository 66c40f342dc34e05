// The append to an 8-bit cache with the rotation of positions on the way, and the rotation of the queries beside it.
#include "common_host.hpp"
#include "drafted.hpp"
#include "kv8.hpp"
#include "kv8_codes.hpp"
#include "kv8_places.hpp"
#include "overlap.hpp"

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
    unsigned wide, pairs;                          // workgroups that the queries of two tokens take; such pairs of a sequence, or 0: pairs of the batch's rows
    int sequences;
    uint64_t share;                                // of the workgroups that append, in 2^-32

    // the position that the nth new token of a sequence, row `row` of the operands, is turned by; `start` is its first new token's place
    __device__ __forceinline__ int position(int row, int nth, int count, int start) const
    {
        if (positions != nullptr)
            return positions[row];
        return start + (tree != nullptr ? others_seen(tree + (int64_t)row * tree_words, tree_words, count, nth) : nth);
    }
};

// A thread's unit of a head: VEC pairs, so that a pair is one thread's, as two runs of VEC elements: half a rotation apart or, INTERLEAVED, next to each other;
// of the elements behind the rotation two runs next to each other.  (Where VEC elements are left there, the same run twice.)
struct Runs {
    int lo, hi;
};
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ Runs runs_of(int u, int half, int dim)
{
    const bool apart = !INTERLEAVED && VEC * u < half;
    const int lo = apart ? VEC * u : 2 * VEC * u, hi = apart ? lo + half : lo + VEC;
    return Runs{lo, hi < dim ? hi : lo};
}
template <typename T, int VEC>
__device__ __forceinline__ void load_run(const T* p, float* x)
{
    constexpr int EACH = VEC * sizeof(T) > 16 ? 16 / sizeof(T) : VEC;
    struct alignas(EACH * sizeof(T)) V { T e[EACH]; };
    V v[VEC / EACH];
#pragma unroll
    for (int i = 0; i < VEC / EACH; ++i)
        v[i] = reinterpret_cast<const V*>(p)[i];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        x[i] = (float)v[i / EACH].e[i % EACH];
}
template <typename T, int VEC>
__device__ __forceinline__ void store_run(T* p, const float* x)
{
    constexpr int EACH = VEC * sizeof(T) > 16 ? 16 / sizeof(T) : VEC;
    struct alignas(EACH * sizeof(T)) V { T e[EACH]; };
    V v[VEC / EACH];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        v[i / EACH].e[i % EACH] = (T)x[i];
#pragma unroll
    for (int i = 0; i < VEC / EACH; ++i)
        reinterpret_cast<V*>(p)[i] = v[i];
}
template <int CODE, int VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* x)
{
    float eight[8] = {};
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        eight[i] = x[i];
    const uint2 w = kv8_codes<CODE>(eight);
    if constexpr (VEC == 8)
        *reinterpret_cast<uint2*>(p) = w;
    else if constexpr (VEC == 4)
        *reinterpret_cast<uint32_t*>(p) = w.x;
    else
        *p = (uint8_t)w.x;
}

// A unit of a row, turned.  (A position that the table does not have: NaN.)
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void load_turned(const AppendRopeArgs& a, const T* row, int position, int u, int dim, float* x)
{
    const Runs at = runs_of<VEC, INTERLEAVED>(u, a.half, dim);
    load_run<T, VEC>(row + at.lo, x);
    load_run<T, VEC>(row + at.hi, x + VEC);
    if (VEC * u < a.half) {
        const bool known = (unsigned)position < (unsigned)a.table_rows;
        const float* turn = a.table + (int64_t)(known ? position : 0) * 2 * a.half + VEC * u;
        const float unknown = known ? 0.0f : NAN;
        float c[VEC], s[VEC];
        load_run<float, VEC>(turn, c);
        load_run<float, VEC>(turn + a.half, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int p = INTERLEAVED ? 2 * j : j, q = INTERLEAVED ? 2 * j + 1 : j + VEC;
            const float first = x[p], second = x[q], cosine = c[j] + unknown, sine = s[j] + unknown;
            x[p] = first * cosine - second * sine;
            x[q] = first * sine + second * cosine;
        }
    }
}

constexpr int ROPE_TOKENS = 2;

// The last sequence that starts at a row or before it, or -1: 64 starts at a time.  (Whatever cu_tokens holds, a sequence that there is.)
__device__ __forceinline__ int sequence_of(const AppendRopeArgs& a, int row)
{
    const int lane = threadIdx.x % 64;
    int seq = 0;
    for (int step = a.sequences > 4096 ? 4096 : a.sequences > 64 ? 64 : 1; step > 0; step /= 64) {
        const int at = seq + lane * step, before = __popcll(__ballot(at < a.sequences && a.cache.cu_tokens[min(at, a.sequences)] <= row));
        if (before == 0)
            return -1;
        seq += (before - 1) * step;
    }
    return seq;
}

// Queries: a thread has a unit of a head of two consecutive tokens, all loads of both in flight before the first is used, as in rope.hip.  The two are a sequence's
// (pairs), or, with cu_tokens, two rows of the batch, whose sequences are looked for: max_tokens may be far above the tokens that there are.  us, pairs of max_tokens of every
// sequence / of rows, 32 / 8 heads of 128: 64 sequences of 128 tokens, max_tokens 128 35.0 / 34.2, 512 38.9 / 34.5, 2048 79 / 47; 256 of 4, 4 13.1 / 13.2, 64 33 / 21; 64 of
// 1, 1 5.6 / 5.5, 8 6.3 / 6.7, 64 11.6 / 8.3.
template <typename T, int VEC, bool INTERLEAVED, int THREADS>
__device__ __forceinline__ void turn_queries(const AppendRopeArgs& a, unsigned group)
{
    const Kv8& c = a.cache;
    const unsigned row_group = group / a.wide;
    int seq = -1, first = 0, count = 0, start = 0;
    auto enter = [&](int its) {
        seq = its;
        first = c.first_token(seq), count = c.token_count(seq, first);
        start = max(c.lengths[seq], 0) - count;
    };
    int row[ROPE_TOKENS], position[ROPE_TOKENS];  // (row -1: not a sequence's)
    if (a.pairs > 0) {
        enter(row_group / a.pairs);
        const int nth = (row_group - (unsigned)seq * a.pairs) * ROPE_TOKENS;
        if (nth >= count)
            return;
#pragma unroll
        for (int k = 0; k < ROPE_TOKENS; ++k) {
            const int token = min(nth + k, count - 1);
            row[k] = nth + k < count ? first + token : -1;
            position[k] = a.position(first + token, token, count, start);
        }
    } else {
#pragma unroll
        for (int k = 0; k < ROPE_TOKENS; ++k) {
            const int at = row_group * ROPE_TOKENS + k;
            if (at < c.tokens && (seq < 0 || at >= first + count)) {
                const int its = sequence_of(a, at);
                if (its >= 0)
                    enter(__builtin_amdgcn_readfirstlane(its));
            }
            const bool there = at < c.tokens && seq >= 0 && at >= first && at < first + count;
            row[k] = there ? at : -1;
            position[k] = there ? a.position(at, at - first, count, start) : 0;
        }
    }
    const int units = (c.head_dim + 2 * VEC - 1) / (2 * VEC);
    const int unit = (group - row_group * a.wide) * THREADS + threadIdx.x, head = unit / units, u = unit - head * units;
    static_assert(ROPE_TOKENS == 2, "one of two rows stands in for the other");
    const int some = max(row[0], row[1]);
    if (some < 0 || head >= a.heads)
        return;
    const uint8_t* x = a.q + (int64_t)head * a.q_head;
    uint8_t* out = a.q_out + (int64_t)head * a.out_head;
    const Runs at = runs_of<VEC, INTERLEAVED>(u, a.half, c.head_dim);
    float y[ROPE_TOKENS][2 * VEC];
#pragma unroll
    for (int k = 0; k < ROPE_TOKENS; ++k)
        load_turned<T, VEC, INTERLEAVED>(a, reinterpret_cast<const T*>(x + (int64_t)(row[k] < 0 ? some : row[k]) * a.q_token), position[k], u, c.head_dim, y[k]);
#pragma unroll
    for (int k = 0; k < ROPE_TOKENS; ++k) {
        if (row[k] < 0)
            continue;
        T* to = reinterpret_cast<T*>(out + (int64_t)row[k] * a.out_token);
        store_run<T, VEC>(to + at.lo, y[k]);
        store_run<T, VEC>(to + at.hi, y[k] + VEC);
    }
}

// Some workgroups append, one a page of a sequence, head and side (keys or values): the append of kvcache.hip, with keys turned as they are read.  The
// others turn queries; the two kinds stand among each other in the grid, since a page's chain of loads leaves the memory to the queries.
// Products and sums in f32; a key is rounded once, to its code.
// Bound: HBM where there are many tokens (6 ragged prompts of up to 2048, 32 / 8 heads of 128, bf16 to E4M3: 235 MB in 48 us, 4.9 TB/s), else the chain
// lengths -> values, page, table row -> largest -> codes: 16 tokens 5.9 us, 16 sequences of 24 with a tree 7.2.  The prompts again and again on the same tensors: 42 us,
// as two calls 53; on the way there, a unit a thread and keys read twice, 59.
template <typename T, int CODE, int VEC, bool INTERLEAVED, int THREADS>
__global__ void __launch_bounds__(THREADS) kvcache_append_rope_kernel(AppendRopeArgs a)
{
    const Kv8& c = a.cache;
    const unsigned before_it = (unsigned)((blockIdx.x * a.share) >> 32);
    if ((unsigned)(((blockIdx.x + 1) * a.share) >> 32) == before_it) {
        turn_queries<T, VEC, INTERLEAVED, THREADS>(a, blockIdx.x - before_it);
        return;
    }
    const bool values = before_it % 2 != 0;
    const unsigned page_head = before_it / 2, nth_page = page_head / (unsigned)c.kv_heads;
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
    const int per_token = (c.head_dim + 2 * VEC - 1) / (2 * VEC), units = fresh * per_token;
    const uint8_t* src = a.src[values] + (int64_t)head * a.head[values];
    auto load = [&](int token, int u, float* x) __attribute__((always_inline)) {  // of the page's new tokens
        const int row_at = first + lo - start + token;
        const T* row = reinterpret_cast<const T*>(src + (int64_t)row_at * a.token[values]);
        if (values) {
            const Runs at = runs_of<VEC, true>(u, 0, c.head_dim);
            load_run<T, VEC>(row + at.lo, x);
            load_run<T, VEC>(row + at.hi, x + VEC);
        } else {
            load_turned<T, VEC, INTERLEAVED>(a, row, a.position(row_at, lo - start + token, count, start), u, c.head_dim, x);
        }
    };
    uint32_t largest = 0;
    constexpr int HELD = 16 / VEC;  // units of a thread that stay in registers, 32 values; others, of pages of more than 32 KB a head, are read again
    float held[HELD][2 * VEC];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int u = min((int)threadIdx.x + h * THREADS, units - 1);
        load(u / per_token, u % per_token, held[h]);
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i)
            largest = max(largest, f2u(held[h][i]) & 0x7FFFFFFFu);
    for (int u = threadIdx.x + HELD * THREADS; u < units; u += THREADS) {
        float x[2 * VEC];
        load(u / per_token, u % per_token, x);
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i)
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
    const float after = kv8_grown_scale<CODE>(before, largest);
    if (threadIdx.x == 0)
        *scale = after;
    uint8_t* dst = side.codes + (int64_t)page * side.page + (int64_t)head * side.head;
    if (before < after) {  // the older tokens' codes in the new unit
        const float ratio = before / after;
        const int chunks = c.head_dim / 8;
        for (int u = threadIdx.x; u < older * chunks; u += THREADS) {
            uint2* p = reinterpret_cast<uint2*>(dst + (int64_t)(u / chunks) * side.token + (u % chunks) * 8);
            *p = kv8_scaled_codes<CODE>(*p, ratio);
        }
    }
    const float inverse = after > 0.0f ? 1.0f / after : 0.0f;
    auto write = [&](int u, float* x) __attribute__((always_inline)) {
        const int token = u / per_token;
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i)
            x[i] = inverse > 0.0f ? x[i] * inverse : 0.0f;  // (a NaN scale: codes of zero)
        const Runs at = values ? runs_of<VEC, true>(u % per_token, 0, c.head_dim) : runs_of<VEC, INTERLEAVED>(u % per_token, a.half, c.head_dim);
        uint8_t* to = dst + (int64_t)(older + token) * side.token;
        store_codes<CODE, VEC>(to + at.lo, x);
        store_codes<CODE, VEC>(to + at.hi, x + VEC);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (threadIdx.x + h * THREADS < (unsigned)units)
            write(threadIdx.x + h * THREADS, held[h]);
    for (int u = threadIdx.x + HELD * THREADS; u < units; u += THREADS) {
        float x[2 * VEC];
        load(u / per_token, u % per_token, x);
        write(u, x);
    }
}

template <typename T, int CODE, int VEC, bool INTERLEAVED, int THREADS>
static int launch_append_rope(AppendRopeArgs a, int sequences, hipStream_t stream)
{
    const long units = (long)a.heads * ((a.cache.head_dim + 2 * VEC - 1) / (2 * VEC));
    const long wide = (units + THREADS - 1) / THREADS, append = 2L * sequences * a.blocks * a.cache.kv_heads;
    // (without cu_tokens a row's sequence is a division away and all have the same tokens)
    const long pairs = a.cache.cu_tokens == nullptr ? (a.cache.max_tokens + ROPE_TOKENS - 1) / ROPE_TOKENS : 0;
    const long groups = append + (pairs > 0 ? sequences * pairs : (a.cache.tokens + ROPE_TOKENS - 1) / ROPE_TOKENS) * wide;
    PTOAMD_REQUIRE(groups <= 0x7FFFFFFF, PTOAMD_E_UNSUPPORTED, "ptoamd_kvcache_append_rope: %d sequences of %d tokens are too many for one launch", sequences,
                   a.cache.max_tokens);
    a.wide = (unsigned)(wide > 0 ? wide : 1);
    a.pairs = (unsigned)pairs;
    a.sequences = sequences;
    a.share = (((uint64_t)append << 32) + groups - 1) / groups;  // (rounded up: after all workgroups, all of the append have been)
    hipLaunchKernelGGL((kvcache_append_rope_kernel<T, CODE, VEC, INTERLEAVED, THREADS>), dim3((unsigned)groups), dim3(THREADS), 0, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("kvcache_append_rope");
    return PTOAMD_OK;
}
// Threads by the bytes that a page's new tokens have of a head, as in kvcache.hip.
template <typename T, int CODE, int VEC, bool INTERLEAVED>
static int choose_threads(const AppendRopeArgs& a, int sequences, hipStream_t stream)
{
    const int page = 1 << a.cache.page_shift;
    const long bytes = (long)(a.cache.max_tokens < page ? a.cache.max_tokens : page) * a.cache.head_dim * sizeof(T);
    if (bytes <= 8192)
        return launch_append_rope<T, CODE, VEC, INTERLEAVED, 128>(a, sequences, stream);
    if (bytes <= 16384)
        return launch_append_rope<T, CODE, VEC, INTERLEAVED, 256>(a, sequences, stream);
    return launch_append_rope<T, CODE, VEC, INTERLEAVED, 512>(a, sequences, stream);
}
// Runs of eight elements where the rotation is made of them and operands start on theirs (16 bytes), else of four, else single elements.
template <typename T, int CODE, bool INTERLEAVED>
static int choose_run(const AppendRopeArgs& a, int sequences, hipStream_t stream)
{
    uint64_t bits = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.q_out | (uint64_t)a.q_token | (uint64_t)a.q_head | (uint64_t)a.out_token |
                    (uint64_t)a.out_head;
    for (int i = 0; i < 2; ++i)
        bits |= (uint64_t)(uintptr_t)a.src[i] | (uint64_t)a.token[i] | (uint64_t)a.head[i];
    const uint64_t table = (uint64_t)(uintptr_t)a.table;
    if (a.half % 8 == 0 && bits % 16 == 0 && table % 16 == 0)
        return choose_threads<T, CODE, 8, INTERLEAVED>(a, sequences, stream);
    if (a.half % 4 == 0 && bits % (4 * sizeof(T)) == 0 && table % 16 == 0)
        return choose_threads<T, CODE, 4, INTERLEAVED>(a, sequences, stream);
    return launch_append_rope<T, CODE, 1, INTERLEAVED, 256>(a, sequences, stream);
}
template <typename T, int CODE>
static int choose_order(const AppendRopeArgs& a, int sequences, hipStream_t stream)
{
    return a.interleaved ? choose_run<T, CODE, true>(a, sequences, stream) : choose_run<T, CODE, false>(a, sequences, stream);
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
    // (queries are written while other workgroups still read all of these)
    const HeadRows result{(uint64_t)(uintptr_t)q_out, tokens, heads, q_out_token_stride * size, q_out_head_stride * size, (int64_t)cache->head_dim * size};
    auto apart = [&](const void* p, int64_t bytes) { return !meet(result, memory_at(p, bytes)); };
    auto apart_from_rows = [&](const void* p, int n, int64_t token, int64_t head) {
        return !meet(result, HeadRows{(uint64_t)(uintptr_t)p, tokens, n, token * size, head * size, (int64_t)cache->head_dim * size});
    };
    PTOAMD_REQUIRE(q_out == q || apart_from_rows(q, heads, q_token_stride, q_head_stride), PTOAMD_E_INVALID, "%s: q_out must be q or not overlap it", what);
    PTOAMD_REQUIRE(apart_from_rows(k, cache->kv_heads, k_token_stride, k_head_stride) && apart_from_rows(v, cache->kv_heads, v_token_stride, v_head_stride),
                   PTOAMD_E_INVALID, "%s: q_out must not overlap k or v", what);
    PTOAMD_REQUIRE(apart(table, (int64_t)table_rows * rot_dim * 4) && apart(positions, tokens * 4L) && apart(tree, (int64_t)tokens * tree_words * 8), PTOAMD_E_INVALID,
                   "%s: q_out must not overlap table, positions or tree", what);
    PTOAMD_REQUIRE(apart(cu_tokens, 4L * (cache->sequences + 1)) && apart(cache->lengths, 4L * cache->sequences) &&
                       apart(cache->block_table, 4L * cache->sequences * cache->max_pages) && apart(cache->k_scale, 4L * cache->pages * cache->kv_heads) &&
                       apart(cache->v_scale, 4L * cache->pages * cache->kv_heads),
                   PTOAMD_E_INVALID, "%s: q_out must not overlap cu_tokens, lengths, block_table or the scales", what);
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
