// Keeping a path of drafted tokens: their keys and values move together in the pages of an 8-bit cache.
#include "common_host.hpp"
#include "kv8.hpp"
#include "kv8_codes.hpp"
#include "kv8_places.hpp"

namespace ptoamd {

struct KeepArgs {
    Kv8 cache;
    const int32_t* kept;
    int32_t* new_lengths;
    int max_kept;
};
constexpr int KEEP_THREADS = 256;
static_assert(KEEP_THREADS >= PTOAMD_MOST_DRAFTED, "a thread looks at an entry of a list");

// The workgroup's largest value.
__device__ __forceinline__ uint32_t largest_of_group(uint32_t x, uint32_t* wave_largest)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        x = max(x, (uint32_t)__shfl_xor((int)x, d));
    __syncthreads();  // (the last use of the room)
    if (threadIdx.x % 64 == 0)
        wave_largest[threadIdx.x / 64] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KEEP_THREADS / 64; ++w)
        x = max(x, wave_largest[w]);
    return x;
}

// One workgroup a sequence, head and side (keys or values); pages that tokens move into one after the other.  Tokens only move down, in ascending order:
// what a page takes is read before it is written, and what is written lies before all that is still to be read.
template <int CODE>
__global__ void __launch_bounds__(KEEP_THREADS) kvcache_keep_kernel(KeepArgs a)
{
    __shared__ int from[PTOAMD_MOST_DRAFTED];
    __shared__ uint32_t wave_largest[KEEP_THREADS / 64];
    const Kv8& c = a.cache;
    const int seq = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    const Kv8Side side = blockIdx.z != 0 ? c.v : c.k;
    const int first = c.first_token(seq), count = c.token_count(seq, first), length = max(c.lengths[seq], 0), start = length - count;
    const bool whole = start >= 0 && length <= c.max_pages << c.page_shift;
    // the entries before the first that is out of order
    const int entries = min(a.max_kept, count);
    int own = -1, before = -1;
    if (tid < entries) {
        own = a.kept[(int64_t)seq * a.max_kept + tid];
        before = tid > 0 ? a.kept[(int64_t)seq * a.max_kept + tid - 1] : -1;
        from[tid] = own;
    }
    const bool good = whole && tid < entries && own > before && own < count;
    const int kept = KEEP_THREADS - (int)largest_of_group(good ? 0u : (uint32_t)(KEEP_THREADS - tid), wave_largest);
    if (head == 0 && blockIdx.z == 0 && tid == 0)
        a.new_lengths[seq] = whole ? start + kept : length;
    if (!whole || kept == 0)
        return;
    const int chunks = c.head_dim / 8, step = KEEP_THREADS / chunks > 0 ? KEEP_THREADS / chunks : 1;  // tokens at a time
    const int slots = (1 << c.page_shift) - 1;
    for (int block = start >> c.page_shift; block <= (start + kept - 1) >> c.page_shift; ++block) {
        const int page = c.page_of(seq, block);
        if (page < 0)
            continue;
        const int lo = max(start, block << c.page_shift) - start, hi = min(start + kept, (block + 1) << c.page_shift) - start;
        uint8_t* dst = side.codes + (int64_t)page * side.page + (int64_t)head * side.head;
        float* scale = side.scales + (int64_t)page * c.kv_heads + head;
        const float old = *scale;
        uint32_t largest = 0;
        bool others = false;
        for (int u = tid; u < (hi - lo) * chunks; u += KEEP_THREADS) {
            const int at = start + from[lo + u / chunks];
            if (at >> c.page_shift == block)
                continue;
            others = true;
            const int source = c.page_of(seq, at >> c.page_shift);
            float most = NAN;
            if (source >= 0) {
                const uint2 w = *reinterpret_cast<const uint2*>(side.codes + (int64_t)source * side.page + (int64_t)head * side.head +
                                                                (int64_t)(at & slots) * side.token + u % chunks * 8);
                uint32_t code = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    code = max(code, f2u(kv8_value<CODE>(((i < 4 ? w.x : w.y) >> (8 * (i % 4))) & 0xFFu)) & 0x7FFFFFFFu);
                most = u2f(code) * side.scales[(int64_t)source * c.kv_heads + head];
            }
            largest = max(largest, f2u(most) & 0x7FFFFFFFu);
        }
        largest = largest_of_group(largest, wave_largest);
        float now = old;
        if (__syncthreads_or(others)) {
            now = u2f(largest) * KV8_PER_LARGEST<CODE>;
            now = old > now ? old : now;
            now = now < 0x1p-126f ? 0.0f : now;
            if (largest >= 0x7F800000u || old != old)
                now = NAN;
            if (tid == 0)
                *scale = now;
        }
        const float grown = old < now ? old / now : 1.0f;
        auto write = [&](int slot, int chunk, uint2 w, float by) {
            if (by != 1.0f) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = kv8_value<CODE>(((i < 4 ? w.x : w.y) >> (8 * (i % 4))) & 0xFFu) * by;
                w = kv8_codes<CODE>(x);
            }
            *reinterpret_cast<uint2*>(dst + (int64_t)slot * side.token + chunk * 8) = w;
        };
        if (grown != 1.0f) {  // the older tokens' codes in the new unit
            const int older = start + lo - (block << c.page_shift);
            for (int u = tid; u < older * chunks; u += KEEP_THREADS)
                write(u / chunks, u % chunks, *reinterpret_cast<const uint2*>(dst + (int64_t)(u / chunks) * side.token + u % chunks * 8), grown);
        }
        for (int token = lo; token < hi; token += step) {
            for (int base = 0; base < min(step, hi - token) * chunks; base += KEEP_THREADS) {
                const int u = base + tid, nth = token + u / chunks, chunk = u % chunks;
                const bool mine = u < min(step, hi - token) * chunks;
                uint2 w = make_uint2(0, 0);
                float by = grown;
                const int at = start + (mine ? from[nth] : 0);
                if (mine) {
                    const int source = at >> c.page_shift == block ? page : c.page_of(seq, at >> c.page_shift);
                    if (source >= 0)
                        w = *reinterpret_cast<const uint2*>(side.codes + (int64_t)source * side.page + (int64_t)head * side.head +
                                                            (int64_t)(at & slots) * side.token + chunk * 8);
                    if (source != page) {
                        const float theirs = source >= 0 ? side.scales[(int64_t)source * c.kv_heads + head] : 0.0f;
                        by = now > 0.0f && source >= 0 ? theirs / now : 0.0f;  // (a NaN scale: codes of zero)
                    }
                }
                __syncthreads();
                if (mine && !(at == start + nth && by == 1.0f))
                    write((start + nth) & slots, chunk, w, by);
            }
        }
        __syncthreads();  // (the next page's reads come after)
    }
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

int ptoamd_kvcache_keep(const ptoamd_kv8_cache* cache, int32_t* new_lengths, const int32_t* kept, int max_kept, const int32_t* cu_tokens, int max_tokens,
                        void* stream)
{
    const char* what = "ptoamd_kvcache_keep";
    PTOAMD_REQUIRE(cache != nullptr, PTOAMD_E_INVALID, "%s: null cache", what);
    PTOAMD_REQUIRE(max_kept >= 0 && max_tokens > 0, PTOAMD_E_INVALID, "%s: max_tokens must be positive, max_kept not negative (%d, %d)", what, max_tokens, max_kept);
    PTOAMD_REQUIRE(max_tokens <= PTOAMD_MOST_DRAFTED, PTOAMD_E_UNSUPPORTED, "%s: at most %d tokens of a sequence are drafted (%d)", what, PTOAMD_MOST_DRAFTED,
                   max_tokens);
    KeepArgs a{};
    // (which rows of a step were whose does not matter here, only how many: any row may be the last)
    const long tokens = cu_tokens != nullptr ? 0x7FFFFFFFL : (long)cache->sequences * max_tokens;
    PTOAMD_REQUIRE(cache->sequences > 0 && tokens <= 0x7FFFFFFFL, PTOAMD_E_INVALID, "%s: sequences must be positive and not too many (%d)", what, cache->sequences);
    const int rc = kv8_from(what, cache, (int)tokens, cu_tokens, max_tokens, &a.cache);
    if (rc != PTOAMD_OK)
        return rc;
    TraceScope trace("KVCACHE_KEEP", "vector", max_kept, cache->kv_heads, cache->head_dim);
    trace.in(kept, cache->sequences, max_kept, "ND", PTOAMD_I32).in(cache->lengths, 1, cache->sequences, "ND", PTOAMD_I32)
        .out(cache->k, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type)
        .out(cache->v, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type);
    PTOAMD_REQUIRE(cache->head_dim % 8 == 0 && cache->head_dim <= 512, PTOAMD_E_UNSUPPORTED, "%s: head_dim must be a multiple of 8 and at most 512 (%d)", what,
                   cache->head_dim);
    PTOAMD_REQUIRE(new_lengths && (kept || max_kept == 0), PTOAMD_E_INVALID, "%s: null operand", what);
    PTOAMD_REQUIRE((reinterpret_cast<uintptr_t>(new_lengths) | reinterpret_cast<uintptr_t>(kept)) % 4 == 0, PTOAMD_E_ALIGNMENT,
                   "%s: kept and new_lengths must be aligned to their elements", what);
    // (all of a sequence's workgroups read its length)
    PTOAMD_REQUIRE(new_lengths + cache->sequences <= cache->lengths || cache->lengths + cache->sequences <= new_lengths, PTOAMD_E_INVALID,
                   "%s: new_lengths must not be lengths", what);
    a.kept = kept;
    a.new_lengths = new_lengths;
    a.max_kept = max_kept;
    const dim3 grid((unsigned)cache->sequences, (unsigned)cache->kv_heads, 2);
    if (cache->code_type == PTOAMD_I8)
        hipLaunchKernelGGL(kvcache_keep_kernel<PTOAMD_I8>, grid, dim3(KEEP_THREADS), 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL(kvcache_keep_kernel<PTOAMD_E4M3>, grid, dim3(KEEP_THREADS), 0, as_stream(stream), a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("kvcache_keep");
    return PTOAMD_OK;
}

}  // extern "C"
