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

// The largest magnitude among eight codes, in units of their scale.
template <int CODE>
__device__ __forceinline__ float largest_code(uint2 w)
{
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        code = max(code, f2u(kv8_value<CODE>(((i < 4 ? w.x : w.y) >> (8 * (i % 4))) & 0xFFu)) & 0x7FFFFFFFu);
    return u2f(code);
}
template <int CODE>
__device__ __forceinline__ uint2 scaled_codes(uint2 w, float by)
{
    return by == 1.0f ? w : kv8_scaled_codes<CODE>(w, by);
}

// One workgroup a sequence, head and side (keys or values).  Tokens only move down, in ascending order.  Lists of up to 64 entries that fit its registers (32
// codes a thread: 64 tokens of heads of 128): everything is read, then everything written, one chain list -> table -> scales and codes -> largest of each page.
// Else pages that tokens move into one after the other: what a page takes is read before it is written, and what is written lies before all that is still to
// be read.
// Bound: the launch and that chain.  48 sequences, 16 heads of 64, up to 24 tokens over three pages of 16: 10.4 us page by page, 6.5 at once.  On either side
// of the bound, us, int8 / E4M3: 16 sequences, 8 heads of 128, pages of 64, 64 tokens of 64 4.4 / 4.4, 65 of 72 7.8 / 8.6; 48, 16 of 64, pages of 16, 64 of 200
// 8.9 / 12.2, 65 17.9 / 24.6 (128 27.9 / 37.9: 2.5 / 3.3 a further page, the chain of each); 64, 8 of 256, pages of 64, 32 of 40 8.1 / 9.1, 33 10.2 / 11.4.
// The longest lists, 64 x 200 of 256, 8 heads of 256, pages of 16: 66 / 94.
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
    const int entries = min(a.max_kept, count);  // of the list, those before the first that is out of order
    const int chunks = c.head_dim / 8, slots = (1 << c.page_shift) - 1;
    constexpr int HELD = 4;
    if (entries <= 64 && entries * chunks <= HELD * KEEP_THREADS) {
        // Every wave has the list for itself, an entry a lane, and the pages that tokens come to, another lane's each.
        const int lane = tid % 64;
        const int own = lane < entries ? a.kept[(int64_t)seq * a.max_kept + lane] : -1, below = __shfl_up(own, 1);
        const uint64_t bad = ~__ballot(whole && lane < entries && own > (lane > 0 ? below : -1) && own < count);
        const int kept = bad != 0 ? __builtin_ctzll(bad) : 64;
        if (head == 0 && blockIdx.z == 0 && tid == 0)
            a.new_lengths[seq] = whole ? start + kept : length;
        if (!whole || kept == 0)
            return;
        constexpr int BLOCKS = 64 / 16 + 1;
        __shared__ uint32_t comes[BLOCKS];  // bits of the largest magnitude that comes into a page from others, and 1; 0: nothing does
        const int first_block = start >> c.page_shift, blocks = ((start + kept - 1) >> c.page_shift) - first_block + 1, units = kept * chunks;
        auto scale_of_page = [&](int page) { return side.scales + (int64_t)page * c.kv_heads + head; };
        const int its_page = lane < kept ? c.page_of(seq, (start + own) >> c.page_shift) : -1;
        const int block_page = lane < blocks ? c.page_of(seq, first_block + lane) : -1;
        if (tid < BLOCKS)
            comes[tid] = 0;
        uint2 held[HELD];
        int token[HELD], source[HELD], page[HELD];  // of a unit: its token, the place and the page that it comes from
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (h * KEEP_THREADS >= units)
                break;
            const int u = tid + h * KEEP_THREADS, nth = min(u / chunks, kept - 1);
            token[h] = nth;
            source[h] = start + __shfl(own, nth);
            page[h] = __shfl(its_page, nth);
            held[h] = *reinterpret_cast<const uint2*>(side.codes + (int64_t)max(page[h], 0) * side.page + (int64_t)head * side.head +
                                                      (int64_t)(source[h] & slots) * side.token + u % chunks * 8);
        }
        const float its_scale = its_page >= 0 ? *scale_of_page(its_page) : NAN, block_scale = block_page >= 0 ? *scale_of_page(block_page) : 0.0f;
        __syncthreads();
        float scale[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (h * KEEP_THREADS >= units)
                break;
            const int u = tid + h * KEEP_THREADS, nth = token[h];
            scale[h] = __shfl(its_scale, nth);
            if (u < units && source[h] >> c.page_shift != (start + nth) >> c.page_shift)
                atomicMax(&comes[((start + nth) >> c.page_shift) - first_block], (f2u(largest_code<CODE>(held[h]) * scale[h]) & 0x7FFFFFFFu) + 1);
        }
        __syncthreads();  // (every scale has been read, too)
        const uint32_t largest = comes[min(lane, BLOCKS - 1)];
        const float block_now = largest != 0 ? kv8_grown_scale<CODE>(block_scale, largest - 1) : block_scale;
        if (tid < blocks && block_page >= 0 && largest != 0)
            *scale_of_page(block_page) = block_now;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (h * KEEP_THREADS >= units)
                break;
            const int u = tid + h * KEEP_THREADS, nth = token[h], place = start + nth, block = (place >> c.page_shift) - first_block;
            const float old = __shfl(block_scale, block), now = __shfl(block_now, block);
            const int to = __shfl(block_page, block);
            float by = old < now ? old / now : 1.0f;
            if (source[h] >> c.page_shift != place >> c.page_shift)  // (a NaN scale, or no page: codes of zero)
                by = now > 0.0f && page[h] >= 0 ? scale[h] / now : 0.0f;
            if (u < units && to >= 0 && !(source[h] == place && by == 1.0f))
                *reinterpret_cast<uint2*>(side.codes + (int64_t)to * side.page + (int64_t)head * side.head + (int64_t)(place & slots) * side.token + u % chunks * 8) =
                    scaled_codes<CODE>(held[h], by);
        }
        const float old = __shfl(block_scale, 0), now = __shfl(block_now, 0);
        const int to = __shfl(block_page, 0);
        if (to >= 0 && old < now)  // the older tokens' codes in the new unit
            for (int u = tid; u < (start & slots) * chunks; u += KEEP_THREADS) {
                uint2* p = reinterpret_cast<uint2*>(side.codes + (int64_t)to * side.page + (int64_t)head * side.head + (int64_t)(u / chunks) * side.token +
                                                    u % chunks * 8);
                *p = scaled_codes<CODE>(*p, old / now);
            }
        return;
    }
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
    const int step = KEEP_THREADS / chunks > 0 ? KEEP_THREADS / chunks : 1;  // tokens at a time
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
                most = largest_code<CODE>(w) * side.scales[(int64_t)source * c.kv_heads + head];
            }
            largest = max(largest, f2u(most) & 0x7FFFFFFFu);
        }
        largest = largest_of_group(largest, wave_largest);
        float now = old;
        if (__syncthreads_or(others)) {
            now = kv8_grown_scale<CODE>(old, largest);
            if (tid == 0)
                *scale = now;
        }
        const float grown = old < now ? old / now : 1.0f;
        auto write = [&](int slot, int chunk, uint2 w, float by) {
            *reinterpret_cast<uint2*>(dst + (int64_t)slot * side.token + chunk * 8) = scaled_codes<CODE>(w, by);
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
    // (all of a sequence's workgroups read its length, its list and its place in the batch)
    auto apart = [&](const int32_t* p, long n) { return p == nullptr || new_lengths + cache->sequences <= p || p + n <= new_lengths; };
    PTOAMD_REQUIRE(apart(cache->lengths, cache->sequences), PTOAMD_E_INVALID, "%s: new_lengths must not be lengths", what);
    PTOAMD_REQUIRE(apart(kept, (long)cache->sequences * max_kept) && apart(cu_tokens, cache->sequences + 1L), PTOAMD_E_INVALID,
                   "%s: new_lengths must not overlap kept or cu_tokens", what);
    PTOAMD_REQUIRE(apart(cache->block_table, (long)cache->sequences * cache->max_pages) &&
                       apart(reinterpret_cast<const int32_t*>(cache->k_scale), (long)cache->pages * cache->kv_heads) &&
                       apart(reinterpret_cast<const int32_t*>(cache->v_scale), (long)cache->pages * cache->kv_heads),
                   PTOAMD_E_INVALID, "%s: new_lengths must not overlap block_table or the scales", what);
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
