// The append to a cache of keys and values held in 8 bits: new tokens are quantised into their pages, one scale a page and head.
#include "common_host.hpp"
#include "kv8.hpp"
#include "kv8_places.hpp"
#include "lds_dma.hpp"

namespace ptoamd {

// The checks that every entry point makes of a cache, and the cache as the kernels take it.
int kv8_from(const char* what, const ptoamd_kv8_cache* c, int tokens, const int32_t* cu_tokens, int max_tokens, Kv8* out)
{
    PTOAMD_REQUIRE(c != nullptr, PTOAMD_E_INVALID, "%s: null cache", what);
    PTOAMD_REQUIRE(c->code_type == PTOAMD_I8 || c->code_type == PTOAMD_E4M3, PTOAMD_E_UNSUPPORTED, "%s: the cache's codes must be int8 or E4M3", what);
    PTOAMD_REQUIRE(c->pages > 0 && c->kv_heads > 0 && c->head_dim > 0 && c->sequences > 0 && c->max_pages > 0, PTOAMD_E_INVALID,
                   "%s: pages, kv_heads, head_dim, sequences and max_pages must be positive (%d, %d, %d, %d, %d)", what, c->pages, c->kv_heads, c->head_dim,
                   c->sequences, c->max_pages);
    int shift = 4;
    while (shift < 8 && (1 << shift) != c->page_size)
        ++shift;
    PTOAMD_REQUIRE(c->page_size == 1 << shift, PTOAMD_E_UNSUPPORTED, "%s: page_size must be 16, 32, 64, 128 or 256 (%d)", what, c->page_size);
    // (places are held in 32 bits, and the attention's loops step up to 1040 of them past a sequence's last key)
    PTOAMD_REQUIRE((long)c->max_pages * c->page_size <= 0x7FFF0000L, PTOAMD_E_UNSUPPORTED, "%s: max_pages pages of %d tokens are too many", what, c->page_size);
    PTOAMD_REQUIRE(c->kv_heads <= 65535 && c->sequences <= 65535, PTOAMD_E_UNSUPPORTED, "%s: more than 65535 key heads or sequences (%d, %d)", what, c->kv_heads,
                   c->sequences);
    PTOAMD_REQUIRE(tokens >= 0 && max_tokens >= 0, PTOAMD_E_INVALID, "%s: tokens and max_tokens must not be negative (%d, %d)", what, tokens, max_tokens);
    PTOAMD_REQUIRE(cu_tokens != nullptr || (long)c->sequences * max_tokens == tokens, PTOAMD_E_INVALID,
                   "%s: without cu_tokens, tokens must be sequences * max_tokens (%d, %d * %d)", what, tokens, c->sequences, max_tokens);
    if (tokens == 0)
        return PTOAMD_OK;
    PTOAMD_REQUIRE(c->k && c->v && c->k_scale && c->v_scale && c->block_table && c->lengths, PTOAMD_E_INVALID, "%s: null operand", what);
    const uint64_t bits = (uint64_t)(uintptr_t)c->k | (uint64_t)(uintptr_t)c->v | (uint64_t)c->k_page_stride | (uint64_t)c->k_head_stride |
                          (uint64_t)c->k_token_stride | (uint64_t)c->v_page_stride | (uint64_t)c->v_head_stride | (uint64_t)c->v_token_stride;
    PTOAMD_REQUIRE(bits % 8 == 0, PTOAMD_E_ALIGNMENT, "%s: the caches' addresses and strides must be multiples of 8 bytes", what);
    out->k = Kv8Side{static_cast<uint8_t*>(c->k), c->k_scale, c->k_page_stride, c->k_head_stride, c->k_token_stride};
    out->v = Kv8Side{static_cast<uint8_t*>(c->v), c->v_scale, c->v_page_stride, c->v_head_stride, c->v_token_stride};
    out->table = c->block_table;
    out->lengths = c->lengths;
    out->cu_tokens = cu_tokens;
    out->pages = c->pages;
    out->kv_heads = c->kv_heads;
    out->page_shift = shift;
    out->head_dim = c->head_dim;
    out->max_pages = c->max_pages;
    out->tokens = tokens;
    out->max_tokens = max_tokens < tokens ? max_tokens : tokens;  // (a loose bound: no sequence has more than all of them)
    return PTOAMD_OK;
}

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

struct AppendArgs {
    Kv8 cache;
    const uint8_t* src[2];           // k, v
    int64_t token[2], head[2];       // strides in bytes
    int blocks;                      // most pages that a sequence's new tokens touch
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, float* x)
{
    struct alignas(WIDE ? 16 : sizeof(T)) V { T e[16 / sizeof(T)]; };
    V v[8 * sizeof(T) / 16];
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
        v[i] = reinterpret_cast<const V*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = (float)v[i * sizeof(T) / 16].e[i % (16 / sizeof(T))];
}

// One workgroup a page of a sequence, head, and side (keys or values).  The new tokens' largest magnitude gives the page's scale, which
// only grows; where it grows, the older tokens' codes are rounded again to the new one.  A thread has 8 elements of a row at a time.
// Magnitudes are compared as integers, so that an infinity or a NaN among them is the largest, whatever the order.
// Bound: HBM (values read once, a byte a value written; the second read of a page's values comes from the L2) and the chain of loads of a
// workgroup that has 12 KB to move (lengths, values, page, scale).  Seven ragged prompts of up to 2048 tokens, 8 heads of 128, pages of 32,
// bf16 to E4M3: 48.5 MB in 13.5 us, 3.6 TB/s; one token of 48 sequences 7 us, a launch.  (Keys and values in one workgroup, their values in
// registers between the passes: 16.4 us in a graph where one side's without took 14.8, and one side's with 15.9.)
template <typename T, int CODE, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS) kvcache_append_kernel(AppendArgs a)
{
    const Kv8& c = a.cache;
    const int seq = blockIdx.x / a.blocks, nth = blockIdx.x - seq * a.blocks, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
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
    const int chunks = c.head_dim / 8, units = fresh * chunks;
    const uint8_t* src = a.src[values] + (int64_t)(first + lo - start) * a.token[values] + (int64_t)head * a.head[values];
    uint32_t largest = 0;
    for (int u = threadIdx.x; u < units; u += THREADS) {
        float x[8];
        load8<T, WIDE>(reinterpret_cast<const T*>(src + (int64_t)(u / chunks) * a.token[values]) + (u % chunks) * 8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
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
    const bool finite = largest < 0x7F800000u;
    float after = u2f(largest) * (CODE == PTOAMD_I8 ? 1.0f / 127.0f : 1.0f / 448.0f);
    after = before > after ? before : after;
    after = after < 0x1p-126f ? 0.0f : after;
    if (!finite || before != before)
        after = NAN;
    if (threadIdx.x == 0)
        *scale = after;
    uint8_t* dst = side.codes + (int64_t)page * side.page + (int64_t)head * side.head;
    if (before < after) {  // the older tokens' codes in the new unit
        const float ratio = before / after;
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
        float x[8];
        load8<T, WIDE>(reinterpret_cast<const T*>(src + (int64_t)(u / chunks) * a.token[values]) + (u % chunks) * 8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = inverse > 0.0f ? x[i] * inverse : 0.0f;  // (a NaN scale: codes of zero)
        *reinterpret_cast<uint2*>(dst + (int64_t)(older + u / chunks) * side.token + (u % chunks) * 8) = kv8_codes<CODE>(x);
    }
}

template <typename T, int CODE, int THREADS>
static int launch_append(const AppendArgs& a, int sequences, bool wide, hipStream_t stream)
{
    const dim3 grid((unsigned)((long)sequences * a.blocks), (unsigned)a.cache.kv_heads, 2);
    if (wide)
        hipLaunchKernelGGL((kvcache_append_kernel<T, CODE, true, THREADS>), grid, dim3(THREADS), 0, stream, a);
    else
        hipLaunchKernelGGL((kvcache_append_kernel<T, CODE, false, THREADS>), grid, dim3(THREADS), 0, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("kvcache_append");
    return PTOAMD_OK;
}
// Threads by the bytes that a page's new tokens have of a head: few enough that small pages' workgroups are many on a CU, enough that large ones are
// loaded at once.  4 sequences of 1024 tokens, 8 heads, us, 128 / 256 / 512 threads: bf16, heads of 64, pages of 16 (2 KB) 6.9 / 8.9 / 13.5; of 128, 32
// (8 KB) 8.4 / 8.3 / 10.4; 64 (16 KB) 10.0 / 8.6 / 8.5; 128 (32 KB) 12.4 / 9.4 / 9.2; of 256, 128 (64 KB) 31 / 19 / 16; f32, of 256, pages of 16 (16 KB)
// 24 / 19 / 19, of 32 (32 KB) 23 / 24 / 20; one token of 256 sequences, heads of 128, 5.9 / 7.9 / 12.5.
template <typename T, int CODE>
static int choose_threads(const AppendArgs& a, int sequences, bool wide, hipStream_t stream)
{
    const int page = 1 << a.cache.page_shift;
    const long bytes = (long)(a.cache.max_tokens < page ? a.cache.max_tokens : page) * a.cache.head_dim * sizeof(T);
    if (bytes <= 8192)
        return launch_append<T, CODE, 128>(a, sequences, wide, stream);
    return bytes <= 16384 ? launch_append<T, CODE, 256>(a, sequences, wide, stream) : launch_append<T, CODE, 512>(a, sequences, wide, stream);
}
template <typename T>
static int dispatch_append(const AppendArgs& a, int code, int sequences, hipStream_t stream)
{
    uint64_t bits = 0;
    for (int i = 0; i < 2; ++i)
        bits |= (uint64_t)(uintptr_t)a.src[i] | (uint64_t)a.token[i] | (uint64_t)a.head[i];
    return code == PTOAMD_I8 ? choose_threads<T, PTOAMD_I8>(a, sequences, bits % 16 == 0, stream)
                             : choose_threads<T, PTOAMD_E4M3>(a, sequences, bits % 16 == 0, stream);
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

int ptoamd_kvcache_append(const ptoamd_kv8_cache* cache, const void* k, const void* v, int type, int tokens, const int32_t* cu_tokens,
                          int max_tokens, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                          void* stream)
{
    AppendArgs a{};
    const int rc = kv8_from("ptoamd_kvcache_append", cache, tokens, cu_tokens, max_tokens, &a.cache);
    if (rc != PTOAMD_OK)
        return rc;
    TraceScope trace("KVCACHE_APPEND", "vector", tokens, cache->kv_heads, cache->head_dim);
    trace.in(k, tokens, (long)cache->kv_heads * cache->head_dim, "ND", type).in(v, tokens, (long)cache->kv_heads * cache->head_dim, "ND", type)
        .out(cache->k, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type)
        .out(cache->v, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type);
    PTOAMD_REQUIRE(type == PTOAMD_F32 || type == PTOAMD_F16 || type == PTOAMD_BF16, PTOAMD_E_UNSUPPORTED,
                   "ptoamd_kvcache_append: keys and values must be f32, f16 or bf16");
    PTOAMD_REQUIRE(cache->head_dim % 8 == 0 && cache->head_dim <= 512, PTOAMD_E_UNSUPPORTED,
                   "ptoamd_kvcache_append: head_dim must be a multiple of 8 and at most 512 (%d)", cache->head_dim);
    if (tokens == 0 || max_tokens == 0)
        return PTOAMD_OK;
    PTOAMD_REQUIRE(k && v, PTOAMD_E_INVALID, "ptoamd_kvcache_append: null operand");
    const int size = type == PTOAMD_F32 ? 4 : 2;
    PTOAMD_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % size == 0, PTOAMD_E_ALIGNMENT,
                   "ptoamd_kvcache_append: k and v must be aligned to their elements");
    a.src[0] = static_cast<const uint8_t*>(k);
    a.src[1] = static_cast<const uint8_t*>(v);
    a.token[0] = k_token_stride * size;
    a.token[1] = v_token_stride * size;
    a.head[0] = k_head_stride * size;
    a.head[1] = v_head_stride * size;
    a.blocks = pages_of(a.cache.max_tokens, a.cache.page_shift);
    PTOAMD_REQUIRE((long)cache->sequences * a.blocks <= 0x7FFFFFFF, PTOAMD_E_UNSUPPORTED, "ptoamd_kvcache_append: too many pages for one launch");
    hipStream_t s = as_stream(stream);
    switch (type) {
        case PTOAMD_F32: return dispatch_append<float>(a, cache->code_type, cache->sequences, s);
        case PTOAMD_F16: return dispatch_append<_Float16>(a, cache->code_type, cache->sequences, s);
        default: return dispatch_append<__bf16>(a, cache->code_type, cache->sequences, s);
    }
}

}  // extern "C"
