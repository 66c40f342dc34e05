// Attention over an 8-bit cache for many queries: prompts and chunks of prompts.
#include "attention_kv8.hpp"

namespace ptoamd {

// A workgroup has 32 rows a wave of one sequence and key head (rows: new tokens times the query heads that share the key head, token-major,
// so those heads share what is staged) and walks the keys that its rows see in tiles of 64 (32 of heads of 256).  A tile's codes are read while the tile before
// is computed, become f16, exactly, once for all waves, and go to LDS in one of two buffers; one barrier a tile.
//   S^T = K q^T (32x32x16): a fragment is 8 elements of one key, q's fragments stay in registers.
//   o^T = V^T p^T : a lane has the scores of keys 8 (i / 4) + 4 (lane / 32) + i % 4 of 32 for its row; with eight of them as its share of a
//                 product's 16 keys the weights are the fragment as they stand, and V's fragment (the same keys of one element) comes from
//                 two transposing LDS reads of four keys each.
// Scores, references and sums are f32; a page's value scale goes into the weight (ValueScale).
template <int D>
struct ManyTile {
    static constexpr int KEYS = D == 256 ? 32 : 64;  // (heads of 256: the registers hold no scores of 64 keys beside q and the sums)
    static constexpr int BYTES = KEYS * D * 2;       // of the keys, and as many of the values
    // Keys: 16 lanes of a read take one chunk of 16 keys: chunks are permuted so that they fall on different banks.
    static __device__ __forceinline__ int key_at(int key, int chunk)
    {
        return key * (2 * D) + ((chunk ^ (D == 64 ? (key >> 1) & 7 : key & 15)) * 16);
    }
    // Values: 32 lanes of a transposing read take 64 bytes of four keys: pieces of 32 bytes are permuted in pairs.
    static __device__ __forceinline__ int value_at(int key, int piece)
    {
        return key * (2 * D) + ((piece ^ (D == 64 ? ((key >> 1) & 1) << 1 : (key & 3) << 1)) * 32);
    }
};

template <typename T, int CODE, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) attention_kv8_many_kernel(AttentionArgs a)
{
    typedef ManyTile<D> Tile;
    constexpr int THREADS = 64 * WAVES, KEYS = Tile::KEYS, STEPS = D / 16, DT = D / 32;
    constexpr int SIDE_UNITS = KEYS * D / 16, UNITS = 2 * SIDE_UNITS / THREADS;  // 16 codes each; a thread's
    extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];                   // [2][keys, values]
    __shared__ float4 scales[2][KEYS / 16];                                                   // of 16 keys: key scale, value scale's log2 and inverse
    const Kv8& c = a.cache;
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), col = lane % 32, hf = lane / 32;
    const int kv_head = blockIdx.x % c.kv_heads, part = blockIdx.y, seq = blockIdx.z;
    const int row_tiles = gridDim.x / c.kv_heads, row_tile = row_tiles - 1 - blockIdx.x / c.kv_heads;  // (those with most keys first)
    const Span span = span_of(a, seq);
    const int rows = span.count * a.group, row0 = row_tile * 32 * WAVES;
    if (row0 >= rows)
        return;
    // the keys that any row of the workgroup sees, and of the part
    const int place0 = span.length - span.count;
    const int from = visible_keys(a, place0 + row0 / a.group, span.length).x;
    const int to = visible_keys(a, place0 + (min(row0 + 32 * WAVES, rows) - 1) / a.group, span.length).y;
    int begin = from & ~31, end = to;
    if (a.splits > 1) {
        begin = max(begin, span.begin + part * a.chunk);
        if (part + 1 < a.splits)
            end = min(end, span.begin + (part + 1) * a.chunk);
    }
    if (begin >= end && part > 0)
        return;

    const int row = row0 + 32 * wave + col, token = row / a.group;
    const bool valid = row < rows;
    const int head = kv_head * a.group + (valid ? row - token * a.group : 0);
    const int2 seen = valid ? visible_keys(a, place0 + token, span.length) : make_int2(0, 0);
    uint4 q[STEPS];
    float cq;
    {
        const uint8_t* p = a.q + (int64_t)(span.first + (valid ? token : 0)) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
            q[st] = valid ? load_row8(p + 2 * (16 * st + 8 * hf), a.wide) : make_uint4(0, 0, 0, 0);
        float largest = largest_of<T, STEPS>(q);
        largest = fmaxf(largest, __shfl_xor(largest, 32));
        const RowScale r = row_scale(largest);
        cq = r.up * (a.scale * 1.44269504088896341f);
        scale_to_f16<T, STEPS>(q, r.down);
    }
    // of the wave's rows: keys that any sees, and that every one sees
    const int wave_row = row0 + 32 * wave, wave_first = place0 + min(wave_row, rows - 1) / a.group, wave_last = place0 + (min(wave_row + 32, rows) - 1) / a.group;
    const bool working = wave_row < rows;
    const int any_from = visible_keys(a, wave_first, span.length).x, any_to = working ? visible_keys(a, wave_last, span.length).y : 0;
    const int every_from = visible_keys(a, wave_last, span.length).x, every_to = working ? visible_keys(a, wave_first, span.length).y : 0;

    // what a thread stages: units of 16 codes; unit u of the tile's: side, key, 16 elements of it
    const int last_key = max(span.length - 1, 0), slot_mask = (1 << c.page_shift) - 1;
    const int32_t* table = c.table + (int64_t)seq * c.max_pages;
    int ids[UNITS], scale_id = 0;
    uint4 raw[UNITS];
    float2 raw_scale = make_float2(0, 0);
    float unit_scale[UNITS];  // of values: the scale of their page
    auto unit_key = [&](int u) { return ((tid + u * THREADS) % SIDE_UNITS) / (D / 16); };
    auto find = [&](int key) {  // page ids of a tile
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
            ids[u] = table[min(key + unit_key(u), last_key) >> c.page_shift];
        if (tid < KEYS / 16)
            scale_id = table[min(key + 16 * tid, last_key) >> c.page_shift];
    };
    auto fetch = [&](int key) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const Kv8Side side = (tid + u * THREADS) / SIDE_UNITS ? c.v : c.k;
            const int64_t page = (unsigned)ids[u] < (unsigned)c.pages ? ids[u] : 0;
            const int slot = min(key + unit_key(u), last_key) & slot_mask;
            unit_scale[u] = side.scales[page * c.kv_heads + kv_head];
            raw[u] = *reinterpret_cast<const uint4*>(side.codes + page * side.page + kv_head * side.head + slot * side.token + (tid + u * THREADS) % (D / 16) * 16);
        }
        if (tid < KEYS / 16) {
            const bool known = (unsigned)scale_id < (unsigned)c.pages;
            const int64_t at = (int64_t)(known ? scale_id : 0) * c.kv_heads + kv_head;
            raw_scale = make_float2(known ? c.k.scales[at] : NAN, known ? c.v.scales[at] : NAN);
        }
    };
    auto stage = [&](int key, int buffer) {
        uint8_t* to_tile = tiles + buffer * 2 * Tile::BYTES;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const bool value = (tid + u * THREADS) / SIDE_UNITS;
            const int k = unit_key(u), chunk = (tid + u * THREADS) % (D / 16) * 2;
            uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            if (value && (key + k < from || key + k >= to || unit_scale[u] < LEAST_SCALE)) {  // a weight of zero does not undo a NaN code that no row sees
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = 0u;
            }
            uint32_t f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t x = kv8_turn<CODE>(w[i]);
                f[2 * i] = kv8_pair_to_f16<CODE, false>(x);
                f[2 * i + 1] = kv8_pair_to_f16<CODE, true>(x);
            }
            uint4* at0 = reinterpret_cast<uint4*>(value ? to_tile + Tile::BYTES + Tile::value_at(k, chunk / 2) : to_tile + Tile::key_at(k, chunk));
            uint4* at1 = reinterpret_cast<uint4*>(value ? to_tile + Tile::BYTES + Tile::value_at(k, chunk / 2) + 16 : to_tile + Tile::key_at(k, chunk + 1));
            *at0 = make_uint4(f[0], f[1], f[2], f[3]);
            *at1 = make_uint4(f[4], f[5], f[6], f[7]);
        }
        if (tid < KEYS / 16) {
            const ValueScale v = value_scale(raw_scale.y);
            scales[buffer][tid] = make_float4(raw_scale.x, v.log2, v.inverse, 0.0f);
        }
    };

    f32x16 o[DT];
    float top = NO_REFERENCE, sum = 0.0f;
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            o[m][i] = 0.0f;

    auto compute = [&](int key, int buffer) {
        const uint8_t* keys = tiles + buffer * 2 * Tile::BYTES;
        const uint8_t* values = keys + Tile::BYTES;
        f32x16 s[KEYS / 32];
#pragma unroll
        for (int kt = 0; kt < KEYS / 32; ++kt) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[kt][i] = 0.0f;
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const uint4 f = *reinterpret_cast<const uint4*>(keys + Tile::key_at(32 * kt + col, 2 * st + hf));
                s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f), __builtin_bit_cast(f16x8, q[st]), s[kt], 0, 0, 0);
            }
        }
        const bool whole = key >= every_from && key + KEYS <= every_to;
        float4 sc[KEYS / 16];  // of 16 keys, 8 of them this lane's
        float scale[KEYS / 16], high = -INFINITY;
        // (the largest of a group's scores times its scale: the scale is not negative)
#pragma unroll
        for (int x = 0; x < KEYS / 16; ++x) {
            sc[x] = scales[buffer][x];
            scale[x] = cq * sc[x].x;
        }
        if (whole) {
#pragma unroll
            for (int x = 0; x < KEYS / 16; ++x) {
                float eight = s[x / 2][8 * (x % 2)];
#pragma unroll
                for (int i = 1; i < 8; ++i)
                    eight = fmaxf(eight, s[x / 2][8 * (x % 2) + i]);
                high = fmaxf(high, fmaf(eight, scale[x], sc[x].y));
            }
        } else {
            const uint32_t first = (uint32_t)(key + 4 * hf - seen.x), count = (uint32_t)(seen.y - seen.x);
#pragma unroll
            for (int x = 0; x < KEYS / 16; ++x)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float w = fmaf(s[x / 2][8 * (x % 2) + i], scale[x], sc[x].y);
                    s[x / 2][8 * (x % 2) + i] = first + (16 * x + 8 * (i / 4) + i % 4) < count ? w : -INFINITY;
                    high = fmaxf(high, s[x / 2][8 * (x % 2) + i]);
                }
#pragma unroll
            for (int x = 0; x < KEYS / 16; ++x) {  // (these are scores already)
                scale[x] = 1.0f;
                sc[x].y = 0.0f;
            }
        }
        if (__ballot(high > top + MOST) != 0) {
            high = fmaxf(high, __shfl_xor(high, 32));
            const float next = fmaxf(top, high - SET_TO), fade = __builtin_amdgcn_exp2f(top - next);
            top = next;
            sum *= fade;
#pragma unroll
            for (int m = 0; m < DT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[m][i] *= fade;
        }
#pragma unroll
        for (int x = 0; x < KEYS / 16; ++x) {
            float w[8], eight = 0.0f;
            const float less = sc[x].y - top;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + i], scale[x], less));
                eight += w[i];
            }
            sum = eight == 0.0f ? sum : fmaf(eight, sc[x].z, sum);  // (a NaN scale that the row does not see)
            const uint4 p = make_uint4(pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7]));
#pragma unroll
            for (int m = 0; m < DT; ++m) {
                // a group of 16 lanes: four keys of 16 elements; each lane names 8 bytes and gets its own element of the four
                const int l16 = lane % 16, k = 16 * x + 4 * hf + l16 / 4, piece = 2 * m + (lane / 16) % 2;
                const uint4 f = read_transposed_16(values + Tile::value_at(k, piece) + l16 % 4 * 8, values + Tile::value_at(k + 8, piece) + l16 % 4 * 8);
                o[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f), __builtin_bit_cast(f16x8, p), o[m], 0, 0, 0);
            }
        }
    };

    if (begin < end) {
        find(begin);
        fetch(begin);
        find(begin + KEYS);
        stage(begin, 0);
        __syncthreads();
        int buffer = 0;
        for (int key = begin; key < end; key += KEYS, buffer ^= 1) {
            if (key + KEYS < end) {
                fetch(key + KEYS);
                find(key + 2 * KEYS);
            }
            if (key < any_to && key + KEYS > any_from)
                compute(key, buffer);
            if (key + KEYS < end)
                stage(key + KEYS, buffer ^ 1);
            __syncthreads();
        }
    }

    sum += __shfl_xor(sum, 32);
    if (!valid)
        return;
    const int64_t at = (int64_t)(span.first + token) * a.heads + head;
    if (a.splits > 1) {
        float* out = a.part_out + ((int64_t)part * c.tokens * a.heads + at) * D + 4 * hf;
#pragma unroll
        for (int m = 0; m < DT; ++m)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(out + 32 * m + 2 * i) = f32x4{o[m][i], o[m][i + 1], o[m][i + 2], o[m][i + 3]};
        if (hf == 0)
            a.part_sum[(int64_t)part * c.tokens * a.heads + at] = make_float2(top, sum);
        return;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = reinterpret_cast<T*>(a.out + (int64_t)(span.first + token) * a.out_token + (int64_t)head * a.out_head) + 4 * hf;
    struct alignas(8) Four { T e[4]; };
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            Four x;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x.e[j] = (T)(sum == 0.0f ? 0.0f : o[m][i + j] * inverse);
            if (a.wide) {
                *reinterpret_cast<Four*>(out + 32 * m + 2 * i) = x;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    out[32 * m + 2 * i + j] = x.e[j];
            }
        }
    if (a.lse != nullptr && hf == 0)
        a.lse[at] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

template <typename T, int CODE, int D, int WAVES>
static int launch_many(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    constexpr int bytes = 4 * ManyTile<D>::BYTES;
    PTOAMD_HIP_CHECK((ensure_dynamic_lds<&attention_kv8_many_kernel<T, CODE, D, WAVES>>(bytes)));
    const long tiles = ((long)a.cache.max_tokens * a.group + 32 * WAVES - 1) / (32 * WAVES);
    hipLaunchKernelGGL((attention_kv8_many_kernel<T, CODE, D, WAVES>), dim3((unsigned)(tiles * a.cache.kv_heads), (unsigned)a.splits, (unsigned)sequences),
                       dim3(64 * WAVES), bytes, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    return PTOAMD_OK;
}
template <typename T, int CODE>
static int choose_size(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    switch (a.cache.head_dim) {
        case 64: return launch_many<T, CODE, 64, 8>(a, sequences, stream);
        case 128: return launch_many<T, CODE, 128, 8>(a, sequences, stream);
        default: return launch_many<T, CODE, 256, 4>(a, sequences, stream);
    }
}
int launch_attention_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream)
{
    if (f16)
        return code == PTOAMD_I8 ? choose_size<_Float16, PTOAMD_I8>(a, sequences, stream) : choose_size<_Float16, PTOAMD_E4M3>(a, sequences, stream);
    return code == PTOAMD_I8 ? choose_size<__bf16, PTOAMD_I8>(a, sequences, stream) : choose_size<__bf16, PTOAMD_E4M3>(a, sequences, stream);
}

}  // namespace ptoamd
