// Attention over a cache of keys and values held in 8 bits: the generic kernel, the choice of a kernel, the entry points.
#include "attention_kv8.hpp"
#include "overlap.hpp"

namespace ptoamd {

// One wave a query and head, in f32 throughout: a lane's key of 64 at a time, then a lane's elements of the result.  Any head_dim that
// is a multiple of 8 up to 512, any number of queries: what the other kernels are checked against, and what head sizes without a kernel
// of their own run on.  TREE: of drafted tokens, which see the older keys and the bits of their row.
template <typename T, int CODE, bool TREE>
__global__ void __launch_bounds__(64) attention_kv8_generic_kernel(AttentionArgs a)
{
    const Kv8& c = a.cache;
    const int nth = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, kv_head = head / a.group, lane = threadIdx.x;
    const int first = c.first_token(seq), count = c.token_count(seq, first);
    if (nth >= count)
        return;
    const int length = c.length(seq), dim = c.head_dim;
    const int old = length - count;
    const uint32_t* bits = TREE ? a.tree + (int64_t)(first + nth) * a.tree_words : nullptr;
    const int2 keys = TREE ? make_int2(first_of_older(bits, a.tree_words, count, nth, old, a.window), length) : visible_keys(a, old + nth, length);
    __shared__ float q[512], weight[64];  // (weights below 0: of keys that are not seen)
    const T* row = reinterpret_cast<const T*>(a.q + (int64_t)(first + nth) * a.q_token + (int64_t)head * a.q_head);
    for (int i = lane; i < dim; i += 64)
        q[i] = (float)row[i];
    float top = -INFINITY, total = 0.0f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        o[i] = 0.0f;
    for (int base = keys.x; base < keys.y; base += 64) {
        __syncthreads();  // q; the weights of the tile before have been read
        const int key = base + lane;
        float s = -INFINITY;
        const bool seen = TREE ? (seen_keys(bits, a.tree_words, base + (lane & 32), keys.x, old, length) >> (lane & 31) & 1u) != 0 : key < keys.y;
        if (seen) {
            const int page = c.page_of(seq, key >> c.page_shift), slot = key & ((1 << c.page_shift) - 1);
            const uint8_t* k = c.k.codes + (int64_t)max(page, 0) * c.k.page + (int64_t)kv_head * c.k.head + (int64_t)slot * c.k.token;
            float dot = 0.0f;
            for (int i = 0; i < dim; i += 8) {
                const uint2 w = *reinterpret_cast<const uint2*>(k + i);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    dot = fmaf(q[i + j], kv8_value<CODE>(((j < 4 ? w.x : w.y) >> (8 * (j % 4))) & 0xFFu), dot);
            }
            s = page < 0 ? NAN : dot * (c.k.scales[(int64_t)page * c.kv_heads + kv_head] * a.scale);
        }
        float high = s;  // (fmaxf leaves NaN out: a NaN score is no maximum and makes a NaN weight)
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
            high = fmaxf(high, __shfl_xor(high, d));
        const float before = top;
        top = fmaxf(top, high);
        const float from = top == -INFINITY ? 0.0f : top;
        const float p = expf(s - from), fade = expf(before - from);
        float sum = p;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
            sum += __shfl_xor(sum, d);
        total = total * fade + sum;
        weight[lane] = seen ? p : -1.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] *= fade;
        for (int j = 0; j < min(64, keys.y - base); ++j) {
            const float w = weight[j];
            if (TREE && w < 0.0f)
                continue;
            const int page = c.page_of(seq, (base + j) >> c.page_shift), slot = (base + j) & ((1 << c.page_shift) - 1);
            const uint8_t* v = c.v.codes + (int64_t)max(page, 0) * c.v.page + (int64_t)kv_head * c.v.head + (int64_t)slot * c.v.token;
            const float wv = page < 0 ? NAN : w * c.v.scales[(int64_t)page * c.kv_heads + kv_head];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 64 * i < dim)
                    o[i] = fmaf(wv, kv8_value<CODE>(v[lane + 64 * i]), o[i]);
        }
    }
    T* out = reinterpret_cast<T*>(a.out + (int64_t)(first + nth) * a.out_token + (int64_t)head * a.out_head);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 64 * i < dim)
            out[lane + 64 * i] = (T)(total == 0.0f ? 0.0f : o[i] * inverse);
    if (a.lse != nullptr && lane == 0)
        a.lse[(int64_t)(first + nth) * a.heads + head] = total == 0.0f ? -INFINITY : top + logf(total);
}

template <typename T, int CODE>
static int launch_generic(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    const dim3 grid((unsigned)a.cache.max_tokens, (unsigned)a.heads, (unsigned)sequences);
    if (a.tree != nullptr)
        hipLaunchKernelGGL((attention_kv8_generic_kernel<T, CODE, true>), grid, dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_kv8_generic_kernel<T, CODE, false>), grid, dim3(64), 0, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("attention_kv8_generic");
    return PTOAMD_OK;
}

// Which kernel runs and how the keys are split, from sizes alone: the same for the workspace's size as for the call.
//   few  : at most 96 rows (new tokens of a sequence times the query heads that share a key head), or 64 (32 of heads of 256) where the keys of
//          all heads and sequences are more than 64 KB a CU.  us, few / many, heads of 128: 8 sequences of 6000 keys, 8 key heads, 16 rows 24 / 62,
//          48 38 / 63, 64 46 / 65, 80 65 / 69; 32 of 8000 128 rows 353 / 278; one of 2000 48 rows 13 / 23, 96 15 / 25.  Of 256, 2 key heads, 32 of
//          8000: 48 130 / 114, 64 168 / 115; 8 of 6000: 40 45 / 42, 64 59 / 45; one of 60000 40 57 / 52.
//   many : more rows, 256 of them a workgroup (128 for heads of 256 elements)
// Of drafted tokens, 128 rows a workgroup (HALVES) where there are no more: us, 256 rows a workgroup / 128, 16 sequences of 8192 keys, 64 / 8 heads of 128
// E4M3, 16 tokens 147 / 105, one of 131072 150 / 110; of 64, 119 / 77; and 32 tokens, 256 rows, 179 / 180, 48 271 / 281, 64 291 / 334.  The few-rows
// kernel takes up to 64 rows (32 of heads of 256), and more where its workgroups of 32 rows (16) are few: 2 a CU of heads of 128, 3 of 64, 4 of 256, or
// 1, 2, 2 of up to two turns of 256 keys; and have 18 turns a CU or fewer, 32 of heads of 64.  us, few / many, E4M3, rows a key head x sequences x keys, 64 / 8 heads
// of 128, around that bound: 256 x 8 x 2304, 2560, 2816 47 / 51, 50 / 54, 53 / 56 (18, 20 and 22 turns); 256 x 1 x 16384, 17408, 18432, 19456 (16 to 19) 40 /
// 49, 62 / 50, 64 / 51, 66 / 51 (the five parts of more than 16384 keys are 1.25 rounds); 512 x 2 x 4096, 4608, 4864 34 / 48, 51 / 49, 52 / 51.  So at 17 and
// 18 the rule is up to a quarter off for one long sequence, as it is in this table for 768 x 2 x 8000 of 64 (many is taken, 73 for 63), 128 x 16 x 1000 (few,
// 33 for 30) and 384 x 8 x 300 of 64 (many, 17 for 15).  Of 128: 512 x 1 x 300, 1000, 3000, 6000, 16000 9 / 21, 14 / 37, 24 / 42, 32 / 45, 72 / 65; 1024 x 1 x
// 3000 30 / 45; 256 x 1 x 16000 41 / 49, 60000 137 / 90; 128 x 16 x 300, 1000, 2000 22 / 18, 33 / 30, 45 / 49; 256 x 8 x 300, 1000, 2000 22 / 21, 32 / 42, 45 /
// 52; 384 x 8 47 / 41, 65 / 66 of 1000, 2000; 80 x 16 x 8192 163 / 100; a quarter to all of 192 x 8 x up to 1000, 2000 21 / 28, 25 / 34; of 64: 512 x 4 x 300,
// 1000, 3000 12 / 17, 18 / 34, 31 / 46; 384 x 8 x 300, 1000, 2000 16 / 18, 23 / 34, 33 / 58; 128 x 32 x 300, 1000 19 / 14, 31 / 24; 768 x 2 x 8000 58 / 73;
// 1464 x 7 x 528, 16 / 2 heads, 19 / 26; 512 x 1 x 60000 133 / 115; 16 / 2 of 256, int8: 512 x 4 x 1000 21 / 43; 512 x 8 x 300, 1000, 2000 19 / 28, 31 / 50, 47
// / 62; 800 x 8 36 / 29, 58 / 61, 88 / 80; 512 x 16 38 / 30, 59 / 65, 90 / 86; 512 x 1 x 16000 53 / 61, 768 95 / 72.
// Few rows are 16, 32, or, where the keys are that many, up to 48 a workgroup and 64 of heads of 128: codes are converted once for all of them. 32
// sequences of 8000 keys, 8 key heads of 128, us, 32 / 48 / 64 rows a workgroup: 32 rows 128 / 153 / 181, 48 226 / 156 / 183, 64 229 / 277 / 188; of 64:
// 48 rows 114 / 85 / 135, 64 105 / 131 / 125; one sequence of 2000 keys, 48 rows 13.4 / 15.7 / 17.7.  (More than 64: 6 sequences of 7301, 154 rows of
// drafted tokens, 8 / 4 heads of 128, 32 / 48 / 64 rows 39 / 62 / 57.)
// Heads of 256 have 16, and of drafted tokens 32 with four waves, which have the registers of two, where workgroups of 16 are more than 5/4 of the CUs:
// us, int8, 16 / 2 heads, 16 / 32 rows a workgroup: 8 sequences of 1000 keys, 256, 512, 800 rows 22 / 29, 40 / 31, 74 / 58; of 300 13 / 24, 25 / 19, 46 /
// 36; 16 of 2000, 256 58 / 47, of up to 2000 41 / 46; 8 / 4 heads, 304 rows, four of up to 1412, 304 workgroups, 24 / 29.
// Parts of the keys.  Few rows: as many as give every CU a workgroup, of two turns of its waves or more, and none where all keys are few turns
// (a second launch and the join cost 4 to 5 us, a turn 0.7 (heads of 64) to 2 us (256): 300 keys 8.1 us whole, 11.9 in two parts; 1060 keys of
// heads of 256 16 in five parts, 23 whole); and at most 4096 keys a part, so that a long sequence among short ones is not one workgroup's.
// Of drafted tokens 16 rows a workgroup where every such tile has a CU and they have no more than four turns of 256 keys a CU (eight of heads of 64):
// us, two tiles a workgroup / one, 64 / 8 heads of 128: 6 tokens over 300 keys 10.8 / 8.4, 1000 14.2 / 11.6, 4000 16.1 / 13.6, 16000 21.6 / 22.2; 4 x 8
// over 1000 17.5 / 15.7, over 4000 22.8 / 24.0; 16 x 3 over 1000 20.1 / 13.9; 16 x 6 over 300, 384 tiles, 11.2 / 15.0; of 64, 6 over 300 7.5 / 5.9,
// 8 x 8 over 2000 15.5 / 12.2, 4000 21.7 / 20.7, 32 over 6000 17.9 / 19.9.  And parts are down to one turn
// of the workgroup's waves, as many as one workgroup a CU leaves; whole up to 1024 keys of heads of 64, 768 of 128, 512 of 256 (256 with 32 rows a workgroup,
// whose turn is 128). us, whole / parts of 256, 512 keys, 64 / 8 heads of 128: 1 token over 600, 1000, 2000 keys 9.6 / 10.5, 12.2 / 10.7, 17.6 / 10.7; 4 x 6
// tokens over 1000, 2000 15.8 / 16.3, 21.4 / 26.8 / 17.9 (two groups of rows: 512 workgroups); 6 over 5000 39 / 25.4 / 16.8; of 64, 4 x 6 over 1000 10.9 /
// 13.1; 16 / 2 of 256, 2 over 600 14.8 / 14.3.
// Of drafted tokens, where workgroups are more than CUs they are of the longer sequences first, so that the last to start are short ones; each finds its
// sequence with the loads that it makes anyway.  us, as sequences come / longer first, E4M3, of any length up to the longest (of which most are short): 40 of
// 4001 keys and 63 tokens, 16 / 16 heads of 64, 68 / 57 (50 / 38); 64 of 3000 and 8, 32 / 8 of 128, 53 / 44 (42 / 31); 48 of 2000 and 16, 16 / 16, 49 / 45
// (35 / 32); 200 of 3000 and 4, 32 / 4, 86 / 82 (57 / 46); all of the longest length 42 to 153, the same.  (In parts of 1024 keys and joined, so that the
// longest is several workgroups': 92, 71, 59 and 124; empty workgroups and the join take more than it gives.)
// Many rows: in equal stretches (Cuts) where that is less than a tile of rows' keys by more than the second start and the join cost (800 keys of
// heads of 128, 1600 of 64, 400 of 256); several sequences, whose lengths the host does not know, count as half of the longest.  us, whole / cut, 32 / 8 heads of 128:
//   128 tokens over 700, 1024, 1500 keys 30 / 35, 38 / 37, 52 / 39; 512 over 700, 1024, 1500, 2500, 16384 30 / 38, 38 / 42, 52 / 47, 78 / 55, 441 / 174;
//   1024 over 1500, 2500 53 / 54, 80 / 71; 421, 376 and 512 over 6104, 4383 and 512 170 / 109; 3 x 512 over 6000 181 / 186; 4 x 256 over 1024, 512,
//   341 and 146 39 / 43, over four times as many 117 / 70; 200, 512, 30 and 400 over 9000, 1200, 400 and 16000 440 / 213; 2 x 1024 over 8192 268 / 296;
//   4 / 1 heads, 47, 114 and 166 over 8642 234 / 39; heads of 64, 4 x 100 over 1024, 2000 33 / 43, 56 / 49; 8 / 2 of 256, 512 over 512, 700, 1024
//   35 / 37, 43 / 38, 55 / 43; 128 over 400, 512, 700 32 / 35, 34 / 35, 42 / 37; 4 x 100 over 512, 1024 36 / 39, 56 / 42.  (The same number of parts for every sequence instead, the best for each call: of these 512 over
//   16384 163, the three of 6104 106, the four of 16000 204; but what the host knows did not tell which number, by a factor of up to 1.7.)
// Parts have room for a sequence that is the only long one, within PART_ROOM: of few rows fewer and longer ones where that is less, of many rows as
// many as the mean tile of rows needs even so (271 MB at most, over three million sizes: rows that fill the card are not cut).
constexpr long PART_ROOM = 256L << 20;  // bytes
struct AttentionPlan {
    enum { GENERIC, FEW, MANY } kernel;
    int splits, chunk, row_tiles, tile_rows;
    int longest;
};
static AttentionPlan plan_attention(const ptoamd_kv8_cache* c, int heads, int tokens, int max_tokens, int max_length, int window, bool tree)
{
    AttentionPlan p{AttentionPlan::GENERIC, 1, 0, 0, 0, false};
    const int dim = built_head(c->head_dim);
    if (dim == 0)
        return p;
    if (max_tokens > tokens)  // (a loose bound)
        max_tokens = tokens;
    const long rows = (long)max_tokens * (heads / c->kv_heads);
    long keys = (long)c->max_pages * c->page_size;
    if (max_length > 0 && max_length < keys)
        keys = max_length;
    if (window > 0 && (long)window + max_tokens + 31 < keys)
        keys = (long)window + max_tokens + 31;
    const long cus = device_compute_units();
    const long items = (long)c->sequences * c->kv_heads;
    const long room = PART_ROOM / ((long)tokens * heads * (dim * 4 + 8));  // parts
    const bool busy = items * keys * dim > 65536 * cus;
    p.kernel = rows <= (!busy ? 96 : dim == 256 ? 32 : 64) ? AttentionPlan::FEW : AttentionPlan::MANY;
    long groups = 0;
    if (tree) {
        // (sequences with fewer tokens than the most have fewer workgroups: those of all tokens, and half a one for what each sequence leaves in its last)
        const long each = dim == 256 ? 16 : 32, turns = (keys + 255) / 256, at_most = items * ((rows + each - 1) / each);
        const long by_tokens = (long)tokens * heads / each + items / 2;
        groups = by_tokens < at_most ? by_tokens : at_most;
        const bool fits = groups <= (turns < 3 ? (dim == 128 ? 1 : 2) : dim == 64 ? 3 : dim == 128 ? 2 : 4) * cus && groups * turns <= (dim == 64 ? 32 : 18) * cus;
        p.kernel = rows <= (dim == 256 ? 32 : 64) || fits ? AttentionPlan::FEW : AttentionPlan::MANY;
    }
    if (p.kernel == AttentionPlan::FEW) {
        p.row_tiles = rows <= 16 || dim == 256 ? 1 : rows <= 32 || !busy || rows > 64 ? 2 : rows <= 48 ? 3 : dim == 128 ? 4 : 2;
        if (tree) {
            const long alone = items * ((rows + 15) / 16);
            if (alone <= cus && alone * ((keys + 255) / 256) <= (dim == 64 ? 8 : 4) * cus)
                p.row_tiles = 1;
            if (dim == 256 && rows > 16 && 4 * groups > 5 * cus)
                p.row_tiles = 2;
        }
        const long step = 32 * few_waves(dim, p.row_tiles, tree);  // the keys that a workgroup's waves have at a time
        const long turns = (keys + step - 1) / step;
        long splits = (cus + items - 1) / items;
        splits = splits < turns / 2 ? splits : turns / 2;
        if (turns <= (dim == 256 ? 4 : 6))
            splits = 1;
        if (tree) {
            const long all = items * ((rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles));
            splits = all < cus ? cus / all : 1;
            p.longest = c->sequences > 1 && all > cus ? (int)keys : 0;
            splits = splits < turns ? splits : turns;
            if (turns <= (dim == 64 ? 4 : dim == 128 ? 3 : 2))
                splits = 1;
        }
        const long even = (keys + 4095) / 4096;
        splits = splits > even ? splits : even;
        const long most = room < 65535 ? room : 65535;  // (parts are a grid's slowest index)
        splits = splits < most ? splits : most;
        if (splits > 1) {
            p.chunk = (int)(((keys + splits - 1) / splits + step - 1) / step * step);
            p.splits = (int)((keys + p.chunk - 1) / p.chunk);
        }
        return p;
    }
    p.tile_rows = many_rows(dim);
    if (tree && rows <= 128)
        p.tile_rows = 128;
    p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    const long tiles = p.row_tiles * items;  // of rows, a workgroup's each if no keys are cut
    const bool countable = (long)p.row_tiles * c->sequences <= Cuts::MOST && (double)tiles * c->max_pages * c->page_size < 1e9;
    const double full = (double)tiles / cus / (c->sequences > 1 ? 2 : 1);
    if (countable && keys * (1 - full) > 448 * full + 102400.0 / dim) {
        // (a tile's parts: its keys, at most twice the mean of one sequence's, in stretches of the mean; of several up to all stretches of a key head)
        const long mean = 2 * cus / tiles + 3, most = c->sequences > 1 ? cus / c->kv_heads + 2 : mean;
        const long parts = most < room ? most : room;
        p.splits = (int)(parts > mean ? parts : mean);
    }
    return p;
}
static size_t part_bytes(const AttentionPlan& p, int heads, int tokens, int head_dim)
{
    if (p.splits <= 1)
        return 0;
    return (p.kernel == AttentionPlan::MANY ? Cuts::BYTES : 0) + (size_t)p.splits * tokens * heads * (head_dim * sizeof(float) + sizeof(float2));
}

int prepare_attention_kernels()
{
    for (int code : {PTOAMD_I8, PTOAMD_E4M3})
        for (bool f16 : {false, true})
            for (int dim : {64, 128, 256})
                for (int tiles : {1, 2, 3, 4}) {
                    if (tiles > (dim == 64 ? 3 : dim == 128 ? 4 : 2))
                        continue;
                    AttentionArgs a{};  // (of no heads: nothing is launched)
                    a.cache.head_dim = dim;
                    a.row_tiles = tiles;
                    a.tile_rows = tiles == 1 ? 128 : 256;  // (of drafted tokens: both)
                    int rc = dim == 256 && tiles > 1 ? PTOAMD_OK : launch_attention_few(a, code, f16, 1, nullptr);
                    if (rc == PTOAMD_OK)
                        rc = launch_attention_many(a, code, f16, 1, nullptr);
                    if (rc == PTOAMD_OK)
                        rc = launch_attention_tree_few(a, code, f16, 1, nullptr);
                    if (rc == PTOAMD_OK)
                        rc = launch_attention_tree_many(a, code, f16, 1, nullptr);
                    if (rc != PTOAMD_OK)
                        return rc;
                }
    return PTOAMD_OK;
}

static size_t workspace_bytes_of(const ptoamd_kv8_cache* cache, int heads, int tokens, int max_tokens, int max_length, int window, bool tree)
{
    if (cache == nullptr || cache->kv_heads <= 0 || heads <= 0 || heads % cache->kv_heads != 0 || tokens <= 0 || max_tokens <= 0 || cache->sequences <= 0 ||
        cache->max_pages <= 0 || cache->page_size <= 0)
        return 0;
    return part_bytes(plan_attention(cache, heads, tokens, max_tokens, max_length, window, tree), heads, tokens, built_head(cache->head_dim));
}

// The call of both entry points: `causal`, or `tree` with rows of tree_words 64-bit words.
static int attention(const char* what, void* out, float* lse, const ptoamd_kv8_cache* cache, const uint64_t* tree, int tree_words, const void* q, int type,
                     int heads, int tokens, const int32_t* cu_tokens, int max_tokens, int max_length, int64_t q_token_stride, int64_t q_head_stride,
                     int64_t out_token_stride, int64_t out_head_stride, float scale, int causal, int window, void* workspace, size_t workspace_bytes,
                     void* stream)
{
    AttentionArgs a{};
    const int checked = kv8_from(what, cache, tokens, cu_tokens, max_tokens, &a.cache);
    if (checked != PTOAMD_OK)
        return checked;
    TraceScope trace(tree != nullptr ? "ATTENTION_KV8_TREE" : "ATTENTION_KV8", "mix", tokens, heads, cache->head_dim);
    trace.in(q, tokens, (long)heads * cache->head_dim, "ND", type)
        .in(cache->k, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type)
        .in(cache->v, cache->pages, (long)cache->kv_heads * cache->page_size * cache->head_dim, "ND", cache->code_type)
        .out(out, tokens, (long)heads * cache->head_dim, "ND", type).out(lse, tokens, heads, "ND", PTOAMD_F32);
    PTOAMD_REQUIRE(type == PTOAMD_F16 || type == PTOAMD_BF16, PTOAMD_E_UNSUPPORTED, "%s: queries must be f16 or bf16", what);
    PTOAMD_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads <= 65535, PTOAMD_E_INVALID,
                   "%s: heads must be a positive multiple of kv_heads, at most 65535 (%d, %d)", what, heads, cache->kv_heads);
    PTOAMD_REQUIRE(cache->head_dim % 8 == 0 && cache->head_dim <= 512, PTOAMD_E_UNSUPPORTED,
                   "%s: head_dim must be a multiple of 8 and at most 512 (%d)", what, cache->head_dim);
    PTOAMD_REQUIRE(scale > 0 && isfinite(scale), PTOAMD_E_INVALID, "%s: scale must be positive and finite", what);
    PTOAMD_REQUIRE(window >= 0 && max_length >= 0, PTOAMD_E_INVALID, "%s: window and max_length must not be negative (%d, %d)", what, window, max_length);
    if (tokens == 0 || max_tokens == 0)
        return PTOAMD_OK;
    PTOAMD_REQUIRE((long)a.cache.max_tokens * (heads / cache->kv_heads) <= 0x7FFF0000L, PTOAMD_E_UNSUPPORTED,
                   "%s: %d tokens of %d heads a key head are too many rows", what, a.cache.max_tokens, heads / cache->kv_heads);
    PTOAMD_REQUIRE(out && q, PTOAMD_E_INVALID, "%s: null operand", what);
    PTOAMD_REQUIRE((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q)) % 2 == 0 && reinterpret_cast<uintptr_t>(lse) % 4 == 0, PTOAMD_E_ALIGNMENT,
                   "%s: q, out and lse must be aligned to their elements", what);
    if (tree != nullptr) {  // (workgroups write results while others still read their rows of bits)
        const HeadRows bits = memory_at(tree, (int64_t)tokens * tree_words * 8);
        PTOAMD_REQUIRE(!meet(bits, HeadRows{(uint64_t)(uintptr_t)out, tokens, heads, out_token_stride * 2, out_head_stride * 2, cache->head_dim * 2L}) &&
                           !meet(bits, memory_at(lse, (int64_t)tokens * heads * 4)),
                       PTOAMD_E_INVALID, "%s: out and lse must not overlap the tree", what);
    }
    a.q = static_cast<const uint8_t*>(q);
    a.out = static_cast<uint8_t*>(out);
    a.lse = lse;
    a.q_token = q_token_stride * 2;
    a.q_head = q_head_stride * 2;
    a.out_token = out_token_stride * 2;
    a.out_head = out_head_stride * 2;
    a.heads = heads;
    a.group = heads / cache->kv_heads;
    a.causal = causal != 0;
    a.window = window;
    a.scale = scale;
    a.tree = reinterpret_cast<const uint32_t*>(tree);
    a.tree_words = 2 * tree_words;
    hipStream_t s = as_stream(stream);
    const bool i8 = cache->code_type == PTOAMD_I8, f16 = type == PTOAMD_F16;
    const AttentionPlan plan = plan_attention(cache, heads, tokens, max_tokens, max_length, window, tree != nullptr);
    const size_t need = part_bytes(plan, heads, tokens, built_head(cache->head_dim));
    PTOAMD_REQUIRE(workspace == nullptr || workspace_bytes >= need, PTOAMD_E_INVALID, "%s: a workspace of %zu bytes is needed (%zu)", what, need, workspace_bytes);
    PTOAMD_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, PTOAMD_E_ALIGNMENT, "%s: the workspace must be 16-byte aligned", what);
    const uint64_t cache_bits = (uint64_t)(uintptr_t)cache->k | (uint64_t)(uintptr_t)cache->v | (uint64_t)cache->k_page_stride | (uint64_t)cache->k_head_stride |
                                (uint64_t)cache->k_token_stride | (uint64_t)cache->v_page_stride | (uint64_t)cache->v_head_stride | (uint64_t)cache->v_token_stride;
    // (what the kernels hold in 32 bits: strides of pages in units of 8 bytes, of the tokens of a page in bytes, places of scales)
    const bool addressable = cache->k_page_stride >= 0 && cache->k_page_stride < 1LL << 34 && cache->v_page_stride >= 0 && cache->v_page_stride < 1LL << 34 &&
                             cache->k_token_stride >= 0 && cache->k_token_stride < 1 << 22 && cache->v_token_stride >= 0 && cache->v_token_stride < 1 << 22 &&
                             (long)cache->pages * cache->kv_heads < 1L << 30;
    if (plan.kernel != AttentionPlan::GENERIC && cache_bits % 16 == 0 && addressable && !options().force_generic) {
        a.wide = ((uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)out | (uint64_t)a.q_token | (uint64_t)a.q_head | (uint64_t)a.out_token | (uint64_t)a.out_head) % 16 == 0;
        a.splits = workspace != nullptr ? plan.splits : 1;
        a.chunk = plan.chunk;
        a.row_tiles = plan.row_tiles;
        a.tile_rows = plan.tile_rows;
        a.sequences = cache->sequences;
        a.longest = plan.longest;
        a.cuts = plan.kernel == AttentionPlan::MANY && a.splits > 1 ? static_cast<int*>(workspace) : nullptr;
        a.part_out = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (a.cuts != nullptr ? Cuts::BYTES : 0));
        a.part_sum = reinterpret_cast<float2*>(a.part_out + (size_t)plan.splits * tokens * heads * built_head(cache->head_dim));
        const bool few = plan.kernel == AttentionPlan::FEW;
        const auto launch = tree != nullptr ? (few ? launch_attention_tree_few : launch_attention_tree_many) : (few ? launch_attention_few : launch_attention_many);
        const int rc = launch(a, cache->code_type, f16, cache->sequences, s);
        if (rc != PTOAMD_OK)
            return rc;
        set_last_kernel(few ? (a.splits > 1 ? "attention_kv8_few_split" : "attention_kv8_few") : (a.splits > 1 ? "attention_kv8_many_split" : "attention_kv8_many"));
        return a.splits > 1 ? launch_attention_join(a, f16, cache->sequences, s) : PTOAMD_OK;
    }
    if (type == PTOAMD_F16)
        return i8 ? launch_generic<_Float16, PTOAMD_I8>(a, cache->sequences, s) : launch_generic<_Float16, PTOAMD_E4M3>(a, cache->sequences, s);
    return i8 ? launch_generic<__bf16, PTOAMD_I8>(a, cache->sequences, s) : launch_generic<__bf16, PTOAMD_E4M3>(a, cache->sequences, s);
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

size_t ptoamd_attention_kv8_workspace_bytes(const ptoamd_kv8_cache* cache, int heads, int tokens, int max_tokens, int max_length, int window)
{
    return workspace_bytes_of(cache, heads, tokens, max_tokens, max_length, window, false);
}

int ptoamd_attention_kv8(void* out, float* lse, const ptoamd_kv8_cache* cache, const void* q, int type, int heads, int tokens,
                         const int32_t* cu_tokens, int max_tokens, int max_length, int64_t q_token_stride, int64_t q_head_stride,
                         int64_t out_token_stride, int64_t out_head_stride, float scale, int causal, int window, void* workspace,
                         size_t workspace_bytes, void* stream)
{
    return attention("ptoamd_attention_kv8", out, lse, cache, nullptr, 0, q, type, heads, tokens, cu_tokens, max_tokens, max_length, q_token_stride, q_head_stride,
                     out_token_stride, out_head_stride, scale, causal, window, workspace, workspace_bytes, stream);
}

size_t ptoamd_attention_kv8_tree_workspace_bytes(const ptoamd_kv8_cache* cache, int heads, int tokens, int max_tokens, int max_length, int window)
{
    return workspace_bytes_of(cache, heads, tokens, max_tokens, max_length, window, true);
}

int ptoamd_attention_kv8_tree(void* out, float* lse, const ptoamd_kv8_cache* cache, const uint64_t* tree, int tree_words, const void* q, int type,
                              int heads, int tokens, const int32_t* cu_tokens, int max_tokens, int max_length, int64_t q_token_stride,
                              int64_t q_head_stride, int64_t out_token_stride, int64_t out_head_stride, float scale, int window, void* workspace,
                              size_t workspace_bytes, void* stream)
{
    const char* what = "ptoamd_attention_kv8_tree";
    const int most = max_tokens < tokens ? max_tokens : tokens;  // (a loose bound)
    if (most > 0) {
        PTOAMD_REQUIRE(tree != nullptr, PTOAMD_E_INVALID, "%s: null operand", what);
        PTOAMD_REQUIRE(reinterpret_cast<uintptr_t>(tree) % 8 == 0, PTOAMD_E_ALIGNMENT, "%s: the tree must be aligned to its words", what);
        PTOAMD_REQUIRE(most <= PTOAMD_MOST_DRAFTED, PTOAMD_E_UNSUPPORTED, "%s: at most %d tokens of a sequence are drafted (%d)", what, PTOAMD_MOST_DRAFTED, most);
        PTOAMD_REQUIRE(tree_words > 0 && tree_words <= PTOAMD_MOST_DRAFTED / 64 && 64 * tree_words >= most, PTOAMD_E_INVALID,
                       "%s: rows of %d words for %d tokens: one for every 64 is needed, at most %d", what, tree_words, most, PTOAMD_MOST_DRAFTED / 64);
        PTOAMD_REQUIRE(window <= 0 || window >= most, PTOAMD_E_UNSUPPORTED, "%s: a window of %d does not hold the %d tokens that may be drafted", what, window, most);
    }
    return attention(what, out, lse, cache, tree, tree_words, q, type, heads, tokens, cu_tokens, max_tokens, max_length, q_token_stride, q_head_stride,
                     out_token_stride, out_head_stride, scale, 1, window, workspace, workspace_bytes, stream);
}

}  // extern "C"
