// Attention over an 8-bit cache for many queries: prompts and chunks of prompts, large drafted trees.
#pragma once
#include "attention_kv8.hpp"

namespace ptoamd {

// A workgroup has 32 rows a wave of one sequence and key head (rows: new tokens times the query heads that share the key head, token-major,
// so those heads share what is staged) and walks the keys that its rows see in tiles of 64.  A tile's codes are read while the tile before
// is computed, become f16, exactly, once for all waves, and go to LDS in one of two buffers.
//   S^T = K q^T (32x32x16): a fragment is 8 elements of one key, q's fragments stay in registers.
//   o^T = V^T p^T : a lane has the scores of keys 8 (i / 4) + 4 (lane / 32) + i % 4 of 32 for its row; with eight of them as its share of a
//                 product's 16 keys the weights are the fragment as they stand, and V's fragment (the same keys of one element) comes from
//                 two transposing LDS reads of four keys each.
// Scores, references and sums are f32; a page's value scale goes into the weight (ValueScale).
// Bound: the matrix and the vector unit by turns.  A tile of 64 keys of heads of 128 takes a SIMD and its two waves 2048 clocks of products and some
// 2900 of vector instructions (an exponential of a score takes 16), which overlap to 4160.  A prompt of 8192 tokens, 32 / 8 heads of 128, E4M3: 550
// to 580 us with the card's clock, 950 to 1000 TFLOP/s (a bf16 product of 8192 x 8192 x 8192: 1407).  On the way there: both waves
// of a SIMD in step 666 us, one a segment behind 606, fragments and staging in a fixed order between the products 574, NaN kept out of the sum where
// scales are staged instead of at every sum 550.  The card clocks it at 2.05 GHz (of 2.4): looking for the largest score only where a weight
// overflows spares a sixth of a score's vector instructions and no time; table entries asked for later in a turn cost 1%.
template <int D>
struct ManyTile {
    static constexpr int KEYS = MANY_KEYS;
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

// The tiles of keys that there are and a workgroup's stretch of them: long enough that a tile of rows has at most splits parts, and 256 keys at
// least (with 1024, three sequences of 8642 keys with one key head took 52 us instead of 39).
template <int D, int WAVES, int ROWS, bool TREE>
__device__ __forceinline__ void count_tiles(const AttentionArgs& a, int tiles, int* cuts)
{
    constexpr int KEYS = MANY_KEYS, LEAST = 256 / KEYS, START = many_start(D, ROWS);
    static_assert(64 * WAVES >= Cuts::MOST, "a thread counts a tile of rows");
    __shared__ int wave_sum[WAVES], wave_most[WAVES];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    int own = 0;
    if (tid < tiles) {
        const int seq = tid / a.row_tiles, row0 = (tid - seq * a.row_tiles) * ROWS;
        const Span span = span_of(a, seq);
        const int rows = span.count * a.group;
        if (row0 < rows) {  // (rows that see no key have a tile too: zeros are written there)
            const int2 any = keys_of_any<TREE>(a, span, row0 / a.group, (min(row0 + ROWS, rows) - 1) / a.group);
            const int from = any.x & ~31, to = any.y;
            own = max((to - from + KEYS - 1) / KEYS, 1) + START;
        }
    }
    int sum = own, most = own;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        const int below = __shfl_up(sum, i);
        sum += lane >= i ? below : 0;
        most = max(most, __shfl_xor(most, i));
    }
    if (lane == 63) {
        wave_sum[wave] = sum;
        wave_most[wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Cuts::MOST / 64; ++w) {
        sum += w < wave ? wave_sum[w] : 0;
        most = max(most, wave_most[w]);
    }
    if (tid < Cuts::MOST)
        cuts[Cuts::FIRST + tid + 1] = sum;
    if (tid == 0)
        cuts[Cuts::FIRST] = 0;
    if (tid == Cuts::MOST - 1) {
        const int units = sum * a.cache.kv_heads, groups = gridDim.x;
        cuts[Cuts::HEAD] = sum;
        cuts[Cuts::STRETCH] = max(max((units + groups - 1) / groups, (most + a.splits - 2) / (a.splits - 1)), LEAST);
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = tid; i < Cuts::SIZE; i += 64 * WAVES)
            a.cuts[i] = cuts[i];
}

// Heads of 256: the sums are in accumulator registers, which only the matrix instructions read.  Left to itself the compiler moves all 128 of them out
// and back in every tile, for the multiplication that few tiles have: 1016 us instead of 815, 8192 tokens of 16 / 4 heads, int8;
// with the registers that this leaves, tiles of 64 keys instead of 32: 753.
// The compiler does not see the waits that a product's result needs before it is read (some twenty clocks) and a written one before a product takes it: the
// score products, some thousand clocks, lie between the sums' last product and this, the exponentials and a barrier between this and their next.
__device__ __forceinline__ float scaled_accumulator(float x, float by)
{
    float t;
    asm("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1" : "+a"(x), "=&v"(t) : "v"(by));
    return x;
}

// TREE: of drafted tokens, whose rows of bits lie in LDS for the tiles of the step's own keys.
// HALVES: half as many rows a workgroup, 128, and two tiles of keys at a time: the waves of a SIMD have the same rows, one those of every second tile, and
// add up at the end.  So rows up to 128 leave no wave without work; each half stages its tiles alone, twice a wave's share.
// Bound: as above, and the staging.  16 sequences of 16 tokens over 8192 keys, 64 / 8 heads of 128, E4M3, 104 us (112 where no cache holds them): the matrix unit is
// busy for 28 % of the clocks, the vector unit for 38 %; with all pages in the L2 95.  Fragments read four products ahead instead of two changed nothing.
constexpr int MANY_TREE_WORDS = PTOAMD_MOST_DRAFTED / 32;
template <typename T, int CODE, int D, int WAVES, bool TREE, bool HALVES>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(WAVES / 4, WAVES / 4))) attention_kv8_many_kernel(AttentionArgs args)
{
    typedef ManyTile<D> Tile;
    constexpr int ROWS = 32 * WAVES / (HALVES ? 2 : 1), START = many_start(D, ROWS);
    constexpr int GROUP = HALVES ? WAVES / 2 : WAVES;  // the waves that share a tile of keys
    constexpr int THREADS = 64 * GROUP, KEYS = Tile::KEYS, STRIDE = HALVES ? 2 * KEYS : KEYS, STEPS = D / 16, DT = D / 32;
    constexpr int SIDE_UNITS = KEYS * D / 16, UNITS = 2 * SIDE_UNITS / THREADS;  // 16 codes each; a thread's
    extern __shared__ __attribute__((aligned(16))) uint8_t all_tiles[];  // two of keys, two of values (HALVES: of each)
    __shared__ float4 all_scales[HALVES ? 2 : 1][2][KEYS / 16];  // of 16 keys: key scale, value scale's log2 and inverse
    __shared__ int cuts[Cuts::SIZE];
    __shared__ uint32_t drafted[TREE ? ROWS : 1][MANY_TREE_WORDS + 1];  // (rows a bank apart)
    // A workgroup has one tile of rows and all their keys, or a stretch of what there is (Cuts): the end of a tile's keys, whole ones, the start of
    // another's.  Stretches go to the XCDs in eighths, so that neighbours, which share keys, share an L2.
    const int turn = gridDim.x % 8 == 0 ? (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8) : (int)blockIdx.x;
    int unit = 0, unit_end = 0;
    if (args.splits > 1) {
        count_tiles<D, WAVES, ROWS, TREE>(args, args.row_tiles * args.sequences, cuts);
        unit = turn * cuts[Cuts::STRETCH];
        unit_end = min(unit + cuts[Cuts::STRETCH], cuts[Cuts::HEAD] * args.cache.kv_heads);
        unit = __builtin_amdgcn_readfirstlane(unit), unit_end = __builtin_amdgcn_readfirstlane(unit_end);
        if (unit >= unit_end)
            return;
    }
    do {
        const ArgumentsAgain again;  // (for each tile of rows anew: what only its start needs is not kept through the loop)
        int tid = threadIdx.x;
        asm("" : "+v"(tid));
        const int half = HALVES ? __builtin_amdgcn_readfirstlane(tid / THREADS) : 0;
        if constexpr (HALVES)
            tid %= THREADS;
        const int lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), col = lane % 32, hf = lane / 32;  // (HALVES: among its half's)
        uint8_t* tiles = all_tiles + half * 4 * Tile::BYTES;
        auto& scales = all_scales[half];
        const AttentionArgs& a = *again.all();
        const Kv8& c = a.cache;
        int kv_head, row_tile, seq, skip = 0, part = -1, most = 1 << 30;
        if (a.splits > 1) {
            const int head_tiles = __builtin_amdgcn_readfirstlane(cuts[Cuts::HEAD]), stretch = __builtin_amdgcn_readfirstlane(cuts[Cuts::STRETCH]);
            kv_head = unit / head_tiles;
            const int rest = unit - kv_head * head_tiles;
            int tile = -1;  // the last that starts at or before it (those without rows have no tiles of keys)
#pragma unroll
            for (int i = 0; i < Cuts::MOST; i += 64)
                tile += __popcll(__ballot(cuts[Cuts::FIRST + i + lane] <= rest));
            const int first = __builtin_amdgcn_readfirstlane(cuts[Cuts::FIRST + tile]), next = __builtin_amdgcn_readfirstlane(cuts[Cuts::FIRST + tile + 1]);
            seq = tile / a.row_tiles;
            row_tile = tile - seq * a.row_tiles;
            const int until = min(next - rest, unit_end - unit) + rest - first - START;
            skip = max(rest - first - START, 0);
            most = until - skip;
            unit += next - rest;
            if (until <= 0)
                continue;  // (the stretch ends before the first of its keys)
            if (most < next - first - START)
                part = turn - (kv_head * head_tiles + first + START) / stretch;
        } else {
            const int row_tiles = gridDim.x / c.kv_heads;
            kv_head = blockIdx.x % c.kv_heads;
            row_tile = row_tiles - 1 - blockIdx.x / c.kv_heads;  // (those with most keys first)
            seq = blockIdx.y;
        }
        const Span span = span_of(a, seq);
        const int rows = span.count * a.group, row0 = row_tile * ROWS;
        if (row0 >= rows)
            return;
        // the keys that any row of the workgroup sees, and of the part
        const int place0 = span.length - span.count;
        const int2 any = keys_of_any<TREE>(a, span, row0 / a.group, (min(row0 + ROWS, rows) - 1) / a.group);
        const int from = any.x, to = any.y;
        const int begin = (from & ~31) + skip * KEYS, end = most < (to - begin + KEYS - 1) / KEYS ? begin + most * KEYS : to;

        const int row = row0 + 32 * wave + col, token = row / a.group;
        const bool valid = row < rows;
        const int head = kv_head * a.group + (valid ? row - token * a.group : 0);
        // The queries, the TREE's rows of bits and, behind them, the first tile's codes are asked for before any of them is waited for.
        constexpr int ROW_WORDS = 32 * MANY_TREE_WORDS / 64;
        uint32_t words[ROW_WORDS];  // (of a wave's own rows)
        if constexpr (TREE)
#pragma unroll
            for (int i = 0; i < ROW_WORDS; ++i) {
                const int its = row0 + 32 * wave + (lane + 64 * i) / MANY_TREE_WORDS, word = lane % MANY_TREE_WORDS;
                words[i] = a.tree[(int64_t)(span.first + (its < rows ? its / a.group : 0)) * a.tree_words + (word < a.tree_words ? word : 0)];
            }
        uint4 q[STEPS];
        {
            const uint8_t* p = a.q + (int64_t)(span.first + (valid ? token : 0)) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
            for (int st = 0; st < STEPS; ++st)
                q[st] = valid && 16 * st < c.head_dim ? load_row8(p + 2 * (16 * st + 8 * hf), a.wide) : make_uint4(0, 0, 0, 0);
        }
        int2 seen = make_int2(0, 0);  // (TREE: x, the first of the older keys)
        float cq = 0.0f, bias = 0.0f;
        // where a row's scores start: without the 128 that the keys' int8 codes carry.  (TREE: taken off where scores are scaled, in one register for 16)
        f32x16 start = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        auto take_queries = [&]() __attribute__((always_inline)) {
            if constexpr (TREE) {
#pragma unroll
                for (int i = 0; i < ROW_WORDS; ++i) {
                    const int its = 32 * wave + (lane + 64 * i) / MANY_TREE_WORDS, word = lane % MANY_TREE_WORDS;
                    drafted[its][word] = row0 + its < rows && word < a.tree_words ? own_bits(words[i], word, span.count) : 0u;
                }
                seen.x = first_of_drafted(a, span, drafted[32 * wave + col], MANY_TREE_WORDS, valid, token);
            } else {
                seen = valid ? visible_keys(a, place0 + token, span.length) : make_int2(0, 0);
            }
            uint32_t largest = largest_of<STEPS>(q);
            largest = max(largest, (uint32_t)__shfl_xor((int)largest, 32));
            const RowScale r = row_scale<T>(largest);
            cq = r.up * (a.scale * 1.44269504088896341f) * KV8_UNIT<CODE>;
            scale_to_f16<T, STEPS>(q, r.down);
            if (CODE == PTOAMD_I8) {
                const uint4 unbias = make_uint4(UNBIAS, UNBIAS, UNBIAS, UNBIAS);
#pragma unroll
                for (int st = 0; st < STEPS; ++st)
                    start = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, unbias), __builtin_bit_cast(f16x8, q[st]), start, 0, 0, 0);
            }
            bias = start[0];  // (all keys')
            if constexpr (TREE)
                start = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        };
        // the keys that every row of the wave sees
        const int wave_row = row0 + 32 * wave;
        const int2 every = keys_of_every<TREE>(a, span, min(wave_row, rows - 1) / a.group, (min(wave_row + 32, rows) - 1) / a.group);
        const int every_from = every.x, every_to = every.y;

        // What a thread stages: units of 16 codes; a unit's side, key and 16 elements are the same for every tile.  A wave's units of a kind are keys of
        // one group of 16, so of one page: its id, scale and address are the scalar unit's work.  Values go one tile behind the keys, as they are used:
        // stage i is the keys of tile i and the values of tile i - 1.
        const int own_begin = begin + half * KEYS;  // (tile i of its own starts at own_begin + i STRIDE)
        const int last_key = max(span.length - 1, 0), slot_mask = (1 << c.page_shift) - 1;
        const int32_t* table = c.table + (int64_t)seq * c.max_pages;
        int ids[UNITS], scale_id = 0;
        uint4 raw[UNITS];
        float2 raw_scale = make_float2(0, 0);
        float unit_scale[UNITS];  // of values: the scale of their page
        uint32_t no_page = 0;     // bit u: the table names no page for unit u (asked of E4M3 codes, which may be NaN; no int8 code is)
        uint32_t source[UNITS], none = 0;
        asm("" : "+v"(none));  // (a vector register's zero: a scale that is not read through the scalar cache, for which a barrier would wait)
        static_assert(SIDE_UNITS % THREADS == 0 || THREADS == 2 * SIDE_UNITS, "a unit is keys or values for all waves, or for half of them");
        auto is_value = [&](int u) { return SIDE_UNITS < THREADS ? wave >= GROUP / 2 : u * THREADS >= SIDE_UNITS; };
        const int wave_key = wave % (SIDE_UNITS < THREADS ? GROUP / 2 : GROUP) * (1024 / D);
        auto unit_key = [&](int u, int stage) { return own_begin + (stage - (is_value(u) ? 1 : 0)) * STRIDE + u * THREADS % SIDE_UNITS / (D / 16) + wave_key; };
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            source[u] = (uint32_t)(lane / (D / 16)) * (uint32_t)(is_value(u) ? c.v.token : c.k.token) + (lane % (D / 16) * 16 < c.head_dim ? lane % (D / 16) * 16 : 0);
        }
        // Where a unit's two halves go in a tile: of keys or values, its first unit's places (a side's units are multiples of 16 keys apart), the second half
        // 16 bytes from the first in either direction.
        static_assert(SIDE_UNITS <= THREADS || THREADS / (D / 16) % 16 == 0, "a unit's permutation is its side's");
        const int own_key = tid % SIDE_UNITS / (D / 16), own_chunk = lane % (D / 16) * 2;
        const int key_target = Tile::key_at(own_key, own_chunk), value_target = Tile::value_at(own_key, own_chunk / 2);
        auto find = [&](int stage) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                ids[u] = load_uniform(table + (min(max(unit_key(u, stage), 0), last_key) >> c.page_shift));
        };
        auto fetch = [&](int u, int stage) __attribute__((always_inline)) {
            const Kv8Side& side = is_value(u) ? c.v : c.k;
            const bool known = (unsigned)ids[u] < (unsigned)c.pages;
            const uint32_t page = known ? ids[u] : 0, slot = unit_key(u, stage) & slot_mask;
            if (CODE != PTOAMD_I8)
                no_page = known ? no_page & ~(1u << u) : no_page | 1u << u;
            const uint8_t* at = side.codes + ((uint64_t)page * (uint32_t)(side.page >> 3) * 8 + kv_head * side.head + slot * (uint32_t)side.token);
            raw[u] = *reinterpret_cast<const uint4*>(at + source[u]);
            unit_scale[u] = side.scales[page * (uint32_t)c.kv_heads + kv_head + none];
        };
        // the seven pieces of a unit's way from codes to LDS, and the eighth that reads the next one
        constexpr int PIECES = 8;
        uint32_t staged[4];
        auto piece = [&](auto u_, auto piece_, int stage) __attribute__((always_inline)) {
            constexpr int u = decltype(u_)::value, which = decltype(piece_)::value;
            if constexpr (which == 0) {
                if (is_value(u)) {  // a weight of zero does not undo a NaN code: of places that no row sees, or of what stands for a page that is none
                    const int own = unit_key(u, stage) + lane / (D / 16);
                    const bool seen_by_some = (own >= from) & (own < to) & (unit_scale[u] >= ((no_page >> u & 1) != 0 ? NAN : LEAST_SCALE));
                    raw[u].x = seen_by_some ? raw[u].x : 0u;
                    raw[u].y = seen_by_some ? raw[u].y : 0u;
                    raw[u].z = seen_by_some ? raw[u].z : 0u;
                    raw[u].w = seen_by_some ? raw[u].w : 0u;
                }
            } else if constexpr (which < 7 && which % 3 != 0) {
                const uint32_t x = kv8_turn<CODE>(which == 1 ? raw[u].x : which == 2 ? raw[u].y : which == 4 ? raw[u].z : raw[u].w);
                staged[which % 3 * 2 - 2] = is_value(u) ? kv8_pair_to_f16<CODE, false>(x) : kv8_key_pair<CODE, false>(x);
                staged[which % 3 * 2 - 1] = is_value(u) ? kv8_pair_to_f16<CODE, true>(x) : kv8_key_pair<CODE, true>(x);
            } else if constexpr (which < 7) {
                uint8_t* to_tile = tiles + (is_value(u) ? 2 + ((stage - 1) & 1) : stage & 1) * Tile::BYTES;
                const int target = ((is_value(u) ? value_target : key_target) ^ (which == 3 ? 0 : 16)) + u * THREADS % SIDE_UNITS / (D / 16) * 2 * D;
                *reinterpret_cast<uint4*>(to_tile + target) = make_uint4(staged[0], staged[1], staged[2], staged[3]);
            } else {
                fetch(u, stage + 1);
            }
        };

        // the scales of 16 keys each, by the first lanes of the first wave: a tile's are read two turns ahead and written one ahead
        auto stage_scales = [&](int stage) {
            if (tid < KEYS / 16) {
                const ValueScale v = value_scale(raw_scale.y);
                // (a NaN scale of a page that a row does not see: its weights are 0, and so is their share of the sum)
                scales[stage & 1][tid] = make_float4(raw_scale.x, v.log2, isnan(v.inverse) ? 0.0f : v.inverse, 0.0f);
                const bool known = (unsigned)scale_id < (unsigned)c.pages;
                const uint32_t at = (known ? scale_id : 0) * (uint32_t)c.kv_heads + kv_head;
                raw_scale = make_float2(known ? c.k.scales[at] : NAN, known ? c.v.scales[at] : NAN);
                scale_id = table[min(own_begin + (stage + 2) * STRIDE + 16 * tid, last_key) >> c.page_shift];
            }
        };

        f32x16 o[DT];
        float top = NO_REFERENCE, sum = 0.0f;
#pragma unroll
        for (int m = 0; m < DT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                o[m][i] = 0.0f;

        f32x16 s[KEYS / 32];
        uint4 p[KEYS / 16];  // the weights of 16 keys, 8 of them this lane's
#pragma unroll
        for (int x = 0; x < KEYS / 16; ++x)
            p[x] = make_uint4(0, 0, 0, 0);
        // The matrix part of turn `tile`: the sums of the tile before, the scores of this one.  A SIMD has 32 clocks for a product that a wave issues in
        // four: in between go the reads of the fragment AHEAD products on, and a piece of the staging.  (The order is fixed by barriers for the
        // compiler, which would by itself read each fragment right before it is used.)
        constexpr int PV = KEYS / 16 * DT, QK = KEYS / 32 * STEPS, AHEAD = 4;
        static_assert(D != 256 || QK >= 8, "score products between the sums' products and scaled_accumulator");
        auto multiply = [&](int tile) __attribute__((always_inline)) {
            const uint8_t* values = tiles + (2 + ((tile - 1) & 1)) * Tile::BYTES;
            const uint8_t* keys = tiles + (tile & 1) * Tile::BYTES;
            uint4 fragments[AHEAD];
            auto read = [&](auto i_) __attribute__((always_inline)) {
                constexpr int i = decltype(i_)::value;
                if constexpr (i < PV) {
                    // a group of 16 lanes: four keys of 16 elements; each lane names 8 bytes and gets its own element of the four
                    constexpr int x = i / DT, m = i % DT;
                    const int l16 = lane % 16, k = 16 * x + 4 * hf + l16 / 4, part = 2 * m + (lane / 16) % 2;
                    fragments[i % AHEAD] = read_transposed_16(values + Tile::value_at(k, part) + l16 % 4 * 8, values + Tile::value_at(k + 8, part) + l16 % 4 * 8);
                } else if constexpr (i < PV + QK) {
                    constexpr int st = (i - PV) / (KEYS / 32), kt = (i - PV) % (KEYS / 32);
                    fragments[i % AHEAD] = *reinterpret_cast<const uint4*>(keys + Tile::key_at(32 * kt + col, 2 * st + hf));
                }
            };
            static_for<AHEAD>(read);
            __builtin_amdgcn_sched_barrier(0);
            static_for<PV + QK>([&](auto i_) __attribute__((always_inline)) {
                constexpr int i = decltype(i_)::value;
                const f16x8 f = __builtin_bit_cast(f16x8, fragments[i % AHEAD]);
                if constexpr (i < PV) {
                    constexpr int x = i / DT, m = i % DT;  // (before the first tile: weights and values of zero)
                    o[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, __builtin_bit_cast(f16x8, p[x]), o[m], 0, 0, 0);
                } else {
                    constexpr int st = (i - PV) / (KEYS / 32), kt = (i - PV) % (KEYS / 32);
                    s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, __builtin_bit_cast(f16x8, q[st]), st == 0 ? start : s[kt], 0, 0, 0);
                }
                read(std::integral_constant<int, i + AHEAD>{});
                static_for<(i + 1) * UNITS * PIECES / (PV + QK) - i * UNITS * PIECES / (PV + QK)>([&](auto n_) __attribute__((always_inline)) {
                    constexpr int n = i * UNITS * PIECES / (PV + QK) + decltype(n_)::value;
                    piece(std::integral_constant<int, n / PIECES>{}, std::integral_constant<int, n % PIECES>{}, tile + 1);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        // the vector part: scores to weights
        auto weigh = [&](int tile) __attribute__((always_inline)) {
            const int key = own_begin + tile * STRIDE, buffer = tile & 1;
            const bool whole = key >= every_from && key + KEYS <= every_to;
            float4 sc[KEYS / 16];  // of 16 keys, 8 of them this lane's
            float scale[KEYS / 16], high = -INFINITY;
            const uint32_t first = TREE ? 0 : (uint32_t)(key + 4 * hf - seen.x), visible = TREE ? 0 : (uint32_t)(seen.y - seen.x);
            uint32_t mine[2];  // (TREE: bits of this lane's keys)
            auto is_seen = [&](uint32_t from, int x, int i) __attribute__((always_inline)) {
                if constexpr (TREE)
                    return (mine[x / 2] & 1u << (16 * (x % 2) + 8 * (i / 4) + i % 4)) != 0;
                else
                    return from + (16 * x + 8 * (i / 4) + i % 4) < visible;
            };
            // (the largest of a group's scores times its scale: the scale is not negative)
#pragma unroll
            for (int x = 0; x < KEYS / 16; ++x) {
                sc[x] = scales[buffer][x];
                scale[x] = cq * sc[x].x;
                if (TREE && CODE == PTOAMD_I8)
                    sc[x].y = fmaf(bias, scale[x], sc[x].y);
            }
            find(tile + 3);
            stage_scales(tile + 1);
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
                if constexpr (TREE)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        mine[h] = seen_by_own(drafted[32 * wave + col], MANY_TREE_WORDS, key + 32 * h, seen.x, place0) >> (4 * hf);
#pragma unroll
                for (int x = 0; x < KEYS / 16; ++x)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float w = fmaf(s[x / 2][8 * (x % 2) + i], scale[x], sc[x].y);
                        high = fmaxf(high, is_seen(first, x, i) ? w : -INFINITY);
                    }
            }
            uint32_t first_again = first;  // (or the compiler keeps all 32 comparisons, 64 scalar registers)
            if constexpr (TREE)
                asm("" : "+v"(mine[0]), "+v"(mine[1]));
            else
                asm("" : "+v"(first_again));
            if (__ballot(high > top + MOST) != 0) {
                high = fmaxf(high, __shfl_xor(high, 32));
                const float next = fmaxf(top, high - SET_TO), fade = __builtin_amdgcn_exp2f(top - next);
                top = next;
                sum *= fade;
#pragma unroll
                for (int m = 0; m < DT; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if constexpr (D == 256)
                            o[m][i] = scaled_accumulator(o[m][i], fade);
                        else
                            o[m][i] *= fade;
                    }
            }
#pragma unroll
            for (int x = 0; x < KEYS / 16; ++x) {
                float w[8], eight;
                const float less = sc[x].y - top;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + i], scale[x], less));
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        w[i] = is_seen(first_again, x, i) ? w[i] : 0.0f;
                }
                p[x] = make_uint4(pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7]));
                eight = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));  // (before they are rounded: the log-sum keeps f32's bits)
                sum = fmaf(eight, sc[x].z, sum);
            }
        };

        // Where there are two waves a SIMD, the second four go one segment behind the first: one wave of a SIMD multiplies while the other weighs.  Keys
        // and values have two buffers each; what multiply(j) writes, stage j + 1, was last read in multiply(j - 1), the segment before at the latest,
        // and is next read in multiply(j + 1), the segment after at the earliest.
        const int count = begin < end ? (end - begin + STRIDE - 1) / STRIDE : 0;
        const int own_count = HALVES ? (max(end - own_begin, 0) + STRIDE - 1) / STRIDE : count;  // (the second half may have one less)
        const bool behind = HALVES ? half != 0 : WAVES == 8 && wave >= 4;
        if (count > 0) {
            find(0);
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                fetch(u, 0);
            take_queries();
            if (tid < KEYS / 16)
                scale_id = table[min(own_begin + 16 * tid, last_key) >> c.page_shift];
            find(1);
            static_for<UNITS * PIECES>([&](auto n_) __attribute__((always_inline)) {
                constexpr int n = decltype(n_)::value;
                piece(std::integral_constant<int, n / PIECES>{}, std::integral_constant<int, n % PIECES>{}, 0);
            });
            find(2);
            stage_scales(-1);  // (tile 0's are read here; what is written is written again)
            stage_scales(0);
            __syncthreads();
            if (behind)
                __syncthreads();
            for (int tile = 0; tile <= count; ++tile) {
                if (WAVES == 8)
                    __builtin_amdgcn_s_setprio(1);  // (ahead of the SIMD's other wave, whatever its age)
                if (!HALVES || tile <= own_count)
                    multiply(tile);
                if (WAVES == 8) {
                    __builtin_amdgcn_s_setprio(0);
                    __syncthreads();
                }
                if (tile < own_count)
                    weigh(tile);
                __syncthreads();
            }
            if (WAVES == 8 && !behind)
                __syncthreads();
        }

        sum += __shfl_xor(sum, 32);
        if constexpr (HALVES) {
            // the second half's sums to the first, on the reference of both, where the tiles were: 16 elements of a lane at a time, lane beside lane
            float* other = reinterpret_cast<float*>(all_tiles) + wave * (DT * 16 + 2) * 64 + lane;
            static_assert(GROUP * (DT * 16 + 2) * 64 * 4 <= 8 * Tile::BYTES, "the second half's sums lie in the tiles' room");
            if (half != 0) {
#pragma unroll
                for (int m = 0; m < DT; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        other[(m * 16 + i) * 64] = o[m][i];
                other[DT * 16 * 64] = top;
                other[(DT * 16 + 1) * 64] = sum;
            }
            __syncthreads();
            if (half == 0) {
                const float its_top = other[DT * 16 * 64], its_sum = other[(DT * 16 + 1) * 64], to_top = fmaxf(top, its_top);
                const float mine = __builtin_amdgcn_exp2f(top - to_top), its = __builtin_amdgcn_exp2f(its_top - to_top);
                top = to_top;
                sum = sum * mine + its_sum * its;
#pragma unroll
                for (int m = 0; m < DT; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[m][i] = o[m][i] * mine + other[(m * 16 + i) * 64] * its;
            }
            __syncthreads();  // (rows leave through the same room)
            if (half != 0) {
                if (unit < unit_end)
                    __syncthreads();  // (the first half's, behind its rows)
                continue;
            }
        }
        const ArgumentsAgain e;
        const int64_t part_row = (int64_t)max(part, 0) * c.tokens * a.heads;
        if (valid && hf == 0) {
            const int64_t at = (int64_t)(span.first + token) * a.heads + head;
            float* lse = e.global<float>(offsetof(AttentionArgs, lse));
            if (part >= 0)
                e.global<float2>(offsetof(AttentionArgs, part_sum))[part_row + at] = make_float2(top, sum);
            else if (lse != nullptr)
                lse[at] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
        }
        // A lane's elements are four in a row here and there: 32 of every row at a time go through LDS, where the tiles were (behind the last barrier
        // nobody reads those), so that two lanes have a row's and store 16 each.
        const float inverse = part >= 0 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
        uint8_t* mine = tiles + wave * 4096;
        static_assert(GROUP * 4096 <= 4 * Tile::BYTES, "a wave's rows of 32 f32 lie in the tiles' room");
        const int own = lane / 2, own_row = row0 + 32 * wave + own, own_token = own_row / a.group, own_head = kv_head * a.group + own_row - own_token * a.group;
        float* part_out = e.global<float>(offsetof(AttentionArgs, part_out)) + (part_row + (int64_t)(span.first + own_token) * a.heads + own_head) * D + 16 * (lane % 2);
        uint8_t* out = e.global<uint8_t>(offsetof(AttentionArgs, out)) + (int64_t)(span.first + own_token) * ARGUMENT(e, out_token) + (int64_t)own_head * ARGUMENT(e, out_head) + 32 * (lane % 2);
        const bool wide = ARGUMENT(e, wide);
        const int head_dim = e.field<int>(offsetof(AttentionArgs, cache) + offsetof(Kv8, head_dim));
#pragma unroll
        for (int m = 0; m < DT; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(mine + col * 128 + ((2 * i + hf) ^ (col & 7)) * 16) =
                    f32x4{o[m][4 * i] * inverse, o[m][4 * i + 1] * inverse, o[m][4 * i + 2] * inverse, o[m][4 * i + 3] * inverse};
            f32x4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = *reinterpret_cast<const f32x4*>(mine + own * 128 + ((4 * (lane % 2) + i) ^ (own & 7)) * 16);
            if (own_row >= rows || 32 * m + 16 * (lane % 2) >= head_dim)
                continue;
            if (part >= 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(part_out + 32 * m + 4 * i) = x[i];
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    store_row8<T>(out + 64 * m + 16 * i, wide, reinterpret_cast<const float*>(&x[2 * i]));
            }
        }
        if (unit < unit_end)
            __syncthreads();  // (the tiles' room is the next one's)
    } while (unit < unit_end);
}

template <typename T, int CODE, int D, int WAVES, bool TREE, bool HALVES>
static int launch_many(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    constexpr int bytes = (HALVES ? 8 : 4) * ManyTile<D>::BYTES;
    PTOAMD_HIP_CHECK((ensure_dynamic_lds<&attention_kv8_many_kernel<T, CODE, D, WAVES, TREE, HALVES>>(bytes)));
    if (a.heads == 0)  // (prepare_attention_kernels)
        return PTOAMD_OK;
    const dim3 grid = a.splits > 1 ? dim3((unsigned)device_compute_units()) : dim3((unsigned)(a.row_tiles * a.cache.kv_heads), (unsigned)sequences);
    hipLaunchKernelGGL((attention_kv8_many_kernel<T, CODE, D, WAVES, TREE, HALVES>), grid, dim3(64 * WAVES), bytes, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    return PTOAMD_OK;
}
template <typename T, int CODE, bool TREE>
static int choose_size(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    switch (built_head(a.cache.head_dim)) {
        case 64:
            if (TREE && a.tile_rows == 128)
                return launch_many<T, CODE, 64, 8, TREE, TREE>(a, sequences, stream);
            return launch_many<T, CODE, 64, 8, TREE, false>(a, sequences, stream);
        case 128:
            if (TREE && a.tile_rows == 128)
                return launch_many<T, CODE, 128, 8, TREE, TREE>(a, sequences, stream);
            return launch_many<T, CODE, 128, 8, TREE, false>(a, sequences, stream);
        default: return launch_many<T, CODE, 256, 4, TREE, false>(a, sequences, stream);
    }
}

}  // namespace ptoamd
