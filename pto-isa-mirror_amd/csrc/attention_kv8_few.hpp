// Attention over an 8-bit cache for few queries: decode, a few tokens guessed ahead, small drafted trees.
#pragma once
#include "attention_kv8.hpp"

namespace ptoamd {

// The rows of a sequence and key head -- its new tokens times the query heads that share the head, token-major -- are the columns of the
// matrix instructions, 16 a tile, NT tiles a workgroup; keys are their rows.  A wave takes 32 keys at a time straight from memory into registers:
//   S^T = K q^T : a lane's fragment is 8 codes of one key.  Which elements of the head make up a step is free as long as q's fragment has
//                 the same, so a lane reads 16 bytes in a row and has two steps of them.
//   o^T = V^T p^T : a lane holds the scores of keys 4 g .. 4 g + 3 and 16 + 4 g .. (g = lane / 16) for its column: with these eight
//                 keys as its share of the product's sum, the weights are the fragment as they stand.  V's fragment is one element of
//                 the same eight keys: the lane reads D / 16 elements in a row of each and pairs them up by byte.
// So nothing passes through LDS, and no lane needs another's data but for the maximum and the sums of a row.  Codes become f16 on the way, exactly:
// E4M3 by conversion, int8 as (code + 128) 2^-24 by a permutation of bytes alone (KV8_UNIT).  The 128 leaves the scores by where their sums start, and
// the values' sums tile by tile by a product of a constant with the same weights, so that what cancels is never larger than one tile.
// A tile is 450 to 600 instructions of a wave, which alone on its SIMD takes 0.9 us for it (heads of 128; 0.66 of 64): of a SIMD's two waves one
// computes while the other's codes arrive.  Scores, references and sums are f32; a page's value scale goes into the weight (ValueScale).
// Every wave has its own keys (turns of 32 a wave through the workgroup's part) and the waves join at the end.
// Bound: HBM.  16 sequences of 8192 keys, 64 / 8 heads of 128, E4M3: 270 MB in 54.4 us, 4.95 TB/s (a large copy: 5.13); a sequence of 131072, int8: 54.8 us.
template <int D>
struct FewTile {
    static constexpr int VW = D / 64;  // dwords a lane reads of one key's values
    uint4 k[2][D / 64];
    uint32_t v[8][VW];
    float scale;  // lanes 0, 1: the key scales of the tile's halves; 2, 3: their value scales (and so on)
    float unknown;  // NaN where the table names no page
};

// TREE: of drafted tokens.  Keys of the step itself are few: their tiles alone look at a row's bits, which every wave has in LDS for itself.  Eight waves a
// workgroup but for three and four tiles of rows of heads of 128 and two of 256 (few_waves): rows are many more than in decode, and twice the waves halve the turns.
// Bound: a wave's instructions and, of short sequences, the chain length -> page -> codes.  7 tokens over 300 keys, 32 / 8 heads of 128, int8, 8.4 us; 8 of 24 over 1000,
// 64 / 8 heads, E4M3, 31; 40 of up to 63 over up to 3503 (665 on average), 16 / 16 of 64, 32: the longest sequence's 14 turns of two workgroups a CU.
template <typename T, int CODE, int D, int NT, int WAVES, bool TREE>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(TREE && D == 64 && NT <= 2 ? 4 : WAVES / 4))) attention_kv8_few_kernel(AttentionArgs a)
{
    constexpr int STEPS = D / 32, VW = D / 64, MT = D / 16, PITCH = D + 4;
    constexpr int RING = 2;  // tiles of a wave in registers
    constexpr int STRIDE = 32 * WAVES;
    constexpr int TREE_WORDS = PTOAMD_MOST_DRAFTED / 32;
    constexpr bool Q_IN_LDS = few_queries_in_lds(D, NT, TREE);
    extern __shared__ __attribute__((aligned(16))) float shared[];  // [WAVES / 2][16 NT][PITCH]
    __shared__ float wave_top[WAVES][16 * NT], wave_sum[WAVES][16 * NT];
    __shared__ uint4 queries[Q_IN_LDS ? NT * STEPS : 1][Q_IN_LDS ? 64 : 1];
    __shared__ uint32_t drafted[TREE ? WAVES : 1][TREE ? 16 * NT : 1][TREE_WORDS + 1];  // (last: the first of the older keys that the row sees)
    const Kv8& c = a.cache;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 16, g = lane / 16;
    // (workgroups go to the XCDs in turn: parts, of which short sequences leave most empty, are the slowest index)
    const int kv_head = blockIdx.x % c.kv_heads, row0 = blockIdx.x / c.kv_heads * 16 * NT, part = blockIdx.z;
    int seq = blockIdx.y;
    const Span span = TREE && a.longest > 0 ? span_in_turn(a, blockIdx.y, &seq) : span_of(a, blockIdx.y);
    const int rows = span.count * a.group;
    const int begin = a.splits > 1 ? span.begin + part * a.chunk : span.begin;
    const int end = part + 1 < a.splits ? min(span.length, begin + a.chunk) : span.length;  // (the last takes what a wrong max_length left out)
    if (row0 >= rows || (begin >= end && part > 0))
        return;

    // A tile in WAVES is a wave's.  RING tiles are in registers or under way, and the page ids of RING more: the ids were asked for ahead of codes
    // that have been waited for when they are used.
    const int first = begin + 32 * wave;
    const int32_t* table = c.table + (int64_t)seq * c.max_pages;
    auto find = [&](int key) { return table[min((key + 16 * (lane & 1)) >> c.page_shift, c.max_pages - 1)]; };  // even lanes: of the first half, odd: the second
    uint32_t k_lane[D / 64];  // (beyond the head: its first elements)
#pragma unroll
    for (int cc = 0; cc < D / 64; ++cc)
        k_lane[cc] = (uint32_t)(col * (int)c.k.token + (64 * cc + 16 * g < c.head_dim ? 64 * cc + 16 * g : 0));
    const uint32_t v_lane = (uint32_t)(4 * g * (int)c.v.token + (col * (D / 16) < c.head_dim ? col * (D / 16) : 0));
    const uint8_t *k_head = c.k.codes + kv_head * c.k.head, *v_head = c.v.codes + kv_head * c.v.head;
    const uint32_t k_page = (uint32_t)(c.k.page >> 3), v_page = (uint32_t)(c.v.page >> 3);  // (pages start on 8 bytes)
    const float* scales = lane & 2 ? c.v.scales : c.k.scales;
    auto fetch = [&](FewTile<D>& tile, int key, int id) __attribute__((always_inline)) {
        const bool known = (unsigned)id < (unsigned)c.pages;
        const int page_lane = known ? id : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(page_lane, h), slot = (uint32_t)(key + 16 * h) & ((1u << c.page_shift) - 1);
            const int bytes = key + 16 * h < end ? 0x7FFFFFFF : 0;  // (a half with no key of the part is not read: its codes are zeros)
            const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(k_head + ((uint64_t)page * k_page * 8 + slot * (uint32_t)c.k.token)), 0, bytes, 0x20000);
            const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(v_head + ((uint64_t)page * v_page * 8 + slot * (uint32_t)c.v.token)), 0, bytes, 0x20000);
#pragma unroll
            for (int cc = 0; cc < D / 64; ++cc)
                if (TREE && D == 256 && cc == 1)  // (a register less: such heads have more than 128 elements)
                    tile.k[h][cc] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane[0], 64, 0));
                else
                    tile.k[h][cc] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane[cc], 0, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * (int)c.v.token;
                if constexpr (VW == 1) {
                    tile.v[4 * h + i][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, v_lane, row, 0);
                } else if constexpr (VW == 2) {
                    const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(vr, v_lane, row, 0));
                    tile.v[4 * h + i][0] = w.x, tile.v[4 * h + i][1] = w.y;
                } else {
                    const uint4 w = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane, row, 0));
                    tile.v[4 * h + i][0] = w.x, tile.v[4 * h + i][1] = w.y, tile.v[4 * h + i][2] = w.z, tile.v[4 * h + i][3] = w.w;
                }
            }
        }
        if constexpr (TREE && D == 256) {
            int again = lane;
            asm("" : "+v"(again));  // (or the address is kept in two registers)
            tile.scale = (again & 2 ? c.v.scales : c.k.scales)[(uint32_t)(page_lane * c.kv_heads + kv_head)];
        } else {
            tile.scale = scales[(uint32_t)(page_lane * c.kv_heads + kv_head)];
        }
        tile.unknown = known ? 0.0f : NAN;  // (added where the scale is used: here it would be waited for)
        __builtin_amdgcn_sched_barrier(0);  // (the order of the loads is what the waits count on)
    };
    int ids[RING];
    FewTile<D> tiles[RING];
#pragma unroll
    for (int s = 0; s < RING; ++s)
        ids[s] = find(first + s * STRIDE);

    const int tree_words = a.tree_words;  // (at most TREE_WORDS)
    if constexpr (TREE) {
        for (int i = lane; i < 16 * NT * tree_words; i += 64) {
            const int row = row0 + i % (16 * NT), word = i / (16 * NT);
            drafted[wave][i % (16 * NT)][word] = row < rows ? drafted_word(a, span, row / a.group, word) : 0u;
        }
    }

    // the queries, as fragments: step st = 2 cc + e of a lane is elements 64 cc + 16 g + 8 e ..
    uint4 q[NT][STEPS];
    int2 seen[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = row0 + 16 * t + col, token = row / a.group;
        const bool valid = row < rows;
        if constexpr (TREE)
            drafted[wave][16 * t + col][TREE_WORDS] = first_of_drafted(a, span, drafted[wave][16 * t + col], tree_words, valid, token);
        else
            seen[t] = valid ? visible_keys(a, span.length - span.count + token, span.length) : make_int2(0, 0);
        const uint8_t* p = a.q + (int64_t)(span.first + (valid ? token : 0)) * a.q_token + (int64_t)(kv_head * a.group + (valid ? row - token * a.group : 0)) * a.q_head;
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
            q[t][st] = valid && 64 * (st / 2) + 16 * g < c.head_dim ? load_row8(p + 2 * (64 * (st / 2) + 16 * g + 8 * (st % 2)), a.wide) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int s = 0; s < RING; ++s) {
        const int id = ids[s];
        ids[s] = find(first + (s + RING) * STRIDE);
        fetch(tiles[s], first + s * STRIDE, id);
    }
    float cq[NT];  // what a product of codes is multiplied with beside the key scale, in units of log2
    f32x4 start[NT];
    float bias[NT];  // (TREE: what `start` is, for all keys, taken off where scores are scaled: one register for four)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        uint32_t largest = largest_of<STEPS>(q[t]);
        largest = max(largest, (uint32_t)__shfl_xor((int)largest, 16));
        largest = max(largest, (uint32_t)__shfl_xor((int)largest, 32));
        const RowScale r = row_scale<T>(largest);
        cq[t] = r.up * (a.scale * 1.44269504088896341f) * KV8_UNIT<CODE>;
        scale_to_f16<T, STEPS>(q[t], r.down);
        // where the products' sums start: without the 128 that int8 codes carry
        start[t] = f32x4{0, 0, 0, 0};
        if (CODE == PTOAMD_I8) {
            const uint4 unbias = make_uint4(UNBIAS, UNBIAS, UNBIAS, UNBIAS);
#pragma unroll
            for (int st = 0; st < STEPS; ++st)
                start[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, unbias), __builtin_bit_cast(f16x8, q[t][st]), start[t], 0, 0, 0);
        }
        bias[t] = start[t][0];
        if (TREE)
            start[t] = f32x4{0, 0, 0, 0};
        if constexpr (Q_IN_LDS)  // (every wave the same, and each reads behind its own)
#pragma unroll
            for (int st = 0; st < STEPS; ++st)
                queries[t * STEPS + st][lane] = q[t][st];
    }
    // tiles of keys that every row sees need no mask; keys that none sees have their codes cleared
    const int every_from = first_key(span.length - 1, a.window);
    const int every_to = TREE ? span.length - span.count : a.causal ? span.length - span.count + 1 : span.length;
    const int any_from = first_key(span.length - span.count, a.window);

    f32x4 o[NT][MT];
    float top[NT], sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        top[t] = NO_REFERENCE;
        sum[t] = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
            o[t][m] = f32x4{0, 0, 0, 0};
    }

    auto compute = [&](FewTile<D>& tile, int key) __attribute__((always_inline)) {
        if constexpr (Q_IN_LDS)
            asm volatile("" ::: "memory");  // (or the queries are read once, into registers)
        const int scale = (int)f2u(tile.scale + tile.unknown);
        const float ks[2] = {u2f(__builtin_amdgcn_readlane(scale, 0)), u2f(__builtin_amdgcn_readlane(scale, 1))};
        const float vs[2] = {u2f(__builtin_amdgcn_readlane(scale, 2)), u2f(__builtin_amdgcn_readlane(scale, 3))};
        f32x4 s[NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
                s[t][h] = start[t];
            static_for<D / 64>([&](auto cc_) {
                constexpr int cc = decltype(cc_)::value;
                const uint4 raw = tile.k[h][cc];
                const uint32_t w[4] = {kv8_turn<CODE>(raw.x), kv8_turn<CODE>(raw.y), kv8_turn<CODE>(raw.z), kv8_turn<CODE>(raw.w)};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint4 f;
                    if constexpr (CODE == PTOAMD_I8)  // (a pair of bytes of one dword)
                        f = make_uint4(__builtin_amdgcn_perm(0, w[2 * e], 0x0C010C00u), __builtin_amdgcn_perm(0, w[2 * e], 0x0C030C02u),
                                       __builtin_amdgcn_perm(0, w[2 * e + 1], 0x0C010C00u), __builtin_amdgcn_perm(0, w[2 * e + 1], 0x0C030C02u));
                    else
                        f = make_uint4(kv8_pair_to_f16<CODE, false>(w[2 * e]), kv8_pair_to_f16<CODE, true>(w[2 * e]),
                                       kv8_pair_to_f16<CODE, false>(w[2 * e + 1]), kv8_pair_to_f16<CODE, true>(w[2 * e + 1]));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint4 its = Q_IN_LDS ? queries[t * STEPS + 2 * cc + e][lane] : q[t][2 * cc + e];
                        s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, f), __builtin_bit_cast(f16x8, its), s[t][h], 0, 0, 0);
                    }
                }
            });
        }
        const bool whole = key >= every_from && key + 32 <= every_to;
        const ValueScale value[2] = {value_scale(vs[0]), value_scale(vs[1])};
        uint4 p[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float w[2][4], high = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float scale = cq[t] * ks[h], add = TREE && CODE == PTOAMD_I8 ? fmaf(bias[t], scale, value[h].log2) : value[h].log2;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[h][i] = fmaf(s[t][h][i], scale, add);
            }
            if (TREE && !whole) {
                const uint32_t* row = drafted[wave][16 * t + col];
                const uint32_t mine = seen_by_own(row, tree_words, key, (int)row[TREE_WORDS], every_to) >> (4 * g);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    w[j / 4][j % 4] = (mine & 1u << (16 * (j / 4) + j % 4)) != 0 ? w[j / 4][j % 4] : -INFINITY;
            } else if (!whole) {
                const uint32_t from = (uint32_t)(key + 4 * g - seen[t].x), count = (uint32_t)(seen[t].y - seen[t].x);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    w[j / 4][j % 4] = from + (16 * (j / 4) + j % 4) < count ? w[j / 4][j % 4] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                high = fmaxf(high, w[j / 4][j % 4]);
            if (__ballot(high > top[t] + MOST) != 0) {
                high = fmaxf(high, __shfl_xor(high, 16));
                high = fmaxf(high, __shfl_xor(high, 32));
                const float to = fmaxf(top[t], high - SET_TO), fade = __builtin_amdgcn_exp2f(top[t] - to);
                top[t] = to;
                sum[t] *= fade;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[t][m][i] *= fade;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[h][i] = __builtin_amdgcn_exp2f(w[h][i] - top[t]);
                const float four = (w[h][0] + w[h][1]) + (w[h][2] + w[h][3]);
                sum[t] = four == 0.0f ? sum[t] : fmaf(four, value[h].inverse, sum[t]);  // (a NaN scale that the row does not see)
            }
            p[t] = make_uint4(pack_f16(w[0][0], w[0][1]), pack_f16(w[0][2], w[0][3]), pack_f16(w[1][0], w[1][1]), pack_f16(w[1][2], w[1][3]));
        }
        // A weight of zero does not undo a NaN code: those of places that no row sees, of pages that count as zeros, and what was read in place of a page
        // that the table does not name (its scale is NaN, which is what makes the rows that do see it NaN).
        if (key < any_from || key + 32 > span.length || !(vs[0] >= LEAST_SCALE) || !(vs[1] >= LEAST_SCALE)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = key + 16 * (j / 4) + 4 * g + j % 4;
#pragma unroll
                for (int w = 0; w < VW; ++w)
                    tile.v[j][w] = at < any_from || at >= span.length || !(vs[j / 4] >= LEAST_SCALE) ? 0u : tile.v[j][w];
            }
        }
        static_for<VW>([&](auto w_) {
            constexpr int w = decltype(w_)::value;
            uint32_t x[8], low[4], high[4];  // low, high (E4M3) of keys 2 j and 2 j + 1: bytes 0 and 1 of both, bytes 2 and 3
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = kv8_turn<CODE>(tile.v[j][w]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                low[j] = __builtin_amdgcn_perm(x[2 * j], x[2 * j + 1], 0x01050004u);
                high[j] = __builtin_amdgcn_perm(x[2 * j], x[2 * j + 1], 0x03070206u);
            }
            static_for<4>([&](auto b_) __attribute__((always_inline)) {
                constexpr int b = decltype(b_)::value;
                uint32_t f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    f[j] = CODE == PTOAMD_I8 ? bytes_to_f16(x[2 * j], x[2 * j + 1], b) : kv8_pair_to_f16<CODE, b % 2 == 1>(b < 2 ? low[j] : high[j]);
                const uint4 frag = make_uint4(f[0], f[1], f[2], f[3]), unbias = make_uint4(UNBIAS, UNBIAS, UNBIAS, UNBIAS);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    f32x4& sums = o[t][4 * w + b];
                    sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, frag), __builtin_bit_cast(f16x8, p[t]), sums, 0, 0, 0);
                    if (CODE == PTOAMD_I8)  // less 128 of every weight, in the same tile: what cancels is as small as the tile's weights
                        sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, unbias), __builtin_bit_cast(f16x8, p[t]), sums, 0, 0, 0);
                }
            });
        });
    };

    bool more = first < end;
    int key = first;
    do {
        static_for<RING>([&](auto s_) __attribute__((always_inline)) {
            constexpr int s = decltype(s_)::value;
            const int at = key + s * STRIDE;
            if (!more || at >= end) {
                more = false;
                return;
            }
            compute(tiles[s], at);
            __builtin_amdgcn_sched_barrier(0);
            const int id = ids[s];
            ids[s] = find(at + 2 * RING * STRIDE);
            fetch(tiles[s], at + RING * STRIDE, id);
        });
        key += RING * STRIDE;
    } while (more);

    // the waves' sums on one reference for each row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] += __shfl_xor(sum[t], 16);
        sum[t] += __shfl_xor(sum[t], 32);
        if (g == 0) {
            wave_top[wave][16 * t + col] = top[t];
            wave_sum[wave][16 * t + col] = sum[t];
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float to = wave_top[0][16 * t + col];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            to = fmaxf(to, wave_top[w][16 * t + col]);
        const float fade = __builtin_amdgcn_exp2f(top[t] - to) * KV8_UNIT<CODE>;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[t][m][i] *= fade;
    }
    // a lane has D / 4 elements of its column's row from 4 g D / 16 on: element (4 g + i) D / 16 + m is o[t][m][i]
    float* mine = shared + (wave % (WAVES / 2)) * (16 * NT * PITCH) + col * PITCH + g * (D / 4);
    auto each = [&](auto&& f) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < MT; m += 4)
                    f(reinterpret_cast<f32x4*>(mine + t * 16 * PITCH + i * MT + m), f32x4{o[t][m][i], o[t][m + 1][i], o[t][m + 2][i], o[t][m + 3][i]});
    };
    if (wave >= WAVES / 2)
        each([](f32x4* at, f32x4 x) { *at = x; });
    __syncthreads();
    if (wave < WAVES / 2)
        each([](f32x4* at, f32x4 x) { *at += x; });
    __syncthreads();
    for (int u = threadIdx.x; u < min(rows - row0, 16 * NT) * (D / 8); u += 64 * WAVES) {
        const int row = u / (D / 8), piece = u % (D / 8) * 8, token = (row0 + row) / a.group, head = kv_head * a.group + row0 + row - token * a.group;
        if (piece >= c.head_dim)
            continue;
        float to = wave_top[0][row];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            to = fmaxf(to, wave_top[w][row]);
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            total += wave_sum[w][row] * __builtin_amdgcn_exp2f(wave_top[w][row] - to);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = shared[row * PITCH + piece + i];
#pragma unroll
        for (int w = 1; w < WAVES / 2; ++w)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] += shared[(16 * NT * w + row) * PITCH + piece + i];
        const int64_t at = (int64_t)(span.first + token) * a.heads + head;
        if (several_parts(a, span)) {
            float* out = a.part_out + ((int64_t)part * c.tokens * a.heads + at) * D + piece;
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *reinterpret_cast<f32x4*>(out + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            if (piece == 0)
                a.part_sum[(int64_t)part * c.tokens * a.heads + at] = make_float2(to, total);
        } else {
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = total == 0.0f ? 0.0f : x[i] * inverse;
            store_row8<T>(a.out + (int64_t)(span.first + token) * a.out_token + (int64_t)head * a.out_head + 2 * piece, a.wide, x);
            if (a.lse != nullptr && piece == 0)
                a.lse[at] = total == 0.0f ? -INFINITY : (to + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
        }
    }
}

template <typename T, int CODE, int D, int NT, int WAVES, bool TREE>
static int launch_few(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    constexpr int bytes = WAVES / 2 * 16 * NT * (D + 4) * 4;
    PTOAMD_HIP_CHECK((ensure_dynamic_lds<&attention_kv8_few_kernel<T, CODE, D, NT, WAVES, TREE>>(bytes)));
    if (a.heads == 0)  // (prepare_attention_kernels)
        return PTOAMD_OK;
    const int row_groups = (a.cache.max_tokens * a.group + 16 * NT - 1) / (16 * NT);
    hipLaunchKernelGGL((attention_kv8_few_kernel<T, CODE, D, NT, WAVES, TREE>), dim3((unsigned)(a.cache.kv_heads * row_groups), (unsigned)sequences, (unsigned)a.splits),
                       dim3(64 * WAVES), bytes, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    return PTOAMD_OK;
}
template <typename T, int CODE, int D, bool TREE>
static int choose_tiles(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    // (two tiles of 256 columns' sums and fragments fit the registers of one wave a SIMD alone, as do four of 128 columns)
    switch (a.row_tiles) {
        case 1: return launch_few<T, CODE, D, 1, few_waves(D, 1, TREE), TREE>(a, sequences, stream);
        case 2: if constexpr (D < 256 || TREE) return launch_few<T, CODE, D, 2, few_waves(D, 2, TREE), TREE>(a, sequences, stream); break;
        case 3: if constexpr (D < 256) return launch_few<T, CODE, D, 3, few_waves(D, 3, TREE), TREE>(a, sequences, stream); break;
        case 4: if constexpr (D == 128) return launch_few<T, CODE, D, 4, few_waves(D, 4, TREE), TREE>(a, sequences, stream); break;
    }
    return PTOAMD_E_INVALID;  // (no plan has it)
}
template <typename T, int CODE, bool TREE>
static int choose_size(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    switch (built_head(a.cache.head_dim)) {
        case 64: return choose_tiles<T, CODE, 64, TREE>(a, sequences, stream);
        case 128: return choose_tiles<T, CODE, 128, TREE>(a, sequences, stream);
        default: return choose_tiles<T, CODE, 256, TREE>(a, sequences, stream);
    }
}

}  // namespace ptoamd
