// Attention over an 8-bit cache for few queries: decode, and a few tokens guessed ahead; the joining of parts.
#include "attention_kv8_few.hpp"

namespace ptoamd {

int launch_attention_few(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream)
{
    if (f16)
        return code == PTOAMD_I8 ? choose_size<_Float16, PTOAMD_I8, false>(a, sequences, stream) : choose_size<_Float16, PTOAMD_E4M3, false>(a, sequences, stream);
    return code == PTOAMD_I8 ? choose_size<__bf16, PTOAMD_I8, false>(a, sequences, stream) : choose_size<__bf16, PTOAMD_E4M3, false>(a, sequences, stream);
}

// The parts of a sequence's keys, joined in their order, so the result does not depend on which part was done first.  A row's D / 4 lanes hold four
// elements each.  ROWS = 1: few rows of many parts, one a workgroup, whose 1024 / D groups of lanes take every (1024 / D)-th part and are added in
// order.  Else ROWS = 1024 / D rows a workgroup, a group of lanes each: no group waits for another.
// (1309 rows of tokens, 32 heads of 128, two parts: 42.3 us with ROWS = 1, some 14 with 8.)
template <typename T, int D, int ROWS, bool TREE>
__global__ void __launch_bounds__(256) attention_kv8_join_kernel(AttentionArgs a)
{
    constexpr int LANES = D / 4, GROUPS = 256 / LANES, STEP = ROWS == 1 ? GROUPS : 1;
    static_assert(ROWS == 1 || ROWS == GROUPS, "a row has a workgroup or a group of lanes");
    __shared__ float4 partial[ROWS == 1 ? GROUPS : 1][LANES];
    __shared__ float group_sum[GROUPS], group_top[GROUPS];
    const int i = threadIdx.x % LANES, group = threadIdx.x / LANES, seq = blockIdx.z;
    const int row = blockIdx.x * ROWS + (ROWS == 1 ? 0 : group), nth = row / a.heads, head = row - nth * a.heads;  // (rows: tokens times heads)
    const Span span = span_of(a, seq);
    if (nth >= span.count)
        return;
    const int64_t at = (int64_t)(span.first + nth) * a.heads + head, stride = (int64_t)a.cache.tokens * a.heads;
    int from = 0, to;
    if (a.cuts != nullptr) {  // (rows of one part are written already)
        const int kv_head = head / a.group, tile = seq * a.row_tiles + (nth * a.group + head - kv_head * a.group) / a.tile_rows;
        const int stretch = a.cuts[Cuts::STRETCH], first = kv_head * a.cuts[Cuts::HEAD] + a.cuts[Cuts::FIRST + tile] + many_start(D, a.tile_rows);
        const int last = kv_head * a.cuts[Cuts::HEAD] + a.cuts[Cuts::FIRST + tile + 1] - 1;
        to = last / stretch - first / stretch + 1;
        if (to == 1)
            return;
    } else {
        if (!several_parts(a, span))
            return;
        const int2 keys = TREE ? keys_of_any<true>(a, span, nth, nth) : visible_keys(a, span.length - span.count + nth, span.length);
        from = min((keys.x - span.begin) / a.chunk, a.splits - 1);
        to = keys.y > keys.x ? min((keys.y - 1 - span.begin) / a.chunk, a.splits - 1) + 1 : from;
    }
    float top = NO_REFERENCE, sum = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    for (int part = from + (ROWS == 1 ? group : 0); part < to; part += STEP)
        top = fmaxf(top, a.part_sum[part * stride + at].x);
#pragma unroll 4
    for (int part = from + (ROWS == 1 ? group : 0); part < to; part += STEP) {
        const float2 s = a.part_sum[part * stride + at];
        const float4 x = *reinterpret_cast<const float4*>(a.part_out + (part * stride + at) * D + 4 * i);
        const float by = __builtin_amdgcn_exp2f(s.x - top);
        sum += s.y * by;
        o = make_float4(o.x + x.x * by, o.y + x.y * by, o.z + x.z * by, o.w + x.w * by);
    }
    if constexpr (ROWS == 1) {
        partial[group][i] = o;
        if (i == 0) {
            group_top[group] = top;
            group_sum[group] = sum;
        }
        __syncthreads();
        if (threadIdx.x >= LANES)
            return;
        top = group_top[0];
#pragma unroll
        for (int k = 1; k < GROUPS; ++k)
            top = fmaxf(top, group_top[k]);
        sum = 0.0f;
        o = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
            const float by = __builtin_amdgcn_exp2f(group_top[k] - top);
            const float4 x = partial[k][i];
            sum += group_sum[k] * by;
            o = make_float4(o.x + x.x * by, o.y + x.y * by, o.z + x.z * by, o.w + x.w * by);
        }
    }
    if (4 * i >= a.cache.head_dim)
        return;
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = reinterpret_cast<T*>(a.out + (int64_t)(span.first + nth) * a.out_token + (int64_t)head * a.out_head) + 4 * i;
    const float x[4] = {sum == 0.0f ? 0.0f : o.x * inverse, sum == 0.0f ? 0.0f : o.y * inverse, sum == 0.0f ? 0.0f : o.z * inverse, sum == 0.0f ? 0.0f : o.w * inverse};
    if (a.wide) {
        T four[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            four[j] = (T)x[j];
        *reinterpret_cast<uint2*>(out) = __builtin_bit_cast(uint2, four);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            out[j] = (T)x[j];
    }
    if (a.lse != nullptr && i == 0)
        a.lse[at] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

template <typename T, int D, bool TREE>
static void launch_join(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    const long rows = (long)a.cache.max_tokens * a.heads;
    constexpr int ROWS = 1024 / D;
    // (rows for four workgroups a compute unit, of a group of lanes each: before that a row's parts are what keeps the card busy.  Of drafted tokens, also where
    // the parts are few: 16 x 6 tokens over 4000 keys in two, 64 / 8 heads of 128, 47.8 us with a row a workgroup, 43.0; one over 1000 in four 10.7 and 11.1)
    if (rows * sequences >= 4L * ROWS * device_compute_units() || (TREE && a.splits <= 4))
        hipLaunchKernelGGL((attention_kv8_join_kernel<T, D, ROWS, TREE>), dim3((unsigned)((rows + ROWS - 1) / ROWS), 1, (unsigned)sequences), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_kv8_join_kernel<T, D, 1, TREE>), dim3((unsigned)rows, 1, (unsigned)sequences), dim3(256), 0, stream, a);
}
template <typename T, bool TREE>
static void choose_join(const AttentionArgs& a, int sequences, hipStream_t stream)
{
    switch (built_head(a.cache.head_dim)) {
        case 64: launch_join<T, 64, TREE>(a, sequences, stream); break;
        case 128: launch_join<T, 128, TREE>(a, sequences, stream); break;
        default: launch_join<T, 256, TREE>(a, sequences, stream); break;
    }
}
int launch_attention_join(const AttentionArgs& a, bool f16, int sequences, hipStream_t stream)
{
    const bool tree = a.tree != nullptr;
    if (f16)
        tree ? choose_join<_Float16, true>(a, sequences, stream) : choose_join<_Float16, false>(a, sequences, stream);
    else
        tree ? choose_join<__bf16, true>(a, sequences, stream) : choose_join<__bf16, false>(a, sequences, stream);
    PTOAMD_HIP_CHECK(hipGetLastError());
    return PTOAMD_OK;
}

}  // namespace ptoamd
