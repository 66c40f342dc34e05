// Drafted trees: which tokens each token of a step sees among those that were drafted with it.
#include "common_host.hpp"
#include "drafted.hpp"

namespace ptoamd {

struct DraftTreeArgs {
    uint64_t* tree;
    const int32_t* parents;
    const int32_t* cu_tokens;
    int words, tokens, max_tokens;
    int all;  // rows that no sequence has become empty ones
};

// One workgroup a sequence, one thread a token.  A row is the token's own bit and its parent's row: after k steps it holds the token and the 2^k - 1
// ancestors next to it, and the step adds the row of the ancestor 2^k away, of which there is none once 2^k passes the deepest path.
// Bound: the launch, and the chain first row -> parents -> log2(depth) steps through LDS.  16 sequences of 24 tokens 2.7 us, 48 of up to 200 4.3;
// chains, whose steps are the most, 48 of 200 5.7, 64 of 256 5.8.
template <int WORDS>
__global__ void __launch_bounds__(64 * WORDS) draft_tree_kernel(DraftTreeArgs a)
{
    __shared__ uint64_t rows[WORDS][64 * WORDS];
    __shared__ int ancestors[64 * WORDS];
    const int seq = blockIdx.x, self = threadIdx.x;
    int first = seq * a.max_tokens, count = a.max_tokens;
    if (a.cu_tokens != nullptr) {
        first = min(max(a.cu_tokens[seq], 0), a.tokens);
        count = min(max(a.cu_tokens[seq + 1], first) - first, min(a.max_tokens, a.tokens - first));
    }
    int ancestor = -1;
    uint64_t row[WORDS];
    const int parent = self < count ? a.parents[first + self] : -1;
    const bool placed = parent >= -1 && parent < self;
    if (placed)
        ancestor = parent;
#pragma unroll
    for (int w = 0; w < WORDS; ++w)
        row[w] = placed && self >> 6 == w ? 1ull << (self & 63) : 0ull;
    while (__syncthreads_or(ancestor >= 0)) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
            rows[w][self] = row[w];
        ancestors[self] = ancestor;
        __syncthreads();
        if (ancestor >= 0) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                row[w] |= rows[w][ancestor];
            ancestor = ancestors[ancestor];
        }
    }
    if (self < count)
        for (int w = 0; w < a.words; ++w) {
            uint64_t x = 0;
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                x = i == w ? row[i] : x;
            a.tree[(int64_t)(first + self) * a.words + w] = x;
        }
    if (a.all && a.cu_tokens != nullptr) {  // (each sequence those behind its own, up to the next one's, and the first those before)
        const int end = first + count, next = seq + 1 < (int)gridDim.x ? min(max(a.cu_tokens[seq + 1], end), a.tokens) : a.tokens;
        for (int64_t i = (int64_t)end * a.words + self; i < (int64_t)next * a.words; i += 64 * WORDS)
            a.tree[i] = 0;
        for (int64_t i = self; seq == 0 && i < (int64_t)first * a.words; i += 64 * WORDS)
            a.tree[i] = 0;
    }
}

static int draft_tree(const char* what, uint64_t* tree, int tree_words, const int32_t* parents, int tokens, int sequences, const int32_t* cu_tokens, int max_tokens,
                      bool all, void* stream)
{
    TraceScope trace("DRAFT_TREE", "vector", tokens, sequences, tree_words);
    trace.in(parents, 1, tokens, "ND", PTOAMD_I32).out(tree, tokens, 2L * tree_words, "ND", PTOAMD_I32);
    PTOAMD_REQUIRE(tokens >= 0 && sequences > 0 && max_tokens >= 0, PTOAMD_E_INVALID,
                   "%s: sequences must be positive, tokens and max_tokens not negative (%d, %d, %d)", what, sequences, tokens, max_tokens);
    PTOAMD_REQUIRE(cu_tokens != nullptr || (long)sequences * max_tokens == tokens, PTOAMD_E_INVALID,
                   "%s: without cu_tokens, tokens must be sequences * max_tokens (%d, %d * %d)", what, tokens, sequences, max_tokens);
    if (tokens == 0 || (max_tokens == 0 && !all))
        return PTOAMD_OK;
    const int most = max_tokens < tokens ? max_tokens : tokens;
    PTOAMD_REQUIRE(most <= PTOAMD_MOST_DRAFTED, PTOAMD_E_UNSUPPORTED, "%s: at most %d tokens of a sequence are drafted (%d)", what,
                   PTOAMD_MOST_DRAFTED, most);
    PTOAMD_REQUIRE(tree_words > 0 && tree_words <= PTOAMD_MOST_DRAFTED / 64 && 64 * tree_words >= most, PTOAMD_E_INVALID,
                   "%s: rows of %d words for %d tokens: one for every 64 is needed, at most %d", what, tree_words, most, PTOAMD_MOST_DRAFTED / 64);
    PTOAMD_REQUIRE(tree && parents, PTOAMD_E_INVALID, "%s: null operand", what);
    PTOAMD_REQUIRE(reinterpret_cast<uintptr_t>(tree) % 8 == 0 && reinterpret_cast<uintptr_t>(parents) % 4 == 0, PTOAMD_E_ALIGNMENT,
                   "%s: tree and parents must be aligned to their elements", what);
    const char *rows = reinterpret_cast<const char*>(tree), *rows_end = rows + (size_t)tokens * tree_words * 8;
    auto apart = [&](const int32_t* p, long n) {
        return p == nullptr || rows_end <= reinterpret_cast<const char*>(p) || reinterpret_cast<const char*>(p + n) <= rows;
    };
    PTOAMD_REQUIRE(apart(parents, tokens) && apart(cu_tokens, sequences + 1L), PTOAMD_E_INVALID, "%s: tree must not overlap parents or cu_tokens", what);
    const DraftTreeArgs a{tree, parents, cu_tokens, tree_words, tokens, most, all};
    hipStream_t s = as_stream(stream);
    if (most <= 64)
        hipLaunchKernelGGL(draft_tree_kernel<1>, dim3((unsigned)sequences), dim3(64), 0, s, a);
    else if (most <= 128)
        hipLaunchKernelGGL(draft_tree_kernel<2>, dim3((unsigned)sequences), dim3(128), 0, s, a);
    else
        hipLaunchKernelGGL(draft_tree_kernel<4>, dim3((unsigned)sequences), dim3(256), 0, s, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("draft_tree");
    return PTOAMD_OK;
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

int ptoamd_draft_tree(uint64_t* tree, int tree_words, const int32_t* parents, int tokens, int sequences, const int32_t* cu_tokens, int max_tokens,
                      void* stream)
{
    return draft_tree("ptoamd_draft_tree", tree, tree_words, parents, tokens, sequences, cu_tokens, max_tokens, false, stream);
}

int ptoamd_draft_tree_all(uint64_t* tree, int tree_words, const int32_t* parents, int tokens, int sequences, const int32_t* cu_tokens, int max_tokens,
                          void* stream)
{
    return draft_tree("ptoamd_draft_tree_all", tree, tree_words, parents, tokens, sequences, cu_tokens, max_tokens, true, stream);
}

}  // extern "C"
