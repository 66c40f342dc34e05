// Attention of drafted tokens over an 8-bit cache, many rows.
#include "attention_kv8_many.hpp"

namespace ptoamd {

int launch_attention_tree_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream)
{
    if (f16)
        return code == PTOAMD_I8 ? choose_size<_Float16, PTOAMD_I8, true>(a, sequences, stream) : choose_size<_Float16, PTOAMD_E4M3, true>(a, sequences, stream);
    return code == PTOAMD_I8 ? choose_size<__bf16, PTOAMD_I8, true>(a, sequences, stream) : choose_size<__bf16, PTOAMD_E4M3, true>(a, sequences, stream);
}

}  // namespace ptoamd
