// Attention over an 8-bit cache for many queries: prompts and chunks of prompts.
#include "attention_kv8_many.hpp"

namespace ptoamd {

int launch_attention_many(const AttentionArgs& a, int code, bool f16, int sequences, hipStream_t stream)
{
    if (f16)
        return code == PTOAMD_I8 ? choose_size<_Float16, PTOAMD_I8, false>(a, sequences, stream) : choose_size<_Float16, PTOAMD_E4M3, false>(a, sequences, stream);
    return code == PTOAMD_I8 ? choose_size<__bf16, PTOAMD_I8, false>(a, sequences, stream) : choose_size<__bf16, PTOAMD_E4M3, false>(a, sequences, stream);
}

}  // namespace ptoamd
