// Which keys of a cache a query sees, by places in its sequence: what the kernels around the cache index with, and their tests on the host.
#pragma once
#include <hip/hip_runtime.h>

namespace ptoamd {

// The first key that a window leaves to the query at `place`, which is negative before the sequence's first token, down to -(2^31 - 1).  Compared
// before it is subtracted: place + 1 - window of a window of up to 2^31 - 1 does not fit 32 bits, and wrapped would be a key far behind the last.
__host__ __device__ __forceinline__ int first_key(int place, int window) { return window > 0 && place + 1 > window ? place + 1 - window : 0; }
// The keys that the query at `place` of a sequence of `length` tokens sees: [x, y).
__host__ __device__ __forceinline__ int2 keys_of(int place, int length, bool causal, int window)
{
    const int behind = place + 1 < 0 ? 0 : place + 1, last = causal && behind < length ? behind : length, first = first_key(place, window);
    return make_int2(first, last > first ? last : first);
}

// The most pages that so many consecutive tokens lie in, wherever the first is; tokens > 0, up to 2^31 - 1.
__host__ __device__ __forceinline__ int pages_of(int tokens, int page_shift)
{
    return ((tokens - 1) >> page_shift) + (((tokens - 1) & ((1 << page_shift) - 1)) != 0) + 1;
}

}  // namespace ptoamd
