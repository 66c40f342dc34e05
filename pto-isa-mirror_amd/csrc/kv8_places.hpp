// Which keys of a cache a query sees, by places in its sequence: what the attention's kernels index with, and its tests on the host.
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

}  // namespace ptoamd
