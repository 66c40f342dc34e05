// What drafted tokens see of each other: rows of bits, as the kernels read them (in 32-bit words), and their tests on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ptoamd.h"
#include "kv8_places.hpp"

namespace ptoamd {

// The n lowest bits, for any n.
__host__ __device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// Bits from .. from + 31 of a row of `words` words; those outside it are 0, `from` may be negative.
__host__ __device__ __forceinline__ uint32_t row_bits(const uint32_t* row, int words, int from)
{
    const int word = from >> 5, shift = from & 31;
    const uint32_t low = (unsigned)word < (unsigned)words ? row[word] : 0u, high = (unsigned)(word + 1) < (unsigned)words ? row[word + 1] : 0u;
    return (uint32_t)((((uint64_t)high << 32) | low) >> shift);
}

// How many of its sequence's `count` drafted tokens the token numbered `self` sees, without itself.
__host__ __device__ __forceinline__ int others_seen(const uint32_t* row, int words, int count, int self)
{
    int n = 0;
    for (int w = 0; w < words; ++w)
        n += __builtin_popcount(row[w] & bits_below(count - 32 * w) & ~(self >> 5 == w ? 1u << (self & 31) : 0u));
    return n;
}

// Which of the keys key .. key + 31 a drafted token sees, in a sequence of `length` tokens of which the first `old` (negative where it has fewer tokens than
// were drafted) are older: those from `first` on of the older ones, and of the others its row's.
__host__ __device__ __forceinline__ uint32_t seen_keys(const uint32_t* row, int words, int key, int first, int old, int length)
{
    return (bits_below(old - key) & ~bits_below(first - key)) | (row_bits(row, words, key - old) & bits_below(length - key));
}
// The same of a row whose bits of tokens that the sequence does not have are 0 already (own_word): no key behind the last has one.
__host__ __device__ __forceinline__ uint32_t seen_by_own(const uint32_t* row, int words, int key, int first, int old)
{
    return (bits_below(old - key) & ~bits_below(first - key)) | row_bits(row, words, key - old);
}
// A row's word without the bits of tokens that a sequence of `count` drafted ones does not have; of a row of `words` words, 0 behind them.
__host__ __device__ __forceinline__ uint32_t own_bits(uint32_t x, int word, int count) { return x & bits_below(count - 32 * word); }
__host__ __device__ __forceinline__ uint32_t own_word(const uint32_t* row, int words, int word, int count)
{
    return word < words ? own_bits(row[word], word, count) : 0u;
}
// The first of the `old` older keys that a window leaves to the token numbered `self`, which stands behind the others that it sees.  (0: no window.)
__host__ __device__ __forceinline__ int first_of_older(const uint32_t* row, int words, int count, int self, int old, int window)
{
    return window > 0 ? first_key(old + others_seen(row, words, count, self), window) : 0;
}

}  // namespace ptoamd
