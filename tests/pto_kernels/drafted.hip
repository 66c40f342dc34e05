// The arithmetic of drafted tokens' rows of bits, for tests on the host.
#include "drafted.hpp"

using namespace ptoamd;

extern "C" uint32_t drafted_bits_below(int n) { return bits_below(n); }
extern "C" uint32_t drafted_row_bits(const uint32_t* row, int words, int from) { return row_bits(row, words, from); }
extern "C" int drafted_others_seen(const uint32_t* row, int words, int count, int self) { return others_seen(row, words, count, self); }
extern "C" uint32_t drafted_seen_keys(const uint32_t* row, int words, int key, int first, int old, int length)
{
    return seen_keys(row, words, key, first, old, length);
}
