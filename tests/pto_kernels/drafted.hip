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
extern "C" uint32_t drafted_own_word(const uint32_t* row, int words, int word, int count) { return own_word(row, words, word, count); }
extern "C" uint32_t drafted_seen_by_own(const uint32_t* row, int words, int key, int first, int old) { return seen_by_own(row, words, key, first, old); }
extern "C" int drafted_first_of_older(const uint32_t* row, int words, int count, int self, int old, int window)
{
    return first_of_older(row, words, count, self, old, window);
}
