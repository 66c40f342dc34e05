// The arithmetic of places and windows that the attention over an 8-bit cache indexes with, for tests on the host.
#include "kv8_places.hpp"

using namespace ptoamd;

extern "C" int kv8_first_key(int place, int window) { return first_key(place, window); }
extern "C" void kv8_keys_of(int place, int length, int causal, int window, int* first, int* end)
{
    const int2 keys = keys_of(place, length, causal != 0, window);
    *first = keys.x;
    *end = keys.y;
}
extern "C" int kv8_pages_of(int tokens, int page_shift) { return pages_of(tokens, page_shift); }
