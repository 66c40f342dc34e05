// Whether two operands overlap, for tests on the host.
#include "overlap.hpp"

using namespace ptoamd;

extern "C" int overlap_meet(uint64_t a, const int64_t* x, uint64_t b, const int64_t* y)
{
    return meet(HeadRows{a, x[0], x[1], x[2], x[3], x[4]}, HeadRows{b, y[0], y[1], y[2], y[3], y[4]});
}
