// Rotary positions: the table of rotations, and the rotation of queries and keys (and of gradients back).
#include <math.h>

#include "common_host.hpp"

namespace ptoamd {

// One angle a thread, in 64 bits: at position 100 000 a frequency of 1 leaves a product in 32 bits off by up to 4e-3, as much as a bf16
// result may be.  The table is made once and costs nothing later.
__global__ void __launch_bounds__(256) rope_table_kernel(float* table, int rows, int half, double log_base, double factor, double low, double high,
                                                         double magnitude)
{
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long)rows * half)
        return;
    const long p = at / half;
    const int i = (int)(at - p * half);
    const double f = exp(-log_base * i / half);  // base^(-2 i / rot_dim)
    const double t = i >= high ? 1.0 : i <= low ? 0.0 : (i - low) / (high - low);
    double sine, cosine;
    sincos((double)p * (f * (1.0 - t) + f * t / factor), &sine, &cosine);
    table[p * 2 * half + i] = (float)(cosine * magnitude);
    table[p * 2 * half + half + i] = (float)(sine * magnitude);
}

struct RopeArgs {
    uint8_t* out;
    const uint8_t* x;
    const float* table;
    const int32_t* positions;
    int64_t x_token, x_head, out_token, out_head;  // bytes
    int table_rows, tokens, heads, head_dim, half;
    int turned, units;  // of a head: units that turn VEC pairs, and all units; the others copy 2 VEC elements
    float sign;         // of the sines: -1 turns a gradient back
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RopeVec {
    T e[VEC];
};

constexpr int ROPE_TOKENS = 2;

// A unit is VEC pairs of one head: two vectors of VEC elements, half a rotation apart or, interleaved, next to each other.  A thread
// has the same unit of two consecutive tokens, all loads of both in flight before the first is used (8192 tokens of 40 heads of 128, bf16:
// one token a thread 36.3 us, two 33.3, four, whose registers take waves off the CUs, 38.2).  A token's rotations are read again for every head,
// from the L1 after the first.  Products and sums in f32, one rounding.
// Bound: HBM, what is turned in once and out once: 172 MB in 33.3 us, 5.2 TB/s, as a large copy.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(512) rope_kernel(RopeArgs a)
{
    typedef RopeVec<T, VEC> Vec;
    constexpr int TOKENS = ROPE_TOKENS;
    const int unit = blockIdx.y * blockDim.x + threadIdx.x;
    const int first = blockIdx.x * TOKENS;
    if (unit >= a.units * a.heads)
        return;
    const int head = unit / a.units, u = unit - head * a.units;
    const bool turns = u < a.turned;
    const int pair = u * VEC;
    const int lo = turns ? (INTERLEAVED ? 2 * pair : pair) : 2 * a.half + (u - a.turned) * 2 * VEC;
    const int end = turns && !INTERLEAVED ? pair + a.half : lo + VEC;
    const int hi = VEC == 1 && end == a.head_dim ? lo : end;  // (an odd element is left over after the pairs: it is its own neighbour)
    Vec x[TOKENS][2];
    float cosine[TOKENS][VEC], sine[TOKENS][VEC];
    int at[TOKENS];
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
        at[k] = a.positions[min(first + k, a.tokens - 1)];
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
        const T* row = reinterpret_cast<const T*>(a.x + (int64_t)min(first + k, a.tokens - 1) * a.x_token + (int64_t)head * a.x_head);
        x[k][0] = *reinterpret_cast<const Vec*>(row + lo);
        x[k][1] = *reinterpret_cast<const Vec*>(row + hi);
    }
    if (turns) {
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const bool known = (unsigned)at[k] < (unsigned)a.table_rows;
            const float* turn = a.table + (int64_t)(known ? at[k] : 0) * 2 * a.half + pair;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                cosine[k][j] = turn[j];
                sine[k][j] = turn[a.half + j];
            }
        }
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const float unknown = (unsigned)at[k] < (unsigned)a.table_rows ? 0.0f : NAN;
            Vec y[2];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float c = cosine[k][j] + unknown, s = fmaf(sine[k][j], a.sign, unknown);
                // the pair's two elements: the j-th of both vectors, or neighbours
                const int v0 = INTERLEAVED ? (2 * j) / VEC : 0, e0 = INTERLEAVED ? (2 * j) % VEC : j;
                const int v1 = INTERLEAVED ? (2 * j + 1) / VEC : 1, e1 = INTERLEAVED ? (2 * j + 1) % VEC : j;
                const float p = (float)x[k][v0].e[e0], q = (float)x[k][v1].e[e1];
                y[v0].e[e0] = (T)(p * c - q * s);
                y[v1].e[e1] = (T)(p * s + q * c);
            }
            x[k][0] = y[0];
            x[k][1] = y[1];
        }
    }
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
        if (first + k >= a.tokens)
            break;
        T* row = reinterpret_cast<T*>(a.out + (int64_t)(first + k) * a.out_token + (int64_t)head * a.out_head);
        *reinterpret_cast<Vec*>(row + lo) = x[k][0];
        *reinterpret_cast<Vec*>(row + hi) = x[k][1];
    }
}

template <typename T, int VEC, bool INTERLEAVED>
static int launch_rope(const RopeArgs& a, hipStream_t stream)
{
    const long units = (long)a.units * a.heads;
    const long wide = (units + 511) / 512;
    const int block = (int)(((units + wide - 1) / wide + 63) / 64 * 64);
    hipLaunchKernelGGL((rope_kernel<T, VEC, INTERLEAVED>), dim3((unsigned)((a.tokens + ROPE_TOKENS - 1) / ROPE_TOKENS), (unsigned)wide), dim3(block), 0, stream, a);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("rope");
    return PTOAMD_OK;
}

// Vectors of 16 bytes where halves, rests and rows allow it, else of 8, else single elements.
template <typename T>
static int dispatch_rope(RopeArgs a, bool interleaved, hipStream_t stream)
{
    uint64_t bits = (uint64_t)(uintptr_t)a.x | (uint64_t)(uintptr_t)a.out | (uint64_t)a.x_token | (uint64_t)a.x_head | (uint64_t)a.out_token | (uint64_t)a.out_head;
    auto fits = [&](int vec) {
        return a.half % vec == 0 && (a.head_dim - 2 * a.half) % (2 * vec) == 0 && bits % (vec * sizeof(T)) == 0;
    };
    constexpr int WIDE = 16 / (int)sizeof(T), NARROW = 8 / (int)sizeof(T);
    const int vec = fits(WIDE) ? WIDE : fits(NARROW) ? NARROW : 1;
    a.turned = a.half / vec;
    a.units = a.turned + (a.head_dim - 2 * a.half + 2 * vec - 1) / (2 * vec);
    if (vec == WIDE)
        return interleaved ? launch_rope<T, WIDE, true>(a, stream) : launch_rope<T, WIDE, false>(a, stream);
    if (vec == NARROW)
        return interleaved ? launch_rope<T, NARROW, true>(a, stream) : launch_rope<T, NARROW, false>(a, stream);
    return interleaved ? launch_rope<T, 1, true>(a, stream) : launch_rope<T, 1, false>(a, stream);
}

}  // namespace ptoamd

using namespace ptoamd;

extern "C" {

int ptoamd_rope_table(float* table, int rows, int rot_dim, double base, double factor, double ramp_low, double ramp_high, double magnitude,
                      void* stream)
{
    TraceScope trace("ROPE_TABLE", "vector", rows, rot_dim, 0);
    trace.out(table, rows, rot_dim, "ND", PTOAMD_F32);
    PTOAMD_REQUIRE(table != nullptr, PTOAMD_E_INVALID, "ptoamd_rope_table: null operand");
    PTOAMD_REQUIRE(rows > 0 && rot_dim > 0 && rot_dim % 2 == 0, PTOAMD_E_INVALID, "ptoamd_rope_table: rows must be positive, rot_dim positive and even (%d, %d)",
                   rows, rot_dim);
    PTOAMD_REQUIRE(base > 0 && factor > 0 && isfinite(base) && isfinite(factor) && isfinite(magnitude), PTOAMD_E_INVALID,
                   "ptoamd_rope_table: base and factor must be positive, and finite like the magnitude");
    PTOAMD_REQUIRE(ramp_low <= ramp_high, PTOAMD_E_INVALID, "ptoamd_rope_table: ramp_low must not be above ramp_high");
    const long blocks = ((long)rows * (rot_dim / 2) + 255) / 256;
    PTOAMD_REQUIRE(blocks <= 0x7FFFFFFF, PTOAMD_E_UNSUPPORTED, "ptoamd_rope_table: %d rows of %d elements are too many for one launch", rows, rot_dim);
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), table, rows, rot_dim / 2, log(base), factor, ramp_low,
                       ramp_high, magnitude);
    PTOAMD_HIP_CHECK(hipGetLastError());
    set_last_kernel("rope_table");
    return PTOAMD_OK;
}

int ptoamd_rope(void* out, const void* x, int type, const float* table, int table_rows, const int32_t* positions, int tokens, int heads,
                int head_dim, int rot_dim, int64_t x_token_stride, int64_t x_head_stride, int64_t out_token_stride, int64_t out_head_stride,
                int interleaved, int backward, void* stream)
{
    TraceScope trace(backward ? "ROPE_BACKWARD" : "ROPE", "vector", tokens, heads, head_dim);
    trace.in(x, tokens, (long)heads * head_dim, "ND", type).in(table, table_rows, rot_dim, "ND", PTOAMD_F32)
        .out(out, tokens, (long)heads * head_dim, "ND", type);
    PTOAMD_REQUIRE(tokens >= 0 && heads > 0 && head_dim > 0 && table_rows > 0, PTOAMD_E_INVALID,
                   "ptoamd_rope: heads, head_dim and table_rows must be positive, tokens not negative (%d, %d, %d, %d)", heads, head_dim, table_rows, tokens);
    PTOAMD_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, PTOAMD_E_INVALID,
                   "ptoamd_rope: rot_dim must be even and at most head_dim (%d of %d)", rot_dim, head_dim);
    PTOAMD_REQUIRE(type == PTOAMD_F32 || type == PTOAMD_F16 || type == PTOAMD_BF16, PTOAMD_E_UNSUPPORTED, "ptoamd_rope: the type must be f32, f16 or bf16");
    PTOAMD_REQUIRE((long)heads * head_dim <= 1 << 24, PTOAMD_E_UNSUPPORTED, "ptoamd_rope: %d heads of %d elements are too many", heads, head_dim);
    if (tokens == 0)
        return PTOAMD_OK;
    PTOAMD_REQUIRE(out && x && table && positions, PTOAMD_E_INVALID, "ptoamd_rope: null operand");
    const int size = type == PTOAMD_F32 ? 4 : 2;
    PTOAMD_REQUIRE((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(x)) % size == 0, PTOAMD_E_ALIGNMENT,
                   "ptoamd_rope: x and out must be aligned to their elements");
    PTOAMD_REQUIRE(out != x || (x_token_stride == out_token_stride && x_head_stride == out_head_stride), PTOAMD_E_INVALID,
                   "ptoamd_rope: in place, out must have the strides of x");
    RopeArgs a{};
    a.out = static_cast<uint8_t*>(out);
    a.x = static_cast<const uint8_t*>(x);
    a.table = table;
    a.positions = positions;
    a.x_token = x_token_stride * size;
    a.x_head = x_head_stride * size;
    a.out_token = out_token_stride * size;
    a.out_head = out_head_stride * size;
    a.table_rows = table_rows;
    a.tokens = tokens;
    a.heads = heads;
    a.head_dim = head_dim;
    a.half = rot_dim / 2;
    a.sign = backward ? -1.0f : 1.0f;
    hipStream_t s = as_stream(stream);
    switch (type) {
        case PTOAMD_F32: return dispatch_rope<float>(a, interleaved != 0, s);
        case PTOAMD_F16: return dispatch_rope<_Float16>(a, interleaved != 0, s);
        default: return dispatch_rope<__bf16>(a, interleaved != 0, s);
    }
}

}  // extern "C"
