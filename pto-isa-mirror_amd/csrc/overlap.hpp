// Whether a call's result overlaps one of its operands, from addresses and strides alone; and its tests on the host.
#pragma once
#include <stdint.h>

namespace ptoamd {

// Rows of heads, in bytes: `heads` pieces of `width` bytes, `head` apart, for each of `tokens` tokens, `token` apart.  A piece of memory is one of them.
struct HeadRows {
    uint64_t at;
    int64_t tokens, heads, token, head, width;
};
inline HeadRows memory_at(const void* p, int64_t bytes) { return HeadRows{(uint64_t)(uintptr_t)p, p != nullptr ? 1 : 0, 1, 0, 0, bytes}; }

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // (b > 0)

// Whether one piece of a and one of b, `delta` apart for the first tokens, share a byte for any two tokens, `token` apart on both sides.
inline bool pieces_meet(int64_t delta, int64_t wide_a, int64_t wide_b, int64_t token, int64_t tokens_a, int64_t tokens_b)
{
    // b's start from a's is delta + d token, d = -(tokens_a - 1) .. tokens_b - 1, and must be in -(wide_b - 1) .. wide_a - 1
    int64_t least = floor_div(-wide_b - delta, token) + 1, most = floor_div(wide_a - 1 - delta, token);
    least = least > -(tokens_a - 1) ? least : -(tokens_a - 1);
    most = most < tokens_b - 1 ? most : tokens_b - 1;
    return least <= most;
}

// Whether a and b share a byte.  Exact where both have the same distances of tokens and of heads (views of one tensor), where one of them is a piece of memory, and where
// heads lie together; of others that have to be looked at element by element, false.
inline bool meet(HeadRows a, HeadRows b)
{
    if (a.tokens <= 0 || a.heads <= 0 || a.width <= 0 || b.tokens <= 0 || b.heads <= 0 || b.width <= 0)
        return false;
    auto range = [](const HeadRows& r, int64_t* from, int64_t* to) {
        const int64_t t = (r.tokens - 1) * r.token, h = (r.heads - 1) * r.head;
        *from = (t < 0 ? t : 0) + (h < 0 ? h : 0);
        *to = (t > 0 ? t : 0) + (h > 0 ? h : 0) + r.width;
    };
    int64_t a0, a1, b0, b1;
    range(a, &a0, &a1);
    range(b, &b0, &b1);
    const int64_t delta = (int64_t)(b.at - a.at);
    if (delta + b0 >= a1 || delta + b1 <= a0)
        return false;
    for (HeadRows* r : {&a, &b}) {
        if (r->heads > 1 && r->head == r->width) {  // together: one piece
            r->width *= r->heads;
            r->heads = 1;
        }
        if (r->heads == 1 && r->tokens > 1 && r->token == r->width) {
            r->width *= r->tokens;
            r->tokens = 1;
        }
    }
    if (a.tokens == 1)
        a.token = b.token;
    if (b.tokens == 1)
        b.token = a.token;
    if (a.heads == 1)
        a.head = b.head;
    if (b.heads == 1)
        b.head = a.head;
    if (a.tokens == 1 && b.tokens == 1)
        a.token = b.token = 1;
    if (a.token != b.token || a.token <= 0 || a.head != b.head)
        return false;
    for (int64_t d = -(a.heads - 1); d <= b.heads - 1; ++d)  // the distance of two heads
        if (pieces_meet(delta + d * a.head, a.width, b.width, a.token, a.tokens, b.tokens))
            return true;
    return false;
}

}  // namespace ptoamd
