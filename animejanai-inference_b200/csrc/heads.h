/*
 * heads.h — host-side checks of tensors of heads (include/aji_b200.h, ajib_heads), shared by the
 * attention operators.
 */
#pragma once

#include <cstdint>

#include "../../include/aji_b200.h"

namespace ajib {

constexpr int kMaxHeadDim = 256;
constexpr int kMaxCount = 1 << 29;  // batch, tokens and heads: sums of three still fit an int

// An element-aligned pointer, strides that are not negative, and offsets that fit 63 bits.
inline bool heads_ok(const ajib_heads *x, int batch, int tokens, int heads, int d)
{
    if (!x || !x->p || ((uintptr_t)x->p & 1) || x->sb < 0 || x->st < 0 || x->sh < 0) return false;
    const __int128 last = (__int128)(batch - 1) * x->sb + (__int128)(tokens - 1) * x->st +
                          (__int128)(heads - 1) * x->sh + d;
    return last < ((__int128)1 << 60);
}

// Whether all elements are distinct: each stride, taken by size, passes what the smaller ones span.
inline bool heads_distinct(const ajib_heads *x, int batch, int tokens, int heads, int d)
{
    int64_t st[3] = {x->sb, x->st, x->sh};
    int n[3] = {batch, tokens, heads};
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2 - i; j++)
            if (st[j] > st[j + 1]) {
                const int64_t s = st[j];
                st[j] = st[j + 1];
                st[j + 1] = s;
                const int c = n[j];
                n[j] = n[j + 1];
                n[j + 1] = c;
            }
    int64_t span = d;
    for (int i = 0; i < 3; i++) {
        if (n[i] == 1) continue;
        if (st[i] < span) return false;
        span += st[i] * (n[i] - 1);
    }
    return true;
}

inline bool heads_same(const ajib_heads *a, const ajib_heads *b)
{
    return a->p == b->p && a->sb == b->sb && a->st == b->st && a->sh == b->sh;
}

// The widest copy, in bytes, that every row of components allows: 16, 8, 4 or 2. (A stride of a
// dimension of one element is never used.)
inline int heads_width(const ajib_heads *x, int batch, int tokens, int heads, int d)
{
    uint64_t bits = (uint64_t)(uintptr_t)x->p | (uint64_t)d * 2;
    if (batch > 1) bits |= (uint64_t)x->sb * 2;
    if (tokens > 1) bits |= (uint64_t)x->st * 2;
    if (heads > 1) bits |= (uint64_t)x->sh * 2;
    return (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : 2;
}

}  // namespace ajib
