/*
 * attention.cuh — what the attention kernels share: the arguments, which keys a query sees, the
 * score, and the warp's matrix instruction.
 *
 * With scores s_j over the keys a query sees, out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m) for
 * any m; the kernels keep m = the running maximum and rescale sums by e^(m_old - m_new) when it
 * grows, so one pass over keys and values suffices. Exponentials are base 2: scores are kept as
 * s * log2(e), folded into the scale, the cap and the bias.
 */
#pragma once

#include <climits>
#include <cstdint>

#include "../../include/aji_b200.h"
#include "half_types.cuh"

namespace ajib {

struct AttnDev {
    const void *q, *k, *v;
    void *out;
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;
    int batch, lq, lk, hq, hk, group, d;
    float scale, cap_in, cap_out;  // s2 = q.k * scale, or cap_out * tanh(q.k * cap_in)
    int left, right;               // INT_MAX / 2: no limit
    int align_end;
    const int *q_len, *k_len, *prefix, *q_doc, *k_doc;
    int doc_rows, bias;
    const float *bias_data;
    int grid_w, reach_y, reach_x;
    int masked;  // some query may not see some key below its k_len
};

namespace dev {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh to 2^-21 of itself, so that a score far below its cap is as good as one without: up to 0.75 an odd
// polynomial of degree 11 (minimax fit of tanh(x) / x in x^2, relative error 3e-8), above it 1 - 2 / (e^2x + 1),
// which cancels near 0. (A fit up to 1 of that error has degree 13: prompts under a cap 73 us for 70. The
// hardware's tanh.approx is good to 2^-11, which a cap of 50 would turn into 0.02 of score, 2 % of a probability.)
constexpr float kTanhTo = 0.75f;
constexpr float kTanh0 = 0.999999971013924f, kTanh1 = -0.33332958879535546f, kTanh2 = 0.13325406018726102f,
                kTanh3 = -0.05334443020680119f, kTanh4 = 0.01958290833624651f, kTanh5 = -0.004716257367942312f;
__device__ __forceinline__ float tanh_of(float x)
{
    const float z = x * x, far = 1.f - 2.f * rcp_fast(exp2_fast(x * (2.f * kLog2e)) + 1.f);
    const float y = fmaf(fmaf(fmaf(fmaf(fmaf(kTanh5, z, kTanh4), z, kTanh3), z, kTanh2), z, kTanh1), z, kTanh0);
    return fabsf(x) <= kTanhTo ? y * x : far;
}

// How many queries / keys sequence b has.
__device__ __forceinline__ int q_count(const AttnDev &p, int b)
{
    return p.q_len ? min(max(__ldg(p.q_len + b), 0), p.lq) : p.lq;
}
__device__ __forceinline__ int k_count(const AttnDev &p, int b)
{
    return p.k_len ? min(max(__ldg(p.k_len + b), 0), p.lk) : p.lk;
}

// What one query of one head needs to know about every key.
struct Query {
    int at;      // its place
    int lo, hi;  // sees keys lo..hi (both included) and those below pre
    int pre;
    int doc;     // INT_MIN: no documents
    int y, x;    // place on the grid (TABLE)
    float slope; // SLOPE, times log2(e)
    const float *table;
};

__device__ __forceinline__ Query query_at(const AttnDev &p, int doc_row, int h, int i, int shift, int pre)
{
    Query r;
    r.at = i + shift;
    r.lo = p.left == INT_MAX / 2 ? INT_MIN : r.at - p.left;
    r.hi = p.right == INT_MAX / 2 ? INT_MAX : r.at + p.right;
    r.pre = pre;
    r.doc = INT_MIN;
    if (p.q_doc) {
        r.doc = __ldg(p.q_doc + (int64_t)doc_row * p.lq + i);
        if (r.doc < 0) r.lo = INT_MAX, r.hi = -1, r.pre = 0;  // padding sees nothing
    }
    r.y = 0;
    r.x = r.at;
    r.slope = 0.f;
    r.table = nullptr;
    if (p.bias == AJIB_BIAS_SLOPE) r.slope = __ldg(p.bias_data + h) * kLog2e;
    if (p.bias == AJIB_BIAS_TABLE) {
        if (p.grid_w) {
            r.y = r.at / p.grid_w;
            r.x = r.at - r.y * p.grid_w;
        }
        r.table = p.bias_data + (int64_t)h * (2 * p.reach_y + 1) * (2 * p.reach_x + 1);
    }
    return r;
}

__device__ __forceinline__ Query query_of(const AttnDev &p, int b, int h, int i, int qn, int kn)
{
    return query_at(p, p.q_doc ? b % p.doc_rows : 0, h, i, p.align_end ? kn - qn : 0, p.prefix ? max(__ldg(p.prefix + b), 0) : 0);
}

__device__ __forceinline__ bool in_reach(const Query &r, int j) { return j < r.pre || (j >= r.lo && j <= r.hi); }

__device__ __forceinline__ float table_bias(const AttnDev &p, const Query &r, int jy, int jx)
{
    const int dy = min(max(jy - r.y, -p.reach_y), p.reach_y), dx = min(max(jx - r.x, -p.reach_x), p.reach_x);
    return __ldg(r.table + (dy + p.reach_y) * (2 * p.reach_x + 1) + dx + p.reach_x) * kLog2e;
}

// The score of key j times log2(e), from its product with the query.
__device__ __forceinline__ float score2(const AttnDev &p, const Query &r, int j, float dot)
{
    float s = p.cap_out > 0.f ? p.cap_out * tanh_of(dot * p.cap_in) : dot * p.scale;
    if (p.bias == AJIB_BIAS_SLOPE) s -= r.slope * (float)abs(r.at - j);
    if (p.bias == AJIB_BIAS_TABLE) {
        const int jy = p.grid_w ? j / p.grid_w : 0;
        s += table_bias(p, r, jy, j - jy * p.grid_w);
    }
    return s;
}

template <typename T> struct MmaOp;
template <> struct MmaOp<__half> {
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ bool odd(uint32_t x) { return (x & 0x7c00u) == 0x7c00u; }  // not finite
};
template <> struct MmaOp<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ bool odd(uint32_t x) { return (x & 0x7f80u) == 0x7f80u; }
};

}  // namespace dev
}  // namespace ajib
