/*
 * attention_odd.cuh — rows of attention that came out not finite, once more.
 *
 * The kernels multiply the probabilities of a tile, zeros for the keys that a query does not see, with the
 * tile's values: 0 * v is NaN for a v that is not finite, although the query does not see it. So a row that is
 * not finite may be wrong, but only if such a value stands at a key that the row does not see: unseen_odd looks
 * for one. A value that every row sees (the first key of a causal prompt) leaves its rows not finite
 * rightly, and they are done.
 *
 * Otherwise 16 rows at a time are computed again from the keys that they see alone, in the components that
 * are not finite: a warp walks the keys in chunks of 16 with the same matrix instruction as the kernels', its
 * operands loaded from global memory where they lie (any stride and alignment). Where a chunk holds values that are not finite and not every row sees all of it, the products are
 * taken key by key, for the rows that see it. So a block's work is at most one such pass over its keys, however
 * many rows are not finite, and it is done when no other warp waits for this one with a limit.
 *
 * What bounds it: a warp's own latency, about 3000 cycles a chunk at 128 components and 4500 at 64 (where the
 * kernel has 80 registers), most of it the instructions of one warp and their fetches: a question asked at run time
 * around each load (aligned or not) made it 7000. 8192 causal tokens, 16 heads of 64 / 128, 250 us: with a NaN in
 * the first key 400 / 540 us, in key 4000 800 / 760, in the last 1900 / 1400, with nothing finite behind the first
 * 5.0 / 4.8 ms.
 */
#pragma once

#include "attention.cuh"

namespace ajib {
namespace dev {

// 16 rows from row0 on, of `rows` of a sequence and key head: row = query * group + head - h0.
struct OddRows {
    int b, h0, group, row0, rows, qn, kn;
};

// Whether a key of [j0, j1) that some of the rows may not see holds a value that is not finite: 32 keys
// every `step`. By one warp; lanes are keys, then components of eight keys at a time.
template <typename T> __device__ __forceinline__ bool unseen_odd(const AttnDev &op, const OddRows &r, int j0, int j1, int step)
{
    const AttnDev p = op;  // (a kernel's arguments by address cost a trip to memory each time)
    const int lane = threadIdx.x & 31, end = min(r.row0 + 16, r.rows) - 1, shift = p.align_end ? r.kn - r.qn : 0;
    const int first = r.row0 / r.group, last = end / r.group, pre = p.prefix ? __ldg(p.prefix + r.b) : 0;
    const uint16_t *const v = (const uint16_t *)p.v + r.b * p.vb + (r.h0 / p.group) * p.vh;
    const int *docs = nullptr;
    int doc = INT_MIN;  // the rows' only document
    if (p.q_doc) {
        const int64_t at = r.b % p.doc_rows;
        docs = p.k_doc + at * p.lk;
        const int id = __ldg(p.q_doc + at * p.lq + min(first + lane, last));  // (at most 16 queries)
        const int lo = __reduce_min_sync(0xffffffffu, id), hi = __reduce_max_sync(0xffffffffu, id);
        doc = lo == hi && lo >= 0 ? lo : INT_MIN;
    }
    for (int64_t jt = j0; jt < j1; jt += step) {
        const int j = (int)jt + lane;
        bool all = j < pre || ((p.left == INT_MAX / 2 || j >= last + shift - p.left) &&
                               (p.right == INT_MAX / 2 || j <= first + shift + p.right));
        if (docs) all = all && j < j1 && doc != INT_MIN && __ldg(docs + j) == doc;
        bool odd = false;
        for (uint32_t w = __ballot_sync(0xffffffffu, j < j1 && !all); w;) {
            const uint16_t *row[8];
#pragma unroll
            for (int y = 0; y < 8; y++) {  // (the last one again where there are no eight)
                row[y] = v + ((int)jt + __ffs(w) - 1) * p.vt;
                if (w & (w - 1) || y == 7) w &= w - 1;
            }
            for (int c = lane; c < p.d; c += 32)
#pragma unroll
                for (int y = 0; y < 8; y++) odd |= MmaOp<T>::odd(row[y][c]);
        }
        if (__any_sync(0xffffffffu, odd)) return true;
    }
    return false;
}

// Components c to c + 7 of a row (zeros behind d). WIDE: d is a multiple of 8, and rows are 16-byte aligned.
template <bool WIDE> __device__ __forceinline__ uint4 eight_of(const uint16_t *row, int c, int d)
{
    if constexpr (WIDE) {
        return c < d ? *reinterpret_cast<const uint4 *>(row + c) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int y = 0; y < 4; y++)
            w[y] = (c + 2 * y < d ? row[c + 2 * y] : 0u) | (c + 2 * y + 1 < d ? (uint32_t)row[c + 2 * y + 1] << 16 : 0u);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Where component c of a row is among the outputs of attend_seen: o[n] holds components 64 z + 8 i + y of
// n = 8 z + y, i = 2 (lane % 4) + {0, 1}.
__device__ __forceinline__ int odd_col(int c) { return (c >> 6) * 8 + (c & 7); }
__device__ __forceinline__ int odd_component(int n, int e) { return (n >> 3) * 64 + 8 * (2 * (threadIdx.x & 3) + e) + (n & 7); }

// The rows over the keys that they see of [j0, j1), 16 keys every `step`, by one warp: maximum (base 2), sum and
// unnormalised outputs of rows lane / 4 (o[n][0], [1]) and lane / 4 + 8 ([2], [3]), for the n of `cols`. The
// order of a product's components, and which columns make an operand of eight, are free: so that a lane loads
// eight components in a row at a time.
template <typename T, int DP, bool WIDE>
__device__ __forceinline__ void attend_seen(const AttnDev &op, const OddRows &rows, int j0, int j1, int step, uint32_t cols,
                                            float (&o)[DP / 8][4], float (&m)[2], float (&l)[2])
{
    static_assert(DP % 64 == 0, "");
    constexpr int N = DP / 8;
    const AttnDev p = op;  // (as above)
    const OddRows r = rows;
    const int lane = threadIdx.x & 31, quad = 2 * (lane & 3), g = r.h0 / p.group;
    const uint16_t *const k = (const uint16_t *)p.k + r.b * p.kb + g * p.kh, *const v = (const uint16_t *)p.v + r.b * p.vb + g * p.vh;
    const int *const docs = p.k_doc ? p.k_doc + (int64_t)(r.b % p.doc_rows) * p.lk : nullptr;
    const bool plain = p.bias == AJIB_BIAS_NONE && !(p.cap_out > 0.f);
    // every row sees the keys [whole_lo, whole_hi] and those below whole_pre
    const int shift = p.align_end ? r.kn - r.qn : 0, first = r.row0 / r.group + shift;
    const int last = (min(r.row0 + 16, r.rows) - 1) / r.group + shift, whole_pre = p.prefix ? __ldg(p.prefix + r.b) : 0;
    const int whole_lo = p.left == INT_MAX / 2 ? INT_MIN : last - p.left, whole_hi = p.right == INT_MAX / 2 ? INT_MAX : first + p.right;
    const uint16_t *q[2];
    Query qr[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int row = min(r.row0 + (lane >> 2) + 8 * x, r.rows - 1), i = row / r.group, h = r.h0 + row - i * r.group;
        q[x] = (const uint16_t *)p.q + r.b * p.qb + i * p.qt + h * p.qh;
        qr[x] = query_of(p, r.b, h, i, r.qn, r.kn);
        m[x] = -INFINITY;
        l[x] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < N; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    int64_t kt = p.kt, vt = p.vt;
    int d = p.d, kn = r.kn;
    float scale = p.scale;
    asm volatile("" : "+l"(kt), "+l"(vt), "+r"(d), "+r"(kn), "+f"(scale));
#pragma unroll 1
    for (int64_t jt = j0; jt < j1; jt += step) {
        const int j = (int)jt;
        const bool full = j + 16 <= kn;  // (keys behind the last one: read as the last, no part in anything)
        const bool all = full && !docs && (j + 16 <= whole_pre || (j >= whole_lo && j + 15 <= whole_hi));
        uint32_t sees[2] = {0xffffu, 0xffffu};  // keys of the chunk that this thread's rows see
        if (!all) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                sees[x] = 0u;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int c = 8 * (y >> 1) + quad + (y & 1), key = j + c;
                    if (key < kn && in_reach(qr[x], key) && (!docs || __ldg(docs + key) == qr[x].doc)) sees[x] |= 1u << c;
                }
                sees[x] |= __shfl_xor_sync(0xffffffffu, sees[x], 1);
                sees[x] |= __shfl_xor_sync(0xffffffffu, sees[x], 2);
            }
            if (!__any_sync(0xffffffffu, sees[0] | sees[1])) continue;
        }
        uint4 kw[2][N / 4], vw[4][N / 8];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int key = j + 8 * n + (lane >> 2);
            const uint16_t *row = k + (full ? key : min(key, kn - 1)) * kt;
#pragma unroll
            for (int z = 0; z < N / 4; z++) kw[n][z] = eight_of<WIDE>(row, 32 * z + 4 * quad, d);
        }
        float s[2][4] = {};
#pragma unroll
        for (int z = 0; z < N / 4; z++) {
            const uint4 a = eight_of<WIDE>(q[0], 32 * z + 4 * quad, d), b = eight_of<WIDE>(q[1], 32 * z + 4 * quad, d);
            const uint32_t a0[4] = {a.x, b.x, a.y, b.y}, a1[4] = {a.z, b.z, a.w, b.w};
#pragma unroll
            for (int n = 0; n < 2; n++) {
                MmaOp<T>::mma(s[n], a0, kw[n][z].x, kw[n][z].y);
                MmaOp<T>::mma(s[n], a1, kw[n][z].z, kw[n][z].w);
            }
        }
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int key = j + 8 * (y >> 1) + quad + (y & 1);
            const uint16_t *row = v + (full ? key : min(key, kn - 1)) * vt;
#pragma unroll
            for (int z = 0; z < N / 8; z++)
                vw[y][z] = cols >> 8 * z & 255 && key < kn ? eight_of<WIDE>(row, 64 * z + 8 * (lane >> 2), d) : make_uint4(0, 0, 0, 0);
        }
        if (plain) {
#pragma unroll
            for (int e = 0; e < 8; e++) s[e >> 2][e & 3] *= scale;
        } else {
#pragma unroll 1
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {  // (a table is only read inside it)
                    const float x = score2(p, qr[e >> 1], min(j + 8 * n + quad + (e & 1), kn - 1), n ? s[1][e] : s[0][e]);
                    if (n) s[1][e] = x;
                    else s[0][e] = x;
                }
        }
        if (!all) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (!(sees[e >> 1 & 1] >> (8 * (e >> 2) + quad + (e & 1)) & 1)) s[e >> 2][e & 3] = -INFINITY;
        }
        float alpha[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            float top = fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(top, m[x]);
            const float base = top == -INFINITY ? 0.f : top;
            alpha[x] = exp2_fast(m[x] - base);
            m[x] = top;
            l[x] *= alpha[x];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                float &e = s[y >> 1][2 * x + (y & 1)];
                e = exp2_fast(e - base);
                l[x] += e;
            }
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                o[n][0] *= alpha[0];
                o[n][1] *= alpha[0];
                o[n][2] *= alpha[1];
                o[n][3] *= alpha[1];
            }
        }
        const uint32_t a[4] = {MmaOp<T>::pack(s[0][0], s[0][1]), MmaOp<T>::pack(s[0][2], s[0][3]), MmaOp<T>::pack(s[1][0], s[1][1]),
                               MmaOp<T>::pack(s[1][2], s[1][3])};
#pragma unroll
        for (int n = 0; n < N; n++) {
            if (!(cols >> n & 1)) continue;
            uint32_t w[4];  // component n % 8 of this lane's eight, of its four keys
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const uint4 &x = vw[y][n >> 3];
                const uint32_t two = (n & 6) == 0 ? x.x : (n & 6) == 2 ? x.y : (n & 6) == 4 ? x.z : x.w;
                w[y] = n & 1 ? two >> 16 : two & 0xffffu;
            }
            const bool odd = !all && (MmaOp<T>::odd(w[0]) || MmaOp<T>::odd(w[1]) || MmaOp<T>::odd(w[2]) || MmaOp<T>::odd(w[3]));
            if (all || !__any_sync(0xffffffffu, odd)) {
                MmaOp<T>::mma(o[n], a, w[0] | w[1] << 16, w[2] | w[3] << 16);
                continue;
            }
#pragma unroll 1
            for (int y = 0; y < 16; y++) {
                // probabilities of key j + y, from the lane of the row's four that has it
                const int from = (lane & ~3) | (y & 7) >> 1;
                const float a0 = y < 8 ? (y & 1 ? s[0][1] : s[0][0]) : (y & 1 ? s[1][1] : s[1][0]);
                const float a1 = y < 8 ? (y & 1 ? s[0][3] : s[0][2]) : (y & 1 ? s[1][3] : s[1][2]);
                const float p0 = __shfl_sync(0xffffffffu, a0, from), p1 = __shfl_sync(0xffffffffu, a1, from);
                const T *value = (const T *)v + (j + y) * vt;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int c = odd_component(n, e);
                    if (c >= d) continue;
                    if (sees[0] >> y & 1) o[n][e] = fmaf(p0, to_f(value[c]), o[n][e]);
                    if (sees[1] >> y & 1) o[n][2 + e] = fmaf(p1, to_f(value[c]), o[n][2 + e]);
                }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
}

// Whether queries, keys and values are aligned for WIDE.
__device__ __forceinline__ bool odd_wide(const AttnDev &p)
{
    const uint64_t bits = (uint64_t)(uintptr_t)p.q | (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v |
                          (uint64_t)(p.qb | p.qt | p.qh | p.kb | p.kt | p.kh | p.vb | p.vt | p.vh | p.d) * 2;
    return (bits & 15) == 0;
}

// The rows whose outputs, which are written already, are not finite: again where it takes that, over the keys
// [j0, j1). By one warp.
template <typename T, int DP> __device__ __forceinline__ void redo_rows(const AttnDev &p, const OddRows &r, int j0, int j1)
{
    const int lane = threadIdx.x & 31;
    uint32_t cols = 0;
    {
        // two lanes a row, every second component
        const int row = r.row0 + (lane >> 1), i = row / r.group;
        const uint16_t *const x = (const uint16_t *)p.out + r.b * p.ob + i * p.ot + (r.h0 + row - i * r.group) * p.oh;
        if (row < r.rows) {
#pragma unroll 8
            for (int c = lane & 1; c < p.d; c += 2)
                if (MmaOp<T>::odd(x[c])) cols |= 1u << odd_col(c);
        }
    }
    const uint32_t which = __ballot_sync(0xffffffffu, cols != 0);  // rows, two bits each
    cols = __reduce_or_sync(0xffffffffu, cols);
    if (!which || !unseen_odd<T>(p, r, j0, j1, 32)) return;
    constexpr int N = DP < 64 ? 64 : DP;
    float o[N / 8][4], m[2], l[2];
    if (odd_wide(p))
        attend_seen<T, N, true>(p, r, j0, j1, 16, cols, o, m, l);
    else
        attend_seen<T, N, false>(p, r, j0, j1, 16, cols, o, m, l);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int at = (lane >> 2) + 8 * x, row = r.row0 + at, i = row / r.group;
        if (row >= r.rows || !(which >> (2 * at) & 3)) continue;
        T *dst = (T *)p.out + r.b * p.ob + i * p.ot + (r.h0 + row - i * r.group) * p.oh;
        const float f = l[x] == 0.f ? 0.f : 1.f / l[x];
#pragma unroll
        for (int n = 0; n < N / 8; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = odd_component(n, e);
                if (cols >> n & 1 && c < p.d) dst[c] = from_f<T>(l[x] == 0.f ? 0.f : o[n][2 * x + e] * f);
            }
    }
}

// This warp's share of the rows' keys (16 of every 64) to the memory that join_warps joins: maxima, sums, outputs.
template <typename T, int DP>
__device__ __forceinline__ void redo_share(const AttnDev &p, const OddRows &r, int j0, int j1, float *jm, float *jl, float *jo)
{
    const int lane = threadIdx.x & 31;
    constexpr int N = DP < 64 ? 64 : DP;
    float o[N / 8][4], m[2], l[2];
    if (odd_wide(p))
        attend_seen<T, N, true>(p, r, j0, j1, 64, 0xffffffffu, o, m, l);
    else
        attend_seen<T, N, false>(p, r, j0, j1, 64, 0xffffffffu, o, m, l);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int at = (lane >> 2) + 8 * x;
        if ((lane & 3) == 0) {
            jm[at] = m[x];
            jl[at] = l[x];
        }
#pragma unroll
        for (int n = 0; n < N / 8; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = odd_component(n, e);
                if (c < p.d) jo[at * DP + c] = o[n][2 * x + e];
            }
    }
}

// A vote of the n threads of named barrier `id`.
__device__ __forceinline__ bool named_bar_any(int id, int n, bool yes)
{
    uint32_t r;
    asm volatile("{\n.reg .pred a, b;\nsetp.ne.u32 a, %1, 0;\nbarrier.cta.red.or.pred b, %2, %3, a;\nselp.u32 %0, 1, 0, b;\n}"
                 : "=r"(r)
                 : "r"((uint32_t)yes), "r"(id), "r"(n)
                 : "memory");
    return r != 0;
}

}  // namespace dev
}  // namespace ajib
