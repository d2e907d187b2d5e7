/*
 * heads.cu — rotary positions and the per-head norms of queries and keys (include/aji_b200.h,
 * ajib_rotary_* and ajib_qk_launch).
 *
 * Both are one pass over the queries and keys: 2 bytes read and 2 written per element against a
 * handful of fp32 operations, so memory bandwidth bounds them. A pair (x1, x2) at angle a becomes
 * (x1 cos a - x2 sin a, x2 cos a + x1 sin a); the norm before it is one sum of squares over the
 * head.
 *
 * Angles: position * frequency reaches 1e5 radians and more, where a float holds no useful
 * fraction of a turn. Frequencies are kept as turns per position in 64-bit fixed point, so that the
 * product wraps whole turns off by itself and the top 32 bits are the angle to 2^-32 of a turn
 * (error below position * 2^-65 turns), for negative positions too.
 */
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "f32x2.cuh"
#include "half_types.cuh"
#include "heads.h"

struct ajib_rotary {
    int dim = 0, layout = 0, axes = 1, grid_w = 0, n = 0;
    double freq[ajib::kMaxHeadDim / 2];    // n = dim / 2 / axes angles per position
    uint64_t turns[ajib::kMaxHeadDim / 2]; // the same, in 2^-64 turns
    double amplitude = 1;
};

namespace ajib {

int sm_count();  // conv.cu

namespace {

using dev::from_f;
using dev::to_f;

constexpr int kQkThreads = 128;

struct QkTensor {
    const void *src;
    void *dst;
    int64_t sb, st, sh, ob, ot, oh;
    const float *w;
    int heads;
};

struct QkDev {
    QkTensor t[2];
    const int *pos, *len;
    int64_t pos_sb, slots;
    int pos0, tokens, d, rot, axes, grid_w, interleaved, norm, split, lanes_log2;
    float eps, amplitude, inv_d, inv_eps;
    uint64_t turns[kMaxHeadDim / 2];
};

// What a position's pairs turn by: itself, or its row and column.
struct Place {
    int64_t row, column;
};
__device__ __forceinline__ Place place_of(const QkDev &p, int position)
{
    if (p.axes != 2) return {position, position};
    int row = position / p.grid_w;
    if (position - row * p.grid_w < 0) row--;
    return {row, position - (int64_t)row * p.grid_w};
}

// cos and sin of pair i, times the amplitude. The angle is within half a turn of zero, where the
// hardware's sine and cosine are good to 2^-20.9: 1/1000 of fp16's half step.
__device__ __forceinline__ void pair_angle(const QkDev &p, const Place &at, int i, float &c, float &s)
{
    const int per = p.axes == 2 ? p.rot >> 2 : p.rot >> 1;
    const uint64_t turn = (uint64_t)(i < per ? at.row : at.column) * p.turns[i < per ? i : i - per];
    const float x = (float)(int)(turn >> 32) * (3.14159265358979f * 0x1p-31f);
    asm("cos.approx.ftz.f32 %0, %1;" : "=f"(c) : "f"(x));
    asm("sin.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(x));
    c *= p.amplitude;
    s *= p.amplitude;
}

__device__ __forceinline__ int position_of(const QkDev &p, int b, int t)
{
    return p.pos ? p.pos[b * p.pos_sb + t] : p.pos0 + t;
}

// A sum of squares that left the range of a float (bf16 heads near 1e19 and beyond, or tiny ones with
// next to no eps) is taken again over values times this power of two: 256 of the largest bf16 values
// then sum to 2^104, one of the smallest to 2^-106. 1: the sum will do. (Below 2^-80 against an eps of
// 2^-40 or more the sum does not matter.)
__device__ __forceinline__ float rescale_of(const QkDev &p, float sum)
{
    return sum > 3.4e38f ? 0x1p-80f : sum < 0x1p-80f && p.eps < 0x1p-40f ? 0x1p80f : 1.f;
}

// What a head is multiplied by, from the sum of the squares of its values times scale (rsqrt: 2 ulp). A scale
// above 1 stays in the values, as the factor of the values alone may pass a float's range.
__device__ __forceinline__ float norm_factor(const QkDev &p, float sum, float scale)
{
    const float down = fminf(scale, 1.f);
    if (p.norm == AJIB_NORM_RMS) return down * rsqrtf(sum * p.inv_d + p.eps * scale * scale);
    const float f = down * rsqrtf(sum), most = scale > 1.f ? p.inv_eps * 0x1p-80f : p.inv_eps;
    return f > most ? most : f;  // not fminf, which drops a NaN
}

// One warp per head of one token, any d, alignment and rotary dim: lane l owns pairs l, l + 32, ...
// and the components behind the turned ones. A lane reads the pair it writes, so in place is safe.
template <typename T>
__global__ void __launch_bounds__(kQkThreads) k_qk_any(const __grid_constant__ QkDev p)
{
    const int64_t slot = ((int64_t)blockIdx.x * kQkThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (slot >= p.slots) return;
    const int heads = p.t[0].heads + p.t[1].heads;
    const int64_t bt = slot / heads;
    int h = (int)(slot - bt * heads);
    const int b = (int)(bt / p.tokens), t = (int)(bt - (int64_t)b * p.tokens);
    if (p.len && t >= p.len[b]) return;
    const QkTensor &x = p.t[h >= p.t[0].heads];
    if (h >= p.t[0].heads) h -= p.t[0].heads;
    const T *src = (const T *)x.src + b * x.sb + t * x.st + h * x.sh;
    T *dst = (T *)x.dst + b * x.ob + t * x.ot + h * x.oh;
    float f = 1.f, up = 1.f;
    if (p.norm) {
        float sum, scale = 1.f;
        for (;;) {
            sum = 0.f;
            for (int i = lane; i < p.d; i += 32) {
                const float v = to_f(src[i]) * scale;
                sum += v * v;
            }
            for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if (scale != 1.f || (scale = rescale_of(p, sum)) == 1.f) break;
        }
        f = norm_factor(p, sum, scale);
        up = fmaxf(scale, 1.f);
    }
    const int npair = p.rot >> 1;
    const Place place = place_of(p, p.rot ? position_of(p, b, t) : 0);
    for (int i = lane; i < npair; i += 32) {
        const int i1 = p.interleaved ? 2 * i : i, i2 = p.interleaved ? 2 * i + 1 : i + npair;
        float x1 = to_f(src[i1]) * up * f, x2 = to_f(src[i2]) * up * f, c, s;
        if (x.w) {
            x1 *= x.w[i1];
            x2 *= x.w[i2];
        }
        pair_angle(p, place, i, c, s);
        dst[i1] = from_f<T>(x1 * c - x2 * s);
        dst[i2] = from_f<T>(x2 * c + x1 * s);
    }
    for (int i = p.rot + lane; i < p.d; i += 32) {
        float v = to_f(src[i]) * up * f;
        if (x.w) v *= x.w[i];
        dst[i] = from_f<T>(v);
    }
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 unpack(uint32_t v)
    {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

using dev::F2;
using dev::f2;
using dev::f2_add;
using dev::f2_fma;
using dev::f2_mul;
using dev::f2_out;

// A lane's chunk of CS components, moved by one access.
template <int CS> struct Chunk;
template <> struct Chunk<8> {
    using V = uint4;
};
template <> struct Chunk<4> {
    using V = uint2;
};
template <> struct Chunk<2> {
    using V = uint32_t;
};

// The sum of the squares of a lane's components times scale.
template <int N> __device__ __forceinline__ float sum_squares(const F2 (&a)[N], const F2 (&e)[N], float scale)
{
    const F2 by = f2(scale, scale);
    F2 sum = f2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const F2 x = f2_mul(a[i], by), y = f2_mul(e[i], by);
        sum = f2_fma(x, x, f2_fma(y, y, sum));
    }
    float lo, hi;
    f2_out(sum, lo, hi);
    return lo + hi;
}

template <typename T, int CS> __device__ __forceinline__ typename Chunk<CS>::V pack_chunk(const F2 (&x)[CS / 2])
{
    union {
        uint32_t w[CS / 2];
        typename Chunk<CS>::V v;
    } u;
#pragma unroll
    for (int i = 0; i < CS / 2; i++) {
        float lo, hi;
        f2_out(x[i], lo, hi);
        u.w[i] = Pair<T>::pack(lo, hi);
    }
    return u.v;
}
template <typename T, int CS> __device__ __forceinline__ void unpack_chunk(const typename Chunk<CS>::V &v, F2 (&x)[CS / 2])
{
    union {
        uint32_t w[CS / 2];
        typename Chunk<CS>::V v;
    } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < CS / 2; i++) {
        const float2 f = Pair<T>::unpack(u.w[i]);
        x[i] = f2(f.x, f.y);
    }
}

enum { kTurnNone = 0, kTurnHalf = 1, kTurnInterleaved = 2 };

// A lane holds two chunks of CS components of a head (accesses of 2 CS bytes, neighbouring lanes on
// neighbouring chunks), a power of two of lanes a head. HALF: chunk g of the turned components' first half
// and of their second, so that pairs meet in a lane; otherwise chunk g of a half of what there is, or two
// in a row where that does not divide. A lane computes its CS angles once and walks the heads of its token,
// `split` groups to a token so that small batches fill the machine too. With a norm a head is in
// flight at a time (60 to 72 registers, 7 or 8 blocks an SM: other warps hide the latency of the sum and
// the root), without one two (80 registers, 6 blocks). Measured, one / two heads: norms of 2040 windows
// 171 / 172 us, norms and rotation of 8192 tokens 43.3 / 41.0, rotation alone of 2 x 4999 tokens 42.3 / 38.9,
// of 8 frames of 8160 73.7 / 69.6. (With a norm 44 to 54 % of issue slots and about as much of DRAM: neither is full.)
// WHOLE: every component turns, or none, and the head divides into pairs of chunks, which spares the
// lanes the question (norms and rotation of 8192 tokens 30 M instructions, 49 us, without it).
template <typename T, int CS, bool NORM, int TURN, bool WHOLE>
__global__ void __launch_bounds__(kQkThreads, NORM ? (TURN ? 7 : 8) : 6) k_qk_vec(const __grid_constant__ QkDev p)
{
    using V = typename Chunk<CS>::V;
    constexpr int N = CS / 2;
    const uint32_t slot = (blockIdx.x * kQkThreads + threadIdx.x) >> p.lanes_log2;  // (lanes below 2^32: run_qk)
    const int lanes = 1 << p.lanes_log2, g = threadIdx.x & (lanes - 1);
    const bool there = slot < (uint32_t)p.slots;
    const uint32_t at = there ? slot : (uint32_t)p.slots - 1;
    const uint32_t bt = at / p.split;
    const int h0 = (int)(at - bt * p.split);
    const int b = (int)(bt / p.tokens), t = (int)(bt - (uint32_t)b * p.tokens);
    constexpr bool apart = TURN == kTurnHalf;
    // the part of the head that this lane has chunks of: what turns (HALF), the rest, or all
    const int turned = apart && !WHOLE ? p.rot / (2 * CS) : 0;
    const bool in_turned = WHOLE || g < turned;
    const int from = apart && !in_turned ? p.rot : 0, size = WHOLE ? p.d : in_turned ? p.rot : p.d - from, k = g - (in_turned ? 0 : turned);
    const bool halves = WHOLE || size % (2 * CS) == 0;
    const int c1 = from + (halves ? CS * k : 2 * CS * k), c2 = c1 + (halves ? size >> 1 : CS);
    // lanes of a warp stay together for the sums: what a lane has no part in, it neither reads nor writes
    const bool here = there && !(p.len && t >= p.len[b]);
    const bool live1 = here && c1 < p.d && (!halves || CS * k < size >> 1), live2 = live1 && (WHOLE || c2 < p.d);
    // HALF: c, s, sn = cos, sin, -sin of the chunk's pairs; INTERLEAVED: c, sn = (cos, cos), (-sin, sin) of
    // the first chunk's pairs and s, ce the same of the second's
    F2 c[N], s[N], sn[N], ce[N];
    if (TURN) {
        float co[CS], si[CS];
#pragma unroll
        for (int i = 0; i < CS; i++) co[i] = 1.f, si[i] = 0.f;
        if (live1 && (WHOLE || c1 < p.rot)) {
            const Place place = place_of(p, position_of(p, b, t));
#pragma unroll
            for (int i = 0; i < CS; i++) {
                const int pair = apart ? c1 + i : (i < N ? c1 >> 1 : (c2 >> 1) - N) + i;
                if (WHOLE || 2 * pair < p.rot) pair_angle(p, place, pair, co[i], si[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            c[i] = apart ? f2(co[2 * i], co[2 * i + 1]) : f2(co[i], co[i]);
            s[i] = apart ? f2(si[2 * i], si[2 * i + 1]) : f2(co[N + i], co[N + i]);
            sn[i] = apart ? f2(-si[2 * i], -si[2 * i + 1]) : f2(-si[i], si[i]);
            ce[i] = f2(-si[N + i], si[N + i]);
        }
    }
    const unsigned all = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << ((threadIdx.x & 31) & ~(lanes - 1));
    int h = h0;
    for (int part = 0; part < 2; part++) {
        const QkTensor &q = p.t[part];
        F2 w1[N], w2[N];
        if (NORM) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                w1[i] = w2[i] = f2(1.f, 1.f);
                if (live1 && q.w) w1[i] = f2(__ldg(q.w + c1 + 2 * i), __ldg(q.w + c1 + 2 * i + 1));
                if (live2 && q.w) w2[i] = f2(__ldg(q.w + c2 + 2 * i), __ldg(q.w + c2 + 2 * i + 1));
            }
        }
        const T *src = (const T *)q.src + b * q.sb + t * q.st + h * q.sh;
        T *dst = (T *)q.dst + b * q.ob + t * q.ot + h * q.oh;
        const int64_t step = p.split * q.sh, out_step = p.split * q.oh;
        constexpr int U = NORM ? 1 : 2;  // heads in flight
        for (; h < q.heads; h += U * p.split) {  // (uniform over the lanes of a head)
            V x[U][2];
#pragma unroll
            for (int u = 0; u < U; u++) {
                x[u][0] = x[u][1] = V{};
                if (h + u * p.split < q.heads) {
                    if (live1) x[u][0] = *reinterpret_cast<const V *>(src + u * step + c1);
                    if (live2) x[u][1] = *reinterpret_cast<const V *>(src + u * step + c2);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                F2 a[N], e[N];
                unpack_chunk<T, CS>(x[u][0], a);
                unpack_chunk<T, CS>(x[u][1], e);
                if (NORM) {
                    float sum = sum_squares<N>(a, e, 1.f);
                    for (int m = lanes >> 1; m; m >>= 1) sum += __shfl_xor_sync(all, sum, m);
                    const float scale = rescale_of(p, sum);
                    if (scale != 1.f) {  // (every lane of the head agrees)
                        sum = sum_squares<N>(a, e, scale);
                        for (int m = lanes >> 1; m; m >>= 1) sum += __shfl_xor_sync(all, sum, m);
                        const float up = fmaxf(scale, 1.f);
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            a[i] = f2_mul(a[i], f2(up, up));
                            e[i] = f2_mul(e[i], f2(up, up));
                        }
                    }
                    const float f = norm_factor(p, sum, scale);
                    const F2 ff = f2(f, f);
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        a[i] = f2_mul(f2_mul(a[i], ff), w1[i]);
                        e[i] = f2_mul(f2_mul(e[i], ff), w2[i]);
                    }
                }
                // (what does not turn has angle 0; an infinity or a NaN there meets no partner)
                if (apart) {
                    if (in_turned) {
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            const F2 x1 = a[i], x2 = e[i];
                            a[i] = f2_fma(x1, c[i], f2_mul(x2, sn[i]));
                            e[i] = f2_fma(x2, c[i], f2_mul(x1, s[i]));
                        }
                    }
                } else if (TURN) {
                    // a chunk is x1, x2 pairs
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        float x1, x2, y1, y2;
                        f2_out(a[i], x1, x2);
                        f2_out(e[i], y1, y2);
                        if (WHOLE || c1 < p.rot) a[i] = f2_fma(a[i], c[i], f2_mul(f2(x2, x1), sn[i]));
                        if (WHOLE || c2 < p.rot) e[i] = f2_fma(e[i], s[i], f2_mul(f2(y2, y1), ce[i]));
                    }
                }
                if (h + u * p.split < q.heads) {
                    if (live1) *reinterpret_cast<V *>(dst + u * out_step + c1) = pack_chunk<T, CS>(a);
                    if (live2) *reinterpret_cast<V *>(dst + u * out_step + c2) = pack_chunk<T, CS>(e);
                }
            }
            src += U * step;
            dst += U * out_step;
        }
        // the same walk goes on in the keys: the first place at or behind the last query head
        h = h0 >= q.heads ? h0 - q.heads : (p.split - (q.heads - h0) % p.split) % p.split;
    }
}

template <typename T, int CS, bool WHOLE>
cudaError_t run_vec_form(const QkDev &p, cudaStream_t s)
{
    const unsigned n = (unsigned)(((p.slots << p.lanes_log2) + kQkThreads - 1) / kQkThreads);
    if (!p.rot)
        k_qk_vec<T, CS, true, kTurnNone, WHOLE><<<n, kQkThreads, 0, s>>>(p);
    else if (p.interleaved && p.norm)
        k_qk_vec<T, CS, true, kTurnInterleaved, WHOLE><<<n, kQkThreads, 0, s>>>(p);
    else if (p.interleaved)
        k_qk_vec<T, CS, false, kTurnInterleaved, WHOLE><<<n, kQkThreads, 0, s>>>(p);
    else if (p.norm)
        k_qk_vec<T, CS, true, kTurnHalf, WHOLE><<<n, kQkThreads, 0, s>>>(p);
    else
        k_qk_vec<T, CS, false, kTurnHalf, WHOLE><<<n, kQkThreads, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int CS>
cudaError_t run_vec(const QkDev &p, cudaStream_t s)
{
    const bool whole = (!p.rot || p.rot == p.d) && p.d % (2 * CS) == 0;
    return whole ? run_vec_form<T, CS, true>(p, s) : run_vec_form<T, CS, false>(p, s);
}

// How many lanes of two chunks of cs components a head takes, 0 where it does not divide into them.
int lanes_of(const QkDev &p, int cs, int width)
{
    if (width < 2 * cs || p.d % cs || p.rot % (p.interleaved ? cs : 2 * cs)) return 0;
    const int turned = p.interleaved ? 0 : p.rot, lanes = turned / (2 * cs) + (p.d - turned + 2 * cs - 1) / (2 * cs);
    return lanes <= 32 ? lanes : 0;
}

template <typename T>
cudaError_t run_qk(QkDev &p, int width, int64_t rows, cudaStream_t s)
{
    const int heads = p.t[0].heads + p.t[1].heads;
    for (int cs = p.norm || p.rot ? 8 : 0; cs >= 2; cs >>= 1) {
        const int g = lanes_of(p, cs, width);
        if (!g) continue;
        p.lanes_log2 = 0;
        while (1 << p.lanes_log2 < g) p.lanes_log2++;
        // groups of lanes to a token: one does all its heads once that gives every SM 2048 lanes; a divisor
        // of both head counts, so that no group idles, if one is near (40 heads of 8192 tokens: 4 groups
        // 45.6 us, 5 53.5)
        const int64_t lanes = rows * g, want = (int64_t)sm_count() * 2048;
        p.split = (int)std::min<int64_t>(heads, std::max<int64_t>(1, (want + lanes - 1) / lanes));
        if (p.split < heads)
            for (int s = p.split; 2 * s >= p.split; s--)
                if (p.t[0].heads % s == 0 && p.t[1].heads % s == 0) {
                    p.split = s;
                    break;
                }
        p.slots = rows * p.split;
        if (p.slots << p.lanes_log2 < 1ll << 31)
            return cs == 8 ? run_vec<T, 8>(p, s) : cs == 4 ? run_vec<T, 4>(p, s) : run_vec<T, 2>(p, s);
    }
    p.slots = rows * heads;
    const int64_t blocks = (p.slots * 32 + kQkThreads - 1) / kQkThreads;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    k_qk_any<T><<<(unsigned)blocks, kQkThreads, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace ajib

using namespace ajib;

extern "C" int ajib_rotary_create(const ajib_rotary_params *p, ajib_rotary **out)
{
    if (!out) return AJIB_ERR_ARGS;
    *out = nullptr;
    if (!p || p->dim < 2 || p->dim > kMaxHeadDim || p->dim % 2) return AJIB_ERR_ARGS;
    if (p->layout != AJIB_ROTARY_HALF && p->layout != AJIB_ROTARY_INTERLEAVED) return AJIB_ERR_ARGS;
    if (p->axes != 1 && p->axes != 2) return AJIB_ERR_ARGS;
    if (p->axes == 2 && (p->dim % 4 || p->grid_w < 1)) return AJIB_ERR_ARGS;
    if (p->scaling < AJIB_ROTARY_PLAIN || p->scaling > AJIB_ROTARY_BANDS) return AJIB_ERR_ARGS;
    if (!std::isfinite(p->amplitude) || p->amplitude < 0) return AJIB_ERR_ARGS;
    const int n = p->dim / p->axes;
    const double pi = 3.141592653589793238462643;
    double f[kMaxHeadDim / 2], amp = 1;
    if (p->freq) {
        for (int i = 0; i < n / 2; i++) {
            f[i] = p->freq[i];
            if (!std::isfinite(f[i]) || f[i] < 0) return AJIB_ERR_ARGS;
        }
    } else {
        double base = p->base;
        if (!std::isfinite(base) || base <= 0) return AJIB_ERR_ARGS;
        if (p->scaling != AJIB_ROTARY_PLAIN && (!std::isfinite(p->factor) || p->factor <= 0)) return AJIB_ERR_ARGS;
        if (p->scaling == AJIB_ROTARY_BASE) {
            if (n <= 2) return AJIB_ERR_ARGS;
            base *= std::pow(p->factor, (double)n / (n - 2));
        }
        for (int i = 0; i < n / 2; i++) f[i] = std::pow(base, -2.0 * i / n);
        if (p->scaling == AJIB_ROTARY_LINEAR)
            for (int i = 0; i < n / 2; i++) f[i] /= p->factor;
        if (p->scaling == AJIB_ROTARY_BANDS) {
            const double fast = p->beta_fast == 0 ? 32 : p->beta_fast, slow = p->beta_slow == 0 ? 1 : p->beta_slow;
            if (!std::isfinite(p->trained) || p->trained <= 0 || !std::isfinite(fast) || !std::isfinite(slow) || slow <= 0 || fast < slow ||
                base <= 1)
                return AJIB_ERR_ARGS;
            // the pair whose frequency turns `beta` times over `trained` positions
            auto pair = [&](double beta) { return n * std::log(p->trained / (beta * 2 * pi)) / (2 * std::log(base)); };
            const double lo = std::fmax(std::floor(pair(fast)), 0), hi = std::fmin(std::ceil(pair(slow)), n - 1);
            for (int i = 0; i < n / 2; i++) {
                const double r = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 0.001), 0), 1);
                f[i] = f[i] / p->factor * r + f[i] * (1 - r);
            }
            amp = 0.1 * std::log(p->factor) + 1;
        }
        for (int i = 0; i < n / 2; i++)
            if (!std::isfinite(f[i])) return AJIB_ERR_ARGS;
    }
    if (p->amplitude > 0) amp = p->amplitude;
    if (!(amp > 0) || !std::isfinite((float)amp)) return AJIB_ERR_ARGS;  // (BANDS with a factor below e^-10)
    ajib_rotary *r = new (std::nothrow) ajib_rotary;
    if (!r) return AJIB_ERR_NO_MEM;
    r->dim = p->dim;
    r->layout = p->layout;
    r->axes = p->axes;
    r->grid_w = p->axes == 2 ? p->grid_w : 0;
    r->n = n / 2;
    r->amplitude = amp;
    for (int i = 0; i < n / 2; i++) {
        r->freq[i] = f[i];
        const long double turn = fmodl((long double)f[i] / (2 * 3.14159265358979323846264338327950288L), 1.0L);
        const long double fixed = rintl(ldexpl(turn, 64));
        r->turns[i] = fixed >= ldexpl(1.0L, 64) ? 0 : (uint64_t)fixed;
    }
    *out = r;
    return AJIB_OK;
}

extern "C" void ajib_rotary_release(ajib_rotary **r)
{
    if (!r || !*r) return;
    delete *r;
    *r = nullptr;
}

extern "C" int ajib_rotary_table(const ajib_rotary *r, double *freq, int n, double *amplitude)
{
    if (!r || n < 0) return AJIB_ERR_ARGS;
    for (int i = 0; freq && i < n && i < r->n; i++) freq[i] = r->freq[i];
    if (amplitude) *amplitude = r->amplitude;
    return r->n;
}

extern "C" int ajib_qk_launch(const ajib_qk *op, const ajib_heads *q, const ajib_heads *k, const ajib_heads *q_out,
                              const ajib_heads *k_out, void *stream)
{
    if (!op || (op->dtype != AJIB_F16 && op->dtype != AJIB_BF16)) return AJIB_ERR_ARGS;
    if (op->batch < 0 || op->tokens < 0 || op->hq < 1 || op->hk < 0 || op->d < 1 || op->d > kMaxHeadDim) return AJIB_ERR_ARGS;
    if (op->batch > kMaxCount || op->tokens > kMaxCount || op->hq > kMaxCount || op->hk > kMaxCount) return AJIB_ERR_ARGS;
    if (op->norm < AJIB_NORM_NONE || op->norm > AJIB_NORM_L2 || !(op->eps >= 0) || !std::isfinite(op->eps)) return AJIB_ERR_ARGS;
    if (op->rotary && op->rotary->dim > op->d) return AJIB_ERR_ARGS;
    if (op->pos && (((uintptr_t)op->pos & 3) || op->pos_sb < 0)) return AJIB_ERR_ARGS;
    if (!op->pos && (int64_t)op->pos0 + op->tokens - 1 > 0x7fffffff) return AJIB_ERR_ARGS;
    if (((uintptr_t)op->len & 3) || ((uintptr_t)op->wq & 3) || ((uintptr_t)op->wk & 3)) return AJIB_ERR_ARGS;
    if (!op->batch || !op->tokens) return AJIB_OK;
    const ajib_heads *in[2] = {q, k}, *out[2] = {q_out, k_out};
    const int heads[2] = {op->hq, op->hk};
    QkDev p{};
    int width = 16;
    for (int i = 0; i < 2 && heads[i]; i++) {
        const int b = op->batch, t = op->tokens, h = heads[i];
        if (!heads_ok(in[i], b, t, h, op->d) || !heads_ok(out[i], b, t, h, op->d)) return AJIB_ERR_ARGS;
        if (!heads_distinct(out[i], b, t, h, op->d)) return AJIB_ERR_ARGS;
        if (in[i]->p == out[i]->p && !heads_same(in[i], out[i])) return AJIB_ERR_ARGS;
        if (i && (out[0]->p == out[1]->p || out[0]->p == in[1]->p || out[1]->p == in[0]->p)) return AJIB_ERR_ARGS;
        p.t[i] = {in[i]->p, out[i]->p, in[i]->sb, in[i]->st, in[i]->sh, out[i]->sb, out[i]->st, out[i]->sh,
                  op->norm ? (i ? op->wk : op->wq) : nullptr, h};
        const int w1 = heads_width(in[i], b, t, h, op->d), w2 = heads_width(out[i], b, t, h, op->d);
        width = width < w1 ? width : w1;
        width = width < w2 ? width : w2;
    }
    p.pos = op->pos;
    p.pos_sb = op->pos_sb;
    p.pos0 = op->pos0;
    p.len = op->len;
    p.tokens = op->tokens;
    p.d = op->d;
    p.norm = op->norm;
    p.eps = op->eps;
    p.inv_d = 1.f / op->d;
    p.inv_eps = 1.f / op->eps;  // (eps 0: infinity)
    p.amplitude = 1.f;
    if (const ajib_rotary *r = op->rotary) {
        p.rot = r->dim;
        p.axes = r->axes;
        p.grid_w = r->grid_w;
        p.interleaved = r->layout == AJIB_ROTARY_INTERLEAVED;
        p.amplitude = (float)r->amplitude;
        for (int i = 0; i < r->n; i++) p.turns[i] = r->turns[i];
    }
    const int64_t rows = (int64_t)op->batch * op->tokens;
    const cudaError_t e = op->dtype == AJIB_F16 ? run_qk<__half>(p, width, rows, (cudaStream_t)stream)
                                                : run_qk<__nv_bfloat16>(p, width, rows, (cudaStream_t)stream);
    if (e == cudaErrorInvalidConfiguration) return AJIB_ERR_UNSUPPORTED;
    return e == cudaSuccess ? AJIB_OK : AJIB_ERR_CUDA;
}
