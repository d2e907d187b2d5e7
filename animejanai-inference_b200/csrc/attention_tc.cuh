/*
 * attention_tc.cuh — attention of long prompts on the fifth-generation tensor cores (tcgen05).
 *
 * A block takes 256 queries of one head as two tiles of 128 and walks the keys in tiles of 128.
 * Warps 0-3 and 4-7 do the softmax of one query tile each (a thread a row), warp 8 issues the TMA
 * copies, warp 9 the matrix products:
 *   S_q = Q_q K^T   (both from shared memory)       -> TMEM, 128 columns each
 *   O_q += P_q V    (P from TMEM, V from shared)    -> TMEM, DP columns each
 * P_q takes the columns of S_q: a thread holds its whole row of scores in registers before it writes
 * probabilities back, so TMEM's 512 columns hold both tiles at 128 components. The products are
 * issued P0 V, S0', P1 V, S1': while one tile's softmax runs, the other tile's products do.
 *
 * The running maximum a row is scaled by only follows the true one when that has grown by more than
 * 2^8: the accumulators are rescaled rarely, and by the softmax threads themselves, at a time when
 * no product touches them. Probabilities are then up to 2^8 instead of 1, which costs neither fp16
 * nor bf16 any precision.
 *
 * What bounds it: per 256 x 128 scores the tensor pipe needs 32 * DP cycles (8192 flop a cycle)
 * and the exponentials 2048 (16 a cycle): even at DP 128, exponentials at 64.
 */
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention_mma.cuh"

namespace ajib {

constexpr int kTcThreads = 384, kTcKeys = 128;

struct TcDev {
    AttnDev a;
    int tiles;      // of 256 queries a head
    int bias_form;  // kBiasNone, kBiasSlope or kBiasLine
    int scaled;     // scores are scaled before the maximum (cap, bias, or a scale that is not positive)
    int wo;         // widest copies (bytes) of out
    int *err;
};

template <int DP> struct TcCfg {
    static constexpr int ST = DP == 128 ? 2 : 4;       // stages of keys and of values
    static constexpr int TILE = 128 * DP * 2;          // a tile of queries, keys or values
    static constexpr int Q = 0, K = 2 * TILE, V = K + ST * TILE, SCRATCH = V + ST * TILE;
    static constexpr int BARS = SCRATCH + 8 * 256 * 4;  // attend_row's queries, a warp each
    static constexpr int NBAR = 2 + 4 * ST + 6;
    static constexpr int BITS = BARS + NBAR * 8 + 16;
    // bits: four words (seen and whole, of both query tiles) for every 32 key tiles
    static int smem(const AttnDev &p)
    {
        const int words = p.q_doc ? (p.lk + kTcKeys * 32 - 1) / (kTcKeys * 32) : 0;
        return BITS + words * 16 + 1024;  // + the alignment of the first tile
    }
};

namespace dev {

// K-major tiles of 64 components a row (128 bytes) as TMA writes them with the 128-byte swizzle:
// 8-row groups 1024 bytes apart. The same tile read as a B operand whose rows are k (values: k =
// keys, n = components) is MN-major: 64 n by 8 k a group, groups along k 1024 bytes apart, blocks
// of 64 n a tile apart (lbo).
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t saddr, uint32_t lbo)
{
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
template <typename T> __host__ __device__ constexpr uint32_t idesc_of(int N, bool b_mn)
{
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v)
{
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// The lowest n bits of a word, n of any sign or size.
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

template <typename T, int DP>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_attn_tc(const __grid_constant__ TcDev P, const __grid_constant__ CUtensorMap mq,
              const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv)
{
    using C = TcCfg<DP>;
    const AttnDev &p = P.a;
    extern __shared__ char sm_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- which queries and keys (the last queries of a prompt, which see most, first) ----
    const int64_t bhs = (int64_t)p.batch * p.hq;
    const int tile = P.tiles - 1 - (int)(blockIdx.x / bhs);
    const int bh = (int)(blockIdx.x % bhs), b = bh / p.hq, h = bh - b * p.hq;
    const int qn = q_count(p, b), kn = k_count(p, b), row0 = tile * 256;
    if (row0 >= qn) return;
    const int shift = p.align_end ? kn - qn : 0;
    const int pre = p.prefix ? __ldg(p.prefix + b) : 0;
    const int first0 = row0 + shift, last1 = min(row0 + 256, qn) - 1 + shift;
    int key_lo, key_hi;
    reach_of(p, first0, last1, pre, kn, key_lo, key_hi);
    const int t0 = key_lo / kTcKeys, t1 = (max(key_hi, key_lo) + kTcKeys - 1) / kTcKeys;
    const bool both = row0 + 128 < qn;
    const int last0 = both ? first0 + 127 : last1, first1 = first0 + 128;

    char *const sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
    const uint32_t s0 = smem_u32(sm);
    const uint32_t bars = s0 + C::BARS;
    const uint32_t q_full = bars, k_full = bars + 16, k_empty = k_full + 8 * C::ST, v_full = k_empty + 8 * C::ST,
                   v_empty = v_full + 8 * C::ST, s_full = v_empty + 8 * C::ST, p_full = s_full + 16, o_full = p_full + 16;
    uint32_t *const tmem_at = (uint32_t *)(sm + C::BARS + C::NBAR * 8);
    uint32_t *const bits = (uint32_t *)(sm + C::BITS);

    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_at), 512);
    } else if (tid == 256) {
        tma_prefetch_desc(&mq);
        tma_prefetch_desc(&mk);
        tma_prefetch_desc(&mv);
        for (int i = 0; i < C::NBAR - 6; i++) mbar_init(bars + 8 * i, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);  // one arrival a softmax warp
            mbar_init(o_full + 8 * i, 1);
        }
        fence_mbar_init();
    }
    const int *const docs = p.k_doc ? p.k_doc + (int64_t)(b % p.doc_rows) * p.lk : nullptr;
    const int word0 = t0 / 32;
    if (docs) {
        // which key tiles hold a document of each query tile, and which nothing but its only one
        const int *qd = p.q_doc + (int64_t)(b % p.doc_rows) * p.lq;
        int lo[2] = {INT_MAX, INT_MAX}, hi[2] = {INT_MIN, INT_MIN};
#pragma unroll
        for (int x = 0; x < 2; x++) {
            for (int i = row0 + 128 * x + lane; i < min(row0 + 128 * x + 128, qn); i += 32) {
                const int id = __ldg(qd + i);
                lo[x] = min(lo[x], id);
                hi[x] = max(hi[x], id);
            }
            lo[x] = __reduce_min_sync(0xffffffffu, lo[x]);
            hi[x] = __reduce_max_sync(0xffffffffu, hi[x]);
        }
        for (int w = word0 + warp; w * 32 < t1; w += kTcThreads / 32) {
            int klo = INT_MAX, khi = INT_MIN;
            // the warp reads a tile together, lane l keeps tile l's range
            for (int x = 0; x < 32; x++) {
                const int t = w * 32 + x;
                if (t < t0 || t >= t1) continue;
                int a = INT_MAX, z = INT_MIN;
#pragma unroll
                for (int y = 0; y < kTcKeys / 32; y++) {
                    const int j = t * kTcKeys + y * 32 + lane;
                    if (j < kn) {
                        const int id = __ldg(docs + j);
                        a = min(a, id);
                        z = max(z, id);
                    }
                }
                a = __reduce_min_sync(0xffffffffu, a);
                z = __reduce_max_sync(0xffffffffu, z);
                if (lane == x) klo = a, khi = z;
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t seen = __ballot_sync(0xffffffffu, khi >= 0 && max(lo[x], 0) <= khi && klo <= hi[x]);
                const uint32_t whole = __ballot_sync(0xffffffffu, lo[x] >= 0 && lo[x] == hi[x] && klo == lo[x] && khi == lo[x]);
                if (lane == 0) {
                    bits[4 * (w - word0) + x] = seen;
                    bits[4 * (w - word0) + 2 + x] = whole;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;

    const bool no_left = p.left == INT_MAX / 2, no_right = p.right == INT_MAX / 2;
    // Whether some query of tile q sees a key of tile t, and whether every one sees all of them.
    auto active = [&](int q, int t) {
        const int j = t * kTcKeys;
        if ((q && !both) || j >= kn) return false;
        if (docs && !(bits[4 * (t / 32 - word0) + q] >> (t & 31) & 1)) return false;
        return j < pre || ((no_left || j + kTcKeys - 1 >= (q ? first1 : first0) - p.left) &&
                           (no_right || j <= (q ? last1 : last0) + p.right));
    };
    auto whole = [&](int q, int t) {
        const int j = t * kTcKeys, end = j + kTcKeys;
        if (end > kn) return false;
        if (docs && !(bits[4 * (t / 32 - word0) + 2 + q] >> (t & 31) & 1)) return false;
        return end <= pre || ((no_left || j >= (q ? last1 : last0) - p.left) &&
                              (no_right || end - 1 <= (q ? first1 : first0) + p.right));
    };

    // 384 threads of 168 registers: the softmax warps take 216 (a row of 128 scores and more), 72 stay
    // for the copies, the products and two idle warps.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---- copies ----
            if (lane == 0) {
                const int g = h / p.group;
                int n = 0;
                bool ok = true;
                for (int t = t0; t < t1 && ok; t++) {
                    if (!active(0, t) && !active(1, t)) continue;
                    const int st = n % C::ST;
                    const uint32_t parity = ((n / C::ST) & 1) ^ 1;
                    if (n == 0) {
                        mbar_arrive_expect_tx(q_full, C::TILE);
                        for (int x = 0; x < DP / 64; x++) tma_load_4d(s0 + C::Q + x * 16384, &mq, q_full, 64 * x, row0, h, b);
                    }
                    if (!(ok = mbar_wait(k_empty + 8 * st, parity, P.err, 201))) break;
                    mbar_arrive_expect_tx(k_full + 8 * st, C::TILE);
                    for (int x = 0; x < DP / 64; x++)
                        tma_load_4d(s0 + C::K + st * C::TILE + x * 16384, &mk, k_full + 8 * st, 64 * x, t * kTcKeys, g, b);
                    if (n == 0 && both) {
                        mbar_arrive_expect_tx(q_full + 8, C::TILE);
                        for (int x = 0; x < DP / 64; x++)
                            tma_load_4d(s0 + C::Q + C::TILE + x * 16384, &mq, q_full + 8, 64 * x, row0 + 128, h, b);
                    }
                    if (!(ok = mbar_wait(v_empty + 8 * st, parity, P.err, 202))) {
                        n++;
                        break;
                    }
                    mbar_arrive_expect_tx(v_full + 8 * st, C::TILE);
                    for (int x = 0; x < DP / 64; x++)
                        tma_load_4d(s0 + C::V + st * C::TILE + x * 16384, &mv, v_full + 8 * st, 64 * x, t * kTcKeys, g, b);
                    n++;
                }
                // every copy has landed before the block ends, also where a wait gave up
                if (n) {
                    mbar_wait(q_full, 0, P.err, 203);
                    if (both) mbar_wait(q_full + 8, 0, P.err, 203);
                }
                for (int i = max(0, n - C::ST); i < n; i++) {
                    mbar_wait(k_full + 8 * (i % C::ST), (i / C::ST) & 1, P.err, 204);
                    if (ok || i < n - 1) mbar_wait(v_full + 8 * (i % C::ST), (i / C::ST) & 1, P.err, 205);
                }
            }
        } else if (warp == 9) {
            // ---- products ----
            constexpr uint32_t id_s = idesc_of<T>(128, false), id_o = idesc_of<T>(DP, true);
            bool pend[2] = {false, false}, acc[2] = {false, false}, q_here[2] = {false, false}, ok = true;
            uint32_t p_phase[2] = {0, 0};
            int n = 0, t_prev = 0;
            // O_q += P_q V of the previous key tile
            auto values = [&](int q, bool &v_here) {
                const int st = (n - 1) % C::ST;
                const uint32_t vs = s0 + C::V + st * C::TILE;
                if (!v_here) {
                    if (!mbar_wait_warp(v_full + 8 * st, ((n - 1) / C::ST) & 1, P.err, 206)) return false;
                    const int live = kn - t_prev * kTcKeys;
                    if (live < kTcKeys && kn < p.lk) {
                        // values behind the last key may be anything: zeros, as 0 * NaN is NaN
                        for (int i = lane; i < (kTcKeys - live) * (DP / 8); i += 32) {
                            const int r = live + i / (DP / 8), c = i % (DP / 8);
                            *reinterpret_cast<uint4 *>(sm + C::V + st * C::TILE + (c >> 3) * 16384 + r * 128 + (c & 7) * 16) =
                                make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    v_here = true;
                }
                if (!mbar_wait_warp(p_full + 8 * q, p_phase[q], P.err, 207)) return false;
                p_phase[q] ^= 1;
                tc_fence_after();
                if (lane == 0) {
#pragma unroll
                    for (int kk = 0; kk < kTcKeys / 16; kk++)
                        mma_f16_ts(tmem + 256 + 128 * q, tmem + 128 * q + 8 * kk, swizzled_desc(vs + kk * 2048, 16384), id_o,
                                   acc[q] || kk > 0);
                }
                acc[q] = true;
                return true;
            };
            for (int t = t0; t < t1 && ok; t++) {
                const bool act[2] = {active(0, t), active(1, t)};
                if (!act[0] && !act[1]) continue;
                const int st = n % C::ST;
                const uint32_t ks = s0 + C::K + st * C::TILE;
                bool v_here = false, k_here = false;
                for (int q = 0; q < 2 && ok; q++) {
                    if (pend[q] && !(ok = values(q, v_here))) break;
                    if (act[q]) {
                        if (!k_here && !(ok = mbar_wait_warp(k_full + 8 * st, (n / C::ST) & 1, P.err, 208))) break;
                        k_here = true;
                        if (!q_here[q] && !(ok = mbar_wait_warp(q_full + 8 * q, 0, P.err, 209))) break;
                        q_here[q] = true;
                        if (lane == 0) {
                            const uint32_t qs = s0 + C::Q + q * C::TILE;
#pragma unroll
                            for (int kk = 0; kk < DP / 16; kk++) {
                                const uint32_t at = (kk >> 2) * 16384 + (kk & 3) * 32;
                                mma_f16(tmem + 128 * q, swizzled_desc(qs + at, 16), swizzled_desc(ks + at, 16), id_s, kk > 0, 0);
                            }
                            mma_commit(s_full + 8 * q);
                        }
                    }
                    pend[q] = act[q];
                }
                if (ok && lane == 0) {
                    mma_commit(k_empty + 8 * st);
                    if (n > 0) mma_commit(v_empty + 8 * ((n - 1) % C::ST));
                }
                __syncwarp();
                t_prev = t;
                n++;
            }
            bool v_here = false;
            for (int q = 0; q < 2 && ok; q++)
                if (pend[q]) ok = values(q, v_here);
            if (lane == 0) {
                mma_commit(o_full);
                mma_commit(o_full + 8);
            }
            __syncwarp();
            mbar_wait_warp(o_full, 0, P.err, 212);  // no product is in flight when the block ends
        }
    } else {
        // ---- softmax ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int q = warp >> 2, r_in = (warp & 3) * 32 + lane, i = row0 + 128 * q + r_in;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + 128 * q, o_at = tmem + lanes + 256 + 128 * q;
        const bool there = i < qn;
        const Query r = query_of(p, b, h, min(i, qn - 1), qn, kn);
        const float sc = P.scaled ? 1.f : p.scale;
        float m = -INFINITY, l = 0.f;  // m: in the units of the scores; times sc it is base 2
        uint32_t phase = 0;
        bool any = false, ok = true;
        for (int t = t0; t < t1; t++) {
            if (!active(q, t)) continue;
            if (!(ok = mbar_wait_warp(s_full + 8 * q, phase, P.err, 210))) break;
            phase ^= 1;
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(s_at + 32 * c, s + 32 * c);
            tmem_wait_ld();
            const int j0 = t * kTcKeys;
            if (P.scaled) {
                if (p.cap_out > 0.f) {
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] = p.cap_out * tanh_exp(s[c] * p.cap_in);
                } else {
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] *= p.scale;
                }
                if (P.bias_form == kBiasSlope) {
                    const float d0 = (float)(r.at - j0);
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] = fmaf(-r.slope, fabsf(d0 - (float)c), s[c]);
                } else if (P.bias_form == kBiasLine) {
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] += table_bias(p, r, 0, j0 + c);
                }
            }
            if (!whole(q, t)) {
                // a bit a key: [0, before) or [lo, hi), below end, of this query's document
                const int lo = max(r.lo, 0) - j0, hi = min(r.hi == INT_MAX ? INT_MAX : r.hi - j0, 127) + 1;
                const int before = min(r.pre - j0, 128), end = min(kn - j0, 128);
                uint32_t seen[4];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    seen[w] = (bits_below(hi - 32 * w) & ~bits_below(lo - 32 * w)) | bits_below(before - 32 * w);
                    seen[w] &= bits_below(end - 32 * w);
                    if (docs && seen[w]) {
                        uint32_t same = 0;
#pragma unroll 4
                        for (int c = 0; c < 32; c++)
                            same |= (uint32_t)(__ldg(docs + min(j0 + 32 * w + c, kn - 1)) == r.doc) << c;
                        seen[w] &= same;
                    }
                }
#pragma unroll
                for (int c = 0; c < 128; c++) s[c] = seen[c >> 5] >> (c & 31) & 1 ? s[c] : -INFINITY;
            }
            float top[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                top[x] = s[x];
#pragma unroll
                for (int c = 4 + x; c < 128; c += 4) top[x] = fmaxf(top[x], s[c]);
            }
            const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            // (m is -inf until a row has seen a key)
            if (__any_sync(0xffffffffu, now * sc > m * sc + 8.f || (m == -INFINITY && now > m))) {
                const float to = fmaxf(m, now), alpha = exp2_fast((m - (to == -INFINITY ? 0.f : to)) * sc);
                if (any) {
                    for (int c = 0; c < DP; c += 32) {
                        float o[32];
                        tmem_ld32(o_at + c, o);
                        tmem_wait_ld();
                        uint32_t w[2][16];
#pragma unroll
                        for (int x = 0; x < 32; x++) w[x >> 4][x & 15] = __float_as_uint(o[x] * alpha);
                        tmem_st16(o_at + c, w[0]);
                        tmem_st16(o_at + c + 16, w[1]);
                    }
                }
                l *= m == -INFINITY ? 0.f : alpha;
                m = to;
            }
            any = true;
            const float base = m == -INFINITY ? 0.f : m * sc;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[16];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const float a = exp2_fast(fmaf(s[32 * c + 2 * x], sc, -base)),
                                z = exp2_fast(fmaf(s[32 * c + 2 * x + 1], sc, -base));
                    sum[(2 * x) & 3] += a;
                    sum[(2 * x + 1) & 3] += z;
                    w[x] = MmaOp<T>::pack(a, z);
                }
                tmem_st16(s_at + 16 * c, w);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * q);
        }

        // ---- out ----
        if (ok && any) ok = mbar_wait_warp(o_full + 8 * q, 0, P.err, 211);
        if (ok && (q == 0 || both)) {
            tc_fence_after();
            const float f = l == 0.f ? 0.f : 1.f / l;
            char *const mine = sm + C::Q + q * C::TILE;  // this warp's 32 rows of the queries, no longer read
            bool odd = false;
            for (int c = 0; c < DP; c += 32) {
                float o[32];
                if (any) {
                    tmem_ld32(o_at + c, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int x = 0; x < 32; x++) {
                    if (!any) o[x] = 0.f;
                    odd |= !(fabsf(o[x]) < INFINITY);
                    o[x] = l == 0.f ? 0.f : o[x] * f;
                }
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int ch = (c >> 3) + x;
                    *reinterpret_cast<uint4 *>(mine + (ch >> 3) * 16384 + r_in * 128 + (((ch & 7) ^ (r_in & 7)) << 4)) =
                        make_uint4(MmaOp<T>::pack(o[8 * x], o[8 * x + 1]), MmaOp<T>::pack(o[8 * x + 2], o[8 * x + 3]),
                                   MmaOp<T>::pack(o[8 * x + 4], o[8 * x + 5]), MmaOp<T>::pack(o[8 * x + 6], o[8 * x + 7]));
                }
            }
            __syncwarp();
            // A row that is not finite again from the keys that it sees alone (0 * v of one that it does not
            // see is NaN when v is not finite).
            uint32_t again = p.masked ? __ballot_sync(0xffffffffu, there && odd) : 0u;
            const int r0 = (warp & 3) * 32;
            for (; again; again &= again - 1) {
                const int x = __ffs(again) - 1;
                float rm, rl, ro[8];
                attend_row<T>(p, b, h, row0 + 128 * q + r0 + x, qn, kn, t0 * kTcKeys, min(t1 * kTcKeys, kn),
                              (float *)(sm + C::SCRATCH) + warp * 256, rm, rl, ro);
                const float rf = rl == 0.f ? 0.f : 1.f / rl;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int c = lane + 32 * e, ch = c >> 3, row = r0 + x;
                    if (c < p.d)
                        *reinterpret_cast<T *>(mine + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4) + (c & 7) * 2) =
                            from_f<T>(rl == 0.f ? 0.f : ro[e] * rf);
                }
                __syncwarp();
            }
            T *const out = (T *)p.out + b * p.ob + h * p.oh;
            const int per = P.wo == 16 ? 8 : P.wo == 4 ? 2 : 1, units = p.d / per;
            for (int idx = lane; idx < 32 * units; idx += 32) {
                const int x = idx / units, c = (idx - x * units) * per, row = r0 + x, ch = c >> 3;
                if (row0 + 128 * q + row >= qn) break;
                T *dst = out + (int64_t)(row0 + 128 * q + row) * p.ot + c;
                const char *src = mine + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4) + (c & 7) * 2;
                if (per == 8)
                    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
                else if (per == 2)
                    *reinterpret_cast<uint32_t *>(dst) = *reinterpret_cast<const uint32_t *>(src);
                else
                    *dst = *reinterpret_cast<const T *>(src);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace dev
}  // namespace ajib
