/*
 * attention_few.cuh — attention of few queries over many keys (new tokens over a cache): up to 16 rows
 * (query, head of the group) a block, the keys split over warps, blocks and joined.
 *
 * Bound by reading keys and values once. A block keeps a ring of 64-key tiles, each copied by one
 * warp with TMA (keys and values, 128-byte swizzle, so that ldmatrix meets no bank conflict); four
 * warps take 16 keys of every tile each, with a maximum, sum and outputs of their own (mma.sync:
 * with 16 rows the tensor cores are idle most of the time in any form). They wait for copies and
 * hand stages back by mbarriers, without meeting until the end. Copies of 32 threads' loads (cp.async)
 * in place of TMA took 4 us a tile and block where one warp is left alone on its scheduler.
 *
 * Keys behind a sequence's last are masked; their values are set to zero in shared memory by the warp
 * that owns them, whatever they held.
 */
#pragma once

#include "attention_mma.cuh"

namespace ajib {

constexpr int kFewThreads = 160;  // four warps of products and one of copies

template <int DP> struct FewCfg {
    static constexpr int ST = DP == 64 ? 4 : 3;
    static constexpr int HALF = kMmaKeys * 128;        // 64 components of a tile's keys
    static constexpr int TILE = kMmaKeys * DP * 2, STAGE = 2 * TILE;
    static constexpr int RING = 16 * DP * 2;           // behind the queries (a multiple of 1024 bytes)
    static constexpr int BARS = RING + ST * STAGE;
    static constexpr int SMEM = BARS + 2 * ST * 8 + 1024;
    static constexpr int BLOCKS = DP == 64 ? 3 : DP == 128 ? 2 : 1;
    static_assert(4 * 16 * (DP + 2) * 4 <= ST * STAGE, "the join reuses the ring");
};

namespace dev {

// Byte offset of component chunk c (16 bytes) of a key's row in a tile as TMA writes it.
__device__ __forceinline__ uint32_t ring_at(int row, int c)
{
    return (c >> 3) * (kMmaKeys * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kFewThreads, FewCfg<DP>::BLOCKS)
    k_attn_few(const __grid_constant__ MmaDev P, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
               int *err)
{
    using C = FewCfg<DP>;
    const AttnDev &p = P.a;
    extern __shared__ char sm_raw[];
    char *const sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
    const uint32_t sm0 = smem_u32(sm), full = sm0 + C::BARS, empty = full + 8 * C::ST;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    // ---- which rows and keys ----
    uint32_t at = blockIdx.x;
    const int split = at % P.nsplit;
    at /= P.nsplit;
    const int tile = at % P.row_tiles;
    at /= P.row_tiles;
    const int hk = at % p.hk, b = at / p.hk;
    const int qn = q_count(p, b), kn = k_count(p, b), row0 = tile * 16, rows = qn * p.group;
    if (row0 >= rows) return;
    const int shift = p.align_end ? kn - qn : 0;
    const int first = row0 / p.group + shift, last = (min(row0 + 16, rows) - 1) / p.group + shift;
    const int pre = p.prefix ? max(__ldg(p.prefix + b), 0) : 0;
    int key_lo, key_hi;
    reach_of(p, first, last, pre, kn, key_lo, key_hi);
    int t0 = key_lo / kMmaKeys, t1 = (key_hi + kMmaKeys - 1) / kMmaKeys;
    const int per = (t1 - t0 + P.nsplit - 1) / P.nsplit;
    t0 = min(t0 + split * per, t1);
    t1 = min(t0 + per, t1);

    if (tid == 128) {
        for (int i = 0; i < C::ST; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 4);
        }
        fence_mbar_init();
    }
    if (tid < 128) {
        if (p.d < DP) {
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < 16 * (DP / 8); i += 128) *reinterpret_cast<uint4 *>(sm + tile_at<DP>(i / (DP / 8), i % (DP / 8))) = zero;
            named_bar_sync(1, 128);
        }
        const T *const q = (const T *)p.q + b * p.qb + (int64_t)hk * p.group * p.qh;
        load_tile<T, DP, 16>(sm0, sm, p.d, P.wq, q, [&](int r) -> const T * {
            const int row = row0 + r, i = row / p.group;
            return row < rows ? q + i * p.qt + (row - i * p.group) * p.qh : nullptr;
        });
        cp_commit();
        cp_wait<0>();
    }
    __syncthreads();

    bool ok = true;
    if (warp == 4) {
        if (elect_one()) {
            int n = 0;
            for (int t = t0; t < t1; t++, n++) {
                const int st = n % C::ST;
                if (!tc_wait(empty + 8 * st, ((n / C::ST) & 1) ^ 1, err, 221)) break;
                mbar_arrive_expect_tx(full + 8 * st, C::STAGE);
                const uint32_t dst = sm0 + C::RING + st * C::STAGE;
                for (int y = 0; y < DP / 64; y++) {
                    tma_load_4d(dst + y * C::HALF, &mk, full + 8 * st, 64 * y, t * kMmaKeys, hk, b);
                    tma_load_4d(dst + C::TILE + y * C::HALF, &mv, full + 8 * st, 64 * y, t * kMmaKeys, hk, b);
                }
            }
            // every copy has landed before the ring is used for the join, also where a wait gave up
            for (int i = max(0, n - C::ST); i < n; i++) tc_wait(full + 8 * (i % C::ST), (i / C::ST) & 1, err, 222);
        }
        __syncwarp();
    }

    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < DP / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    if (warp < 4) {
        Query qr[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int row = min(row0 + (lane >> 2) + 8 * x, rows - 1), i = row / p.group;
            qr[x] = query_at(p, 0, hk * p.group + row - i * p.group, i, shift, pre);
        }
        constexpr bool QREG = DP <= 128;
        uint32_t qf[QREG ? DP / 16 : 1][4];
        if (QREG) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++) ldsm4(qf[QREG ? kk : 0], sm0 + tile_at<DP>(lane & 15, 2 * kk + (lane >> 4)));
        }
        const int key_at = warp * 16, c0 = key_at + 2 * (lane & 3);  // this thread's keys: c0 + {0, 1, 8, 9} of a tile
        int n = 0;
        for (int t = t0; t < t1; t++, n++) {
            const int st = n % C::ST, j0 = t * kMmaKeys;
            const uint32_t ks = sm0 + C::RING + st * C::STAGE, vs = ks + C::TILE;
            if (!(ok = tc_wait_warp(full + 8 * st, (n / C::ST) & 1, err, 223))) break;
            // this warp's keys behind the last one
            const int live = kn - j0 - key_at;
            if (live < 16) {
                char *v = sm + C::RING + st * C::STAGE + C::TILE;
                for (int i = lane; i < 16 * (DP / 8); i += 32) {
                    const int r = i / (DP / 8);
                    if (r >= live) *reinterpret_cast<uint4 *>(v + ring_at(key_at + r, i % (DP / 8))) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
            float s[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++) {
                if (kk * 16 < p.d) {
                    uint32_t a[4], bb[4];
                    if (QREG) {
#pragma unroll
                        for (int x = 0; x < 4; x++) a[x] = qf[QREG ? kk : 0][x];
                    } else {
                        ldsm4(a, sm0 + tile_at<DP>(lane & 15, 2 * kk + (lane >> 4)));
                    }
                    ldsm4(bb, ks + ring_at(key_at + (lane >> 4) * 8 + (lane & 7), 2 * kk + (lane >> 3 & 1)));
                    MmaOp<T>::mma(s[0], a, bb[0], bb[1]);
                    MmaOp<T>::mma(s[1], a, bb[2], bb[3]);
                }
            }
            bool all = j0 + kMmaKeys <= kn;
            if (all && !(j0 + kMmaKeys <= pre))
                all = (p.left == INT_MAX / 2 || j0 >= last - p.left) &&
                      (p.right == INT_MAX / 2 || j0 + kMmaKeys - 1 <= first + p.right);
            if (P.plain) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[e >> 2][e & 3] *= p.scale;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int j = min(j0 + c0 + (e >> 2) * 8 + (e & 1), kn - 1);  // (a table is only read inside it)
                    s[e >> 2][e & 3] = score2(p, qr[e >> 1 & 1], j, s[e >> 2][e & 3]);
                }
            }
            if (!all) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int j = j0 + c0 + (e >> 2) * 8 + (e & 1);
                    if (!(j < kn && in_reach(qr[e >> 1 & 1], j))) s[e >> 2][e & 3] = -INFINITY;
                }
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
                for (int e = 0; e < 4; e++) {
                    float &v = s[e >> 1][2 * x + (e & 1)];
                    v = exp2_fast(v - base);
                    l[x] += v;
                }
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int i = 0; i < DP / 8; i++) {
                    o[i][0] *= alpha[0];
                    o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1];
                    o[i][3] *= alpha[1];
                }
            }
            const uint32_t a[4] = {MmaOp<T>::pack(s[0][0], s[0][1]), MmaOp<T>::pack(s[0][2], s[0][3]),
                                   MmaOp<T>::pack(s[1][0], s[1][1]), MmaOp<T>::pack(s[1][2], s[1][3])};
#pragma unroll
            for (int i = 0; i < DP / 8; i += 2) {
                if (i * 8 < p.d) {
                    uint32_t bb[4];
                    ldsm4t(bb, vs + ring_at(key_at + (lane & 15), i + (lane >> 4)));
                    MmaOp<T>::mma(o[i], a, bb[0], bb[1]);
                    MmaOp<T>::mma(o[i + 1], a, bb[2], bb[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * st);
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        }
    }
    __syncthreads();  // the copies have landed and are read: the ring is free
    if (warp < 4) {
        join_warps<T, DP>(P, b, hk, row0, rows, split, qn, kn, t0 * kMmaKeys, min(t1 * kMmaKeys, kn), o, m, l,
                          (float *)(sm + C::RING));
    }
}

}  // namespace dev
}  // namespace ajib
