/*
 * attention_mma.cuh — attention on warp-level tensor instructions (mma.sync m16n8k16, fp32
 * accumulators): heads of more than 128 components, layouts that TMA does not copy, documents with few
 * queries and clamped grid tables; what attention_tc.cuh and attention_few.cuh do not take. Probabilities are
 * rounded to the type of v, which the instruction wants of both operands; their sum is of the unrounded ones.
 *
 * Rows of a tile are (query, head of the group) pairs, row = query * group + head, so that the heads
 * that share keys share their reads. A block of 4 warps walks the keys in tiles of 64, copied ahead
 * of use (cp.async) into a ring of stages; scores and probabilities stay in registers (the
 * accumulator layout of q k^T is the operand layout of p v).
 *   ROWS: 64 rows a block, 16 a warp, every warp reads every key.
 *   KEYS: 16 rows a block; each warp takes 16 keys of each tile and the four are joined at the end.
 *         With few queries the keys are also split over blocks (nsplit), joined by k_attn_join.
 */
#pragma once

#include "attention.cuh"
#include "attention_odd.cuh"
#include "sm100.cuh"

namespace ajib {

constexpr int kMmaThreads = 128, kMmaKeys = 64;

// How the table's bias of a key is found: key by key from its row and column, with or without clamps.
enum { kBiasNone = 0, kBiasSlope = 1, kBiasGridDirect = 2, kBiasLine = 3, kBiasGrid = 4 };

struct MmaDev {
    AttnDev a;
    int rows, row_tiles, nsplit;  // rows = lq * group of a (sequence, key head)
    int bias_form;
    int plain;        // scores are the scaled products alone
    int wq, wkv, wo;  // widest copies (bytes) of q, of k and v, of out
    float *part;      // [sequence, key head, row][nsplit][d] unnormalised outputs
    float2 *part_ml;  // [..][nsplit] maximum (base 2) and sum
};

namespace dev {

// mbar_wait with a hint (10 us) of how long the hardware may keep a waiting thread asleep: the roles of the
// pipelined kernels (attention_tc.cuh, attention_few.cuh) wait for one another most of the time, and polling took
// their issue slots. tiles: how many key tiles (at most 2.2 us each) may rightly come between, for which 40 us each
// are added to the 2 s.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, int *err, int code, int tiles = 0)
{
    if (mbar_test_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(bar), "r"(parity), "r"(10000u)
            : "memory");
        if (done) return true;
        if (globaltimer() - t0 > 2000000000ull + (uint64_t)tiles * 40000ull) {
            atomicCAS(err, 0, code);
            return false;
        }
    }
}
__device__ __forceinline__ bool tc_wait_warp(uint32_t bar, uint32_t parity, int *err, int code, int tiles = 0)
{
    return __all_sync(0xffffffffu, tc_wait(bar, parity, err, code, tiles));
}
// One lane of a converged warp. (Told by a lane number instead, the compiler takes the operands of the
// branch's products and copies for divergent, and each issue costs 140 cycles instead of a few.)
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
// Copies that fill with zeros when `bytes` is 0 (the address must still be one of the tensor's).
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of component chunk c (8 components, 16 bytes) of a row in a tile of DP components a
// row: chunks are permuted so that eight rows' equal chunks (one ldmatrix) fall in eight bank groups.
template <int DP> __device__ __forceinline__ uint32_t tile_at(int row, int c)
{
    if (DP == 32) return row * 64 + ((c ^ (row >> 1 & 3)) << 4);
    return row * (DP * 2) + ((c ^ (row & 7)) << 4);
}

// Copies one row-indexed tile of n rows: row(r) gives the source row, or NULL for zeros. Components
// behind d are not written (they hold zeros from the start).
template <typename T, int DP, int N, typename RowFn>
__device__ __forceinline__ void load_tile(uint32_t dst, char *dst_generic, int d, int width, const T *any, RowFn &&row)
{
    const int tid = threadIdx.x;
    if (width == 16) {
        constexpr int CH = DP / 8;
        static_assert(N * CH % kMmaThreads == 0 || N * CH < kMmaThreads, "");
#pragma unroll
        for (int n = 0; n < (N * CH + kMmaThreads - 1) / kMmaThreads; n++) {
            const int idx = tid + n * kMmaThreads, r = idx / CH, c = idx % CH;
            if ((N * CH >= kMmaThreads || idx < N * CH) && c * 8 < d) {
                const T *s = row(r);
                cp16(dst + tile_at<DP>(r, c), s ? s + c * 8 : any, s ? 16 : 0);
            }
        }
    } else if (width == 4) {
        for (int idx = tid; idx < N * (DP / 2); idx += kMmaThreads) {
            const int r = idx / (DP / 2), c = idx % (DP / 2);
            if (c * 2 < d) {
                const T *s = row(r);
                cp4(dst + tile_at<DP>(r, c >> 2) + (c & 3) * 4, s ? s + c * 2 : any, s ? 4 : 0);
            }
        }
    } else {
        for (int idx = tid; idx < N * DP; idx += kMmaThreads) {
            const int r = idx / DP, c = idx % DP;
            if (c < d) {
                const T *s = row(r);
                *reinterpret_cast<T *>(dst_generic + tile_at<DP>(r, c >> 3) + (c & 7) * 2) = s ? s[c] : from_f<T>(0.f);
            }
        }
    }
}

// The smallest and largest of a key tile's n documents, with as many loads in flight as fit.
template <int KT> __device__ __forceinline__ void document_range(const int *ids, int n, int &lo, int &hi)
{
    if (((uintptr_t)ids & 15) == 0 && n == KT) {
#pragma unroll 8
        for (int v = 0; v < KT; v += 4) {
            const int4 id = __ldg(reinterpret_cast<const int4 *>(ids + v));
            lo = min(min(lo, min(id.x, id.y)), min(id.z, id.w));
            hi = max(max(hi, max(id.x, id.y)), max(id.z, id.w));
        }
    } else {
#pragma unroll 8
        for (int v = 0; v < n; v++) {
            const int id = __ldg(ids + v);
            lo = min(lo, id);
            hi = max(hi, id);
        }
    }
}

// Keys [lo, hi) that some query standing from `first` to `last` sees; [0, 0) where there is none (queries that
// stand a window past the last key).
__device__ __forceinline__ void reach_of(const AttnDev &p, int first, int last, int pre, int kn, int &lo, int &hi)
{
    lo = p.left == INT_MAX / 2 ? 0 : max(first - p.left, 0);
    hi = p.right == INT_MAX / 2 ? kn : min(kn, last + p.right + 1);
    if (pre > 0) {
        lo = 0;
        hi = max(hi, min(pre, kn));
    }
    if (lo >= hi) lo = hi = 0;
}

template <int DP, bool KEYS> struct MmaCfg {
    static constexpr int BM = KEYS ? 16 : 64;
    static constexpr int NST = DP >= 256 ? 2 : DP == 128 ? (KEYS ? 3 : 2) : KEYS ? 4 : 3;
    static constexpr int Q_BYTES = BM * DP * 2;
    static constexpr int TILE = kMmaKeys * DP * 2;
    static constexpr int META = 3 * kMmaKeys * 4;  // documents, rows, columns of a tile's keys
    static constexpr int STAGE = 2 * TILE + META;
    static constexpr int JOIN = 4 * 16 * (DP + 2) * 4;
    static constexpr int BITS = Q_BYTES + NST * STAGE;
    static_assert(!KEYS || JOIN <= NST * STAGE, "the join reuses the stages");
    // bits: two words (seen, whole) for every 32 tiles when there are documents
    static int smem(const AttnDev &p)
    {
        const int words = p.q_doc ? (p.lk + kMmaKeys * 32 - 1) / (kMmaKeys * 32) : 0;
        return BITS + words * 8;
    }
};

// Joins the results of four warps (threads 0 to 127) over keys of their own for the same 16 rows, in
// memory of 4 * 16 * (DP + 2) floats, and writes them out, or to the workspace where the keys are
// split. Rows that are not finite are looked into (attention_odd.cuh): keys [j_begin, j_end), 16 a warp.
template <typename T, int DP>
__device__ __forceinline__ void join_warps(const MmaDev &P, int b, int hk, int row0, int rows, int split, int qn, int kn,
                                           int j_begin, int j_end, const float (&o)[DP / 8][4], const float (&m)[2],
                                           const float (&l)[2], float *memory)
{
    const AttnDev &p = P.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *const jm = memory, *const jl = jm + 64, *const jo = jl + 64;  // [warp][16], [warp][16], [warp][16][DP]
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = (lane >> 2) + 8 * x;
        if ((lane & 3) == 0) {
            jm[warp * 16 + r] = m[x];
            jl[warp * 16 + r] = l[x];
        }
#pragma unroll
        for (int n = 0; n < DP / 8; n++)
            *reinterpret_cast<float2 *>(jo + (warp * 16 + r) * DP + n * 8 + 2 * (lane & 3)) =
                make_float2(o[n][2 * x], o[n][2 * x + 1]);
    }
    named_bar_sync(1, 128);
    uint32_t left = 15;  // rows warp + 4 y to write
    for (bool again = p.masked;; again = false) {
        uint32_t odd_rows = 0;
        for (int y = 0; y < 4 && row0 + warp + 4 * y < rows; y++) {
            if (!(left >> y & 1)) continue;
            const int r = warp + 4 * y, row = row0 + r, i = row / p.group, h = hk * p.group + row - i * p.group;
            float top = -INFINITY, sum = 0.f, ro[8], f[4];
#pragma unroll
            for (int w = 0; w < 4; w++) top = fmaxf(top, jm[w * 16 + r]);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                f[w] = exp2_fast(jm[w * 16 + r] - (top == -INFINITY ? 0.f : top));
                sum += jl[w * 16 + r] * f[w];
            }
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = lane + 32 * e;
                ro[e] = 0.f;
                if (c < p.d) {
#pragma unroll
                    for (int w = 0; w < 4; w++) ro[e] += jo[(w * 16 + r) * DP + c] * f[w];
                    odd |= !(fabsf(ro[e]) < INFINITY);
                }
            }
            if (again && __any_sync(0xffffffffu, odd)) {
                odd_rows |= 1u << y;
                continue;
            }
            if (P.nsplit > 1) {
                const int64_t slot = (((int64_t)b * p.hk + hk) * P.rows + row) * P.nsplit + split;
                if (lane == 0) P.part_ml[slot] = make_float2(top, sum);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (lane + 32 * e < p.d) P.part[slot * p.d + lane + 32 * e] = ro[e];
            } else {
                T *dst = (T *)p.out + b * p.ob + i * p.ot + h * p.oh;
                const float g = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (lane + 32 * e < p.d) dst[lane + 32 * e] = from_f<T>(sum == 0.f ? 0.f : ro[e] * g);
            }
        }
        if (!again || !named_bar_any(1, 128, odd_rows != 0)) break;
        left = odd_rows;
        const OddRows these = {b, hk * p.group, p.group, row0, rows, qn, kn};
        if (named_bar_any(1, 128, unseen_odd<T>(p, these, j_begin + 32 * warp, j_end, 128))) {
            redo_share<T, DP>(p, these, j_begin + 16 * warp, j_end, jm + warp * 16, jl + warp * 16, jo + warp * 16 * DP);
            named_bar_sync(1, 128);
        }
    }
}

// (a call: inlined it costs the kernel's loops registers)
template <typename T, int DP> __device__ __noinline__ void redo_rows_apart(const AttnDev &p, const OddRows &r, int j0, int j1)
{
    redo_rows<T, DP>(p, r, j0, j1);
}

template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(kMmaThreads) k_attn_mma(const __grid_constant__ MmaDev P)
{
    using C = MmaCfg<DP, KEYS>;
    const AttnDev &p = P.a;
    extern __shared__ __align__(128) char sm[];
    const uint32_t sm0 = smem_u32(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    char *const stage0 = sm + C::Q_BYTES;
    uint32_t *const bits = (uint32_t *)(sm + C::BITS);

    // ---- which rows and keys ----
    int64_t at = blockIdx.x;
    const int split = KEYS ? (int)(at % P.nsplit) : 0;
    if (KEYS) at /= P.nsplit;
    // a prompt's last rows see the most keys: first, so that no long block starts last
    const int tile = P.row_tiles - 1 - (int)(at % P.row_tiles);
    at /= P.row_tiles;
    const int hk = (int)(at % p.hk), b = (int)(at / p.hk);
    const int qn = q_count(p, b), kn = k_count(p, b), row0 = tile * C::BM;
    const int rows = qn * p.group;
    if (row0 >= rows) return;
    const int shift = p.align_end ? kn - qn : 0;
    const int first = row0 / p.group + shift, last = (min(row0 + C::BM, rows) - 1) / p.group + shift;
    const int pre = p.prefix ? __ldg(p.prefix + b) : 0;
    int key_lo, key_hi;
    reach_of(p, first, last, pre, kn, key_lo, key_hi);
    int t0 = key_lo / kMmaKeys, t1 = (key_hi + kMmaKeys - 1) / kMmaKeys;
    if (KEYS && P.nsplit > 1) {
        const int per = (t1 - t0 + P.nsplit - 1) / P.nsplit;
        t0 = min(t0 + split * per, t1);
        t1 = min(t0 + per, t1);
    }

    // ---- queries in, padding components zeroed ----
    const T *const q = (const T *)p.q + b * p.qb + (int64_t)hk * p.group * p.qh;
    const T *const k = (const T *)p.k + b * p.kb + hk * p.kh;
    const T *const v = (const T *)p.v + b * p.vb + hk * p.vh;
    if (p.d < DP) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const int c0 = p.d / 8;  // a chunk that is only partly padding is written whole, before its copies
        for (int r = tid; r < C::BM; r += kMmaThreads)
            for (int c = c0; c < DP / 8; c++) *reinterpret_cast<uint4 *>(sm + tile_at<DP>(r, c)) = zero;
        for (int r = tid; r < 2 * C::NST * kMmaKeys; r += kMmaThreads) {
            char *t = stage0 + (r / (2 * kMmaKeys)) * C::STAGE + (r / kMmaKeys & 1) * C::TILE;
            for (int c = c0; c < DP / 8; c++) *reinterpret_cast<uint4 *>(t + tile_at<DP>(r % kMmaKeys, c)) = zero;
        }
        __syncthreads();
    }
    load_tile<T, DP, C::BM>(sm0, sm, p.d, P.wq, q, [&](int r) -> const T * {
        const int row = row0 + r, i = row / p.group;
        return row < rows ? q + i * p.qt + (row - i * p.group) * p.qh : nullptr;
    });
    cp_commit();

    // ---- documents: which key tiles hold one of this block's, and which nothing else ----
    const int *const docs = p.k_doc ? p.k_doc + (int64_t)(b % p.doc_rows) * p.lk : nullptr;
    const int word0 = t0 / 32;
    if (docs) {
        const int *qd = p.q_doc + (int64_t)(b % p.doc_rows) * p.lq;
        int lo = INT_MAX, hi = INT_MIN;
        for (int i = row0 / p.group + lane; i <= (min(row0 + C::BM, rows) - 1) / p.group; i += 32) {
            const int x = __ldg(qd + i);
            lo = min(lo, x);
            hi = max(hi, x);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        for (int w = word0 + warp; w * 32 < t1; w += kMmaThreads / 32) {
            // lane l looks at tile w * 32 + l, so that its loads are in flight together
            const int t = w * 32 + lane;
            int klo = INT_MAX, khi = INT_MIN;
            if (t >= t0 && t < t1) document_range<kMmaKeys>(docs + t * kMmaKeys, min(kn - t * kMmaKeys, kMmaKeys), klo, khi);
            const uint32_t seen = __ballot_sync(0xffffffffu, khi >= 0 && max(lo, 0) <= khi && klo <= hi);
            const uint32_t whole = __ballot_sync(0xffffffffu, lo >= 0 && lo == hi && klo == lo && khi == lo);
            if (lane == 0) {
                bits[2 * (w - word0)] = seen;
                bits[2 * (w - word0) + 1] = whole;
            }
        }
        __syncthreads();
    }
    auto next = [&](int t) {  // the first tile from t on that some row sees a key of
        for (; t < t1; t++) {
            const int j = t * kMmaKeys;
            if (docs && !(bits[2 * (t / 32 - word0)] >> (t & 31) & 1)) continue;
            if (j < pre) break;
            if ((p.left == INT_MAX / 2 || j + kMmaKeys - 1 >= first - p.left) &&
                (p.right == INT_MAX / 2 || j <= last + p.right))
                break;
        }
        return t;
    };
    auto load = [&](int t, int slot) {
        if (t < t1) {
            const uint32_t dst = sm0 + C::Q_BYTES + slot * C::STAGE;
            char *g = stage0 + slot * C::STAGE;
            const int j0 = t * kMmaKeys;
            load_tile<T, DP, kMmaKeys>(dst, g, p.d, P.wkv, k, [&](int r) -> const T * { return j0 + r < kn ? k + (j0 + r) * p.kt : nullptr; });
            load_tile<T, DP, kMmaKeys>(dst + C::TILE, g + C::TILE, p.d, P.wkv, v,
                                       [&](int r) -> const T * { return j0 + r < kn ? v + (j0 + r) * p.vt : nullptr; });
            int *meta = (int *)(g + 2 * C::TILE);
            if (tid < kMmaKeys) {
                const int j = j0 + tid, jj = j < kn ? j : 0;  // (a table is only read inside it)
                if (docs) meta[tid] = j < kn ? __ldg(docs + j) : -1;
                if (P.bias_form == kBiasGridDirect || P.bias_form == kBiasGrid) {
                    const int y = jj / p.grid_w, x = jj - y * p.grid_w;
                    meta[kMmaKeys + tid] = P.bias_form == kBiasGridDirect ? y * (2 * p.reach_x + 1) + x : y;
                    meta[2 * kMmaKeys + tid] = x;
                }
            }
        }
        cp_commit();
    };
    int tl = next(t0), tc = tl;
#pragma unroll
    for (int n = 0; n < C::NST - 1; n++) {
        load(tl, n);
        if (tl < t1) tl = next(tl + 1);
    }

    // ---- this thread's two rows ----
    const int m0 = KEYS ? 0 : warp * 16;  // the warp's first row
    Query qr[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int row = min(row0 + m0 + (lane >> 2) + 8 * x, rows - 1), i = row / p.group;
        qr[x] = query_of(p, b, hk * p.group + row - i * p.group, i, qn, kn);
        if (P.bias_form == kBiasGridDirect)
            qr[x].table += (p.reach_y - qr[x].y) * (2 * p.reach_x + 1) + p.reach_x - qr[x].x;
    }
    constexpr bool QREG = DP <= 128;
    uint32_t qf[QREG ? DP / 16 : 1][4];
    const uint32_t q_at = (m0 + (lane & 15));  // ldmatrix: rows by lane & 15, halves of 16 components by lane >> 4
    if (QREG) {
        cp_wait<C::NST - 1>();
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) ldsm4(qf[QREG ? kk : 0], sm0 + tile_at<DP>(q_at, 2 * kk + (lane >> 4)));
    }

    constexpr int NT = KEYS ? 2 : 8;
    const int key_at = KEYS ? warp * 16 : 0;
    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < DP / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (int it = 0; tc < t1; it++) {
        cp_wait<C::NST - 2>();
        __syncthreads();
        load(tl, (it + C::NST - 1) % C::NST);
        if (tl < t1) tl = next(tl + 1);
        const int slot = it % C::NST;
        const uint32_t ks = sm0 + C::Q_BYTES + slot * C::STAGE, vs = ks + C::TILE;
        const int *meta = (const int *)(stage0 + slot * C::STAGE + 2 * C::TILE);
        const int j0 = tc * kMmaKeys;

        // s = q k^T
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
            if (kk * 16 < p.d) {
                uint32_t a[4];
                if (QREG) {
#pragma unroll
                    for (int x = 0; x < 4; x++) a[x] = qf[QREG ? kk : 0][x];
                } else {
                    ldsm4(a, sm0 + tile_at<DP>(q_at, 2 * kk + (lane >> 4)));
                }
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t bb[4];
                    ldsm4(bb, ks + tile_at<DP>(key_at + n * 8 + (lane >> 4) * 8 + (lane & 7), 2 * kk + (lane >> 3 & 1)));
                    MmaOp<T>::mma(s[n], a, bb[0], bb[1]);
                    MmaOp<T>::mma(s[n + 1], a, bb[2], bb[3]);
                }
            }
        }

        // scores, base 2
        if (p.cap_out > 0.f) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] = p.cap_out * tanh_of(s[n][e] * p.cap_in);
        } else {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] *= p.scale;
        }
        const int c0 = key_at + 2 * (lane & 3);  // this thread's keys: j0 + c0 + 8 n + {0, 1}
        if (P.bias_form == kBiasSlope) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[n][e] -= qr[e >> 1].slope * (float)abs(qr[e >> 1].at - (j0 + c0 + 8 * n + (e & 1)));
        } else if (P.bias_form == kBiasGridDirect) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[n][e] = fmaf(__ldg(qr[e >> 1].table + meta[kMmaKeys + c0 + 8 * n + (e & 1)]), kLog2e, s[n][e]);
        } else if (P.bias_form == kBiasLine) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] += table_bias(p, qr[e >> 1], 0, j0 + c0 + 8 * n + (e & 1));
        } else if (P.bias_form == kBiasGrid) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int c = c0 + 8 * n + (e & 1);
                    s[n][e] += table_bias(p, qr[e >> 1], meta[kMmaKeys + c], meta[2 * kMmaKeys + c]);
                }
        }

        // masks: none where every row of the block sees every key of the tile
        bool all = j0 + kMmaKeys <= kn;
        if (all && !(j0 + kMmaKeys <= pre))
            all = (p.left == INT_MAX / 2 || j0 >= last - p.left) &&
                  (p.right == INT_MAX / 2 || j0 + kMmaKeys - 1 <= first + p.right);
        if (all && docs) all = bits[2 * (tc / 32 - word0) + 1] >> (tc & 31) & 1;
        if (!all) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int c = c0 + 8 * n + (e & 1), j = j0 + c;
                    const Query &r = qr[e >> 1];
                    if (!(j < kn && in_reach(r, j) && (!docs || meta[c] == r.doc))) s[n][e] = -INFINITY;
                }
        }

        // running maximum and sum
        float alpha[2], base[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            float top = s[0][2 * x];
#pragma unroll
            for (int n = 0; n < NT; n++) top = fmaxf(top, fmaxf(s[n][2 * x], s[n][2 * x + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(top, m[x]);
            base[x] = top == -INFINITY ? 0.f : top;
            alpha[x] = exp2_fast(m[x] - base[x]);
            m[x] = top;
            l[x] *= alpha[x];
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[n][e] = exp2_fast(s[n][e] - base[e >> 1]);
                l[e >> 1] += s[n][e];
            }
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
            o[n][0] *= alpha[0];
            o[n][1] *= alpha[0];
            o[n][2] *= alpha[1];
            o[n][3] *= alpha[1];
        }

        // o += p v (probabilities rounded to T)
#pragma unroll
        for (int kk = 0; kk < NT / 2; kk++) {
            const uint32_t a[4] = {MmaOp<T>::pack(s[2 * kk][0], s[2 * kk][1]), MmaOp<T>::pack(s[2 * kk][2], s[2 * kk][3]),
                                   MmaOp<T>::pack(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                   MmaOp<T>::pack(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
            for (int n = 0; n < DP / 8; n += 2) {
                if (n * 8 < p.d) {
                    uint32_t bb[4];
                    ldsm4t(bb, vs + tile_at<DP>(key_at + kk * 16 + (lane & 15), n + (lane >> 4)));
                    MmaOp<T>::mma(o[n], a, bb[0], bb[1]);
                    MmaOp<T>::mma(o[n + 1], a, bb[2], bb[3]);
                }
            }
        }
        tc = next(tc + 1);
    }
    cp_wait<0>();
#pragma unroll
    for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    const int j_begin = t0 * kMmaKeys, j_end = min(t1 * kMmaKeys, kn);

    if (!KEYS) {
        // rows that are not finite (attention_odd.cuh)
        bool odd = false;
        if (p.masked) {
#pragma unroll
            for (int n = 0; n < DP / 8; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= !(fabsf(o[n][e]) < INFINITY);
        }
        __syncwarp();
        char *const mine = sm;  // rows m0 .. m0 + 15 of the queries' tile: this warp's alone
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const float f = l[x] == 0.f ? 0.f : 1.f / l[x];
#pragma unroll
            for (int n = 0; n < DP / 8; n++) {
                const float a = l[x] == 0.f ? 0.f : o[n][2 * x] * f, c = l[x] == 0.f ? 0.f : o[n][2 * x + 1] * f;
                *reinterpret_cast<uint32_t *>(mine + tile_at<DP>(m0 + (lane >> 2) + 8 * x, n) + (lane & 3) * 4) =
                    MmaOp<T>::pack(a, c);
            }
        }
        __syncwarp();
        T *const out = (T *)p.out + b * p.ob + (int64_t)hk * p.group * p.oh;
        const int per = P.wo == 16 ? 8 : P.wo == 4 ? 2 : 1, units = p.d / per;
        for (int idx = lane; idx < 16 * units; idx += 32) {
            const int r = idx / units, c = (idx - r * units) * per, row = row0 + m0 + r, i = row / p.group;
            if (row >= rows) break;
            T *dst = out + i * p.ot + (row - i * p.group) * p.oh + c;
            const char *src = mine + tile_at<DP>(m0 + r, c >> 3) + (c & 7) * 2;
            if (per == 8)
                *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
            else if (per == 2)
                *reinterpret_cast<uint32_t *>(dst) = *reinterpret_cast<const uint32_t *>(src);
            else
                *dst = *reinterpret_cast<const T *>(src);
        }
        if (__any_sync(0xffffffffu, odd)) {
            __syncwarp();
            redo_rows_apart<T, DP>(p, {b, hk * p.group, p.group, row0 + m0, rows, qn, kn}, j_begin, j_end);
        }
        return;
    }

    // ---- KEYS: join the four warps, then finish or hand on this split ----
    __syncthreads();
    join_warps<T, DP>(P, b, hk, row0, rows, split, qn, kn, j_begin, j_end, o, m, l, (float *)stage0);
}

constexpr int kMaxSplits = 128;

// Joins the splits, always in the same order: a block a row, whose warps take every fourth split each
// with four of them in flight.
template <typename T>
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ MmaDev P)
{
    __shared__ float f[kMaxSplits], wm[4], wl[4], wo[4][256];
    const AttnDev &p = P.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bh = blockIdx.x / P.rows;
    const int row = (int)(blockIdx.x - bh * P.rows), b = bh / p.hk, hk = (int)(bh - (uint32_t)b * p.hk);
    const int i = row / p.group, h = hk * p.group + row - i * p.group;
    const int64_t slot = (int64_t)blockIdx.x * P.nsplit;
    if (i >= q_count(p, b)) return;
    griddep_wait();  // launched while the splits may still run
    const float2 ml = tid < P.nsplit ? P.part_ml[slot + tid] : make_float2(-INFINITY, 0.f);
    float top = ml.x;
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (lane == 0) wm[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    f[tid] = exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
    float sum = ml.y * f[tid];
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) wl[warp] = sum;
    __syncthreads();
    sum = (wl[0] + wl[1]) + (wl[2] + wl[3]);
    for (int c = lane; c < p.d; c += 32) {
        float a = 0.f;
#pragma unroll 4
        for (int s = warp; s < P.nsplit; s += 4) a = fmaf(P.part[(slot + s) * p.d + c], f[s], a);
        wo[warp][c] = a;
    }
    __syncthreads();
    T *dst = (T *)p.out + b * p.ob + i * p.ot + h * p.oh;
    const float g = sum == 0.f ? 0.f : 1.f / sum;
    for (int c = tid; c < p.d; c += 128)
        dst[c] = from_f<T>(sum == 0.f ? 0.f : ((wo[0][c] + wo[1][c]) + (wo[2][c] + wo[3][c])) * g);
}

}  // namespace dev
}  // namespace ajib
