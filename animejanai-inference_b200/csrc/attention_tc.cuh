/*
 * attention_tc.cuh — attention of prompts and windows on the fifth-generation tensor cores (tcgen05).
 *
 * A block takes 256 queries of one head as two tiles of 128 and walks the keys in tiles (128 keys with
 * up to 128 components a head, 64 with up to 64). Warps 0-3 and 4-7 do the softmax of one query tile
 * each, a thread a row; warp 8 issues the TMA copies; warps 9 and 10 the products of a query tile each:
 *   S = Q K^T   (both from shared memory)     -> TMEM
 *   O += P V    (P from TMEM, V from shared)  -> TMEM
 * P takes the columns of S, half as many, once they are read: 128-key tiles fill TMEM's 512 columns,
 * 64-key tiles half of it, so that two blocks share an SM. (A products warp for both query tiles waited
 * for one tile's softmax while the other's was ready.) Warp 11 hands out the items (sequence, head, 256
 * queries) with their reach of keys and, where there are documents, which key tiles hold one of a
 * query tile's, two items ahead. Blocks stay and walk items, so that copies and products of the next one run
 * while the softmax warps still write the last one out.
 *
 * The running maximum a row is scaled by only follows the true one when that has grown by more than
 * 2^8: the outputs are rescaled rarely, by the softmax threads themselves, at a time when no product
 * touches them. Probabilities are then up to 2^8 instead of 1, which costs neither fp16 nor bf16 any
 * precision. They are rounded to the type of v, which the product wants of both operands (against fp32
 * probabilities a third more error at most, fp16 2.8e-4 and bf16 2.2e-3 of the outputs' size); their sum is of
 * the unrounded ones.
 *
 * What bounds it: per 256 x 128 scores the tensor pipe needs 32 * DP cycles (8192 flop a cycle) and the
 * exponentials 2048 (16 a cycle): even at DP 128, where 4096 x 4096 tokens of 16 heads take 120 us (1.14
 * PFLOP/s, 69 % of the measured matrix rate) and an 8192-token causal prompt 222 us (1.25 PFLOP/s of
 * the pairs that are seen; events, idle card). At DP 64 it is the instructions of the softmax: 11 an element
 * with a table's bias and region masks, half of the issue slots of an SM (2040 windows of 256 tokens, 6 heads of
 * 32: 550 us; 32 % of the exponential unit, 28 % of DRAM).
 *
 * Tried and left out: taking turns at the exponential unit, a quarter of the exponentials as a polynomial
 * on the FMA pipe (233 against 222 us together, they pay only while products wait for one another);
 * two passes over the scores at DP 128 (275); one block of 128-key tiles an SM at DP 64 (windows 650, prompt
 * 243 against 220).
 */
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention_mma.cuh"
#include "f32x2.cuh"

namespace ajib {

constexpr int kTcThreads = 384;

// What happens to scores beside the scale; a kernel each, as code that is jumped over costs
// instruction fetches. kFormAny looks at the op for everything.
enum { kFormPlain = 0, kFormCap = 1, kFormSlope = 2, kFormGrid = 3, kFormAny = 4 };

struct TcDev {
    AttnDev a;
    int64_t items;   // (sequence, head, 256 queries)
    int tiles;       // of 256 queries a head
    int head_major;  // blocks walk runs of items of one head (a table in shared memory), else long ones first
    int bias_form;
    int scaled;      // scores are scaled before the maximum (cap, bias, or a scale that is not positive)
    int wo;          // widest stores (bytes) of out
    int table_st;    // kBiasGridDirect: row stride of the table in shared memory
    int words;       // documents: 32-tile words a bit set has room for
    int *err;
};

template <int DP> struct TcCfg {
    static constexpr int KT = DP;                      // keys of a tile
    static constexpr int BLOCKS = DP == 64 ? 2 : 1;    // on an SM
    static constexpr int ST = DP == 64 ? 3 : 2;        // stages of keys and of values
    static constexpr int QTILE = 128 * DP * 2, TILE = KT * DP * 2, HALF = KT * 128;  // HALF: a tile's 64 components
    static constexpr int Q = 0, K = 2 * QTILE, V = K + ST * TILE, BARS = V + ST * TILE;
    static constexpr int NBAR = 4 + 4 * ST + 6 + 4 + 4;
    static constexpr int COLUMNS = 2 * KT + 2 * DP;     // of TMEM: scores of both query tiles, then outputs
    // One block of 384 threads an SM: 168 registers, of which the softmax warps take 216 and the others 72.
    // Two blocks: 80 each.
    static constexpr int REGS = 216, REGS_REST = 72;
    static constexpr int ITEMS = (BARS + NBAR * 8 + 31) / 16 * 16, MORE = ITEMS + 2 * 128;
    // behind: the bit sets (two, four words each for every 32 key tiles: seen and whole, of both query
    // tiles), or the table (one a softmax warpgroup) and its keys' places
    static int bit_words(const ajib_attn *op) { return op->q_doc ? (op->lk + KT * 32 - 1) / (KT * 32) : 0; }
    // Rows of the table start table_stride apart, so that the 32 queries of a warp, neighbours on the
    // grid, read 32 different banks.
    static int table_stride(const ajib_attn *op)
    {
        const int n = 2 * op->reach_x + 1;
        return n + ((op->grid_w - n) % 32 + 32) % 32;
    }
    static int64_t smem(const ajib_attn *op)
    {
        int64_t n = MORE + 1024 + (int64_t)bit_words(op) * 32;  // 1024: the alignment of the first tile
        if (op->bias == AJIB_BIAS_TABLE && op->grid_w)
            n += 2 * ((int64_t)table_stride(op) * (2 * op->reach_y + 1) * 4 + 16) + ((op->lk + KT - 1) / KT * KT) * 4;
        return n;
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

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// tanh of two in [-0.75, 0.75] (tanh_of's polynomial).
__device__ __forceinline__ F2 f2_tanh(F2 x)
{
    const F2 z = f2_mul(x, x);
    F2 y = f2_fma(f2(kTanh5, kTanh5), z, f2(kTanh4, kTanh4));
    y = f2_fma(y, z, f2(kTanh3, kTanh3));
    y = f2_fma(y, z, f2(kTanh2, kTanh2));
    y = f2_fma(y, z, f2(kTanh1, kTanh1));
    y = f2_fma(y, z, f2(kTanh0, kTanh0));
    return f2_mul(y, x);
}

template <int N> __device__ __forceinline__ float row_max(const float *s)
{
    float top[4];
#pragma unroll
    for (int y = 0; y < 4; y++) {
        top[y] = s[y];
#pragma unroll
        for (int c = 4 + y; c < N - 4; c += 8) top[y] = max3(top[y], s[c], s[c + 4]);
        top[y] = fmaxf(top[y], s[N - 4 + y]);
    }
    return max3(fmaxf(top[0], top[1]), top[2], top[3]);
}

// The lowest n bits of a word, n of any sign or size.
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

// One item's queries and keys, worked out by one warp for all of them.
struct __align__(16) TcItem {
    int b, h, row0, qn, kn;    // b < 0: no more items
    int shift, pre;            // query i stands at i + shift; keys below pre are seen by all
    int doc_row, word0;        // of documents: their row, and the first word of the bit sets
    int both;                  // there are queries in the second tile
    int t0, t1;                // key tiles that any query sees
    int before, before_whole;  // tiles below are seen for their prefix, in part / whole
    int full;                  // tiles below hold 128 keys
    // key tiles [from, to) are seen by some, [whole_from, whole_to) by every query of a tile
    int from0, to0, whole_from0, whole_to0, from1, to1, whole_from1, whole_to1;
};

template <int KT>
__device__ __forceinline__ void tile_range(const AttnDev &p, int first, int last, int kn, int &from, int &to, int &whole_from,
                                           int &whole_to)
{
    const bool no_left = p.left == INT_MAX / 2, no_right = p.right == INT_MAX / 2;
    from = no_left ? 0 : max(first - p.left, 0) / KT;
    to = (max(no_right ? kn : min(kn, last + p.right + 1), 0) + KT - 1) / KT;
    whole_from = no_left ? 0 : (max(last - p.left, 0) + KT - 1) / KT;
    whole_to = no_right ? INT_MAX : max(first + p.right + 1, 0) / KT;
}

template <int KT>
__device__ __forceinline__ bool item_of(const AttnDev &p, int b, int h, int tile, TcItem &x)
{
    x.b = b;
    x.h = h;
    x.qn = q_count(p, x.b);
    x.kn = k_count(p, x.b);
    x.row0 = tile * 256;
    if (x.row0 >= x.qn) return false;
    const int shift = p.align_end ? x.kn - x.qn : 0;
    const int pre = p.prefix ? min(max(__ldg(p.prefix + x.b), 0), x.kn) : 0;
    x.doc_row = p.q_doc ? b % p.doc_rows : 0;
    x.shift = shift;
    x.pre = pre;
    x.both = x.row0 + 128 < x.qn;
    const int first = x.row0 + shift, last = min(x.row0 + 256, x.qn) - 1 + shift;
    tile_range<KT>(p, first, x.both ? first + 127 : last, x.kn, x.from0, x.to0, x.whole_from0, x.whole_to0);
    tile_range<KT>(p, first + 128, last, x.kn, x.from1, x.to1, x.whole_from1, x.whole_to1);
    if (!x.both) x.to1 = 0;
    x.before = (pre + KT - 1) / KT;
    x.before_whole = pre / KT;
    x.full = x.kn / KT;
    x.t1 = max(max(x.before, x.to0), x.to1);
    // (no further: queries that stand a window past the last key reach none, and the bit sets begin at t0)
    x.t0 = min(x.before ? 0 : x.both ? min(x.from0, x.from1) : x.from0, x.t1);
    x.word0 = x.t0 / 32;
    return true;
}

// The items of a block in turn: a run of them (head_major), or one of each row of gridDim.x, every
// second row backwards, which evens out a triangle.
struct TcWalk {
    uint32_t at, end;
    int k, b, h, tile;
    __device__ __forceinline__ void start(const TcDev &P)
    {
        at = 0;
        end = (uint32_t)P.items;
        k = b = h = tile = 0;
        if (P.head_major) {
            at = (uint32_t)(P.items * blockIdx.x / gridDim.x);
            end = (uint32_t)(P.items * (blockIdx.x + 1) / gridDim.x);
            tile = at % P.tiles;
            b = at / P.tiles;
            h = b / P.a.batch;
            b -= h * P.a.batch;
        }
    }
    template <int KT> __device__ __forceinline__ bool next(const TcDev &P, TcItem &x)
    {
        const AttnDev &p = P.a;
        while (at < end) {
            bool found;
            if (P.head_major) {
                found = item_of<KT>(p, b, h, tile, x);
                at++;
                if (++tile == P.tiles) {
                    tile = 0;
                    if (++b == p.batch) {
                        b = 0;
                        h++;
                    }
                }
            } else {
                // the last queries of a prompt, which see most keys, first; heads that share keys side by side
                uint32_t item = at + (k++ & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                at += gridDim.x;
                if (item >= end) continue;
                const uint32_t row = item / p.hq, last = row / p.batch;
                found = item_of<KT>(p, row - last * p.batch, item - row * p.hq, P.tiles - 1 - (int)last, x);
            }
            if (found) return true;
        }
        return false;
    }
};

// Whether some query of tile q sees a key of tile t. bits: the item's documents, or NULL.
__device__ __forceinline__ bool tc_active(const TcItem &x, const uint32_t *bits, int q, int t)
{
    const bool reach = t < x.before ? !q || x.both : q ? t >= x.from1 && t < x.to1 : t >= x.from0 && t < x.to0;
    return reach && !(bits && !(bits[4 * (t / 32 - x.word0) + q] >> (t & 31) & 1));
}

// The bit sets of an item's documents, and its key tiles narrowed to those between the first and the
// last that holds one. One warp, a lane a key tile.
template <int KT> __device__ __forceinline__ void document_tiles(const AttnDev &p, TcItem &x, uint32_t *bits)
{
    const int lane = threadIdx.x & 31;
    const int *qd = p.q_doc + (int64_t)x.doc_row * p.lq, *kd = p.k_doc + (int64_t)x.doc_row * p.lk;
    int lo[2] = {INT_MAX, INT_MAX}, hi[2] = {INT_MIN, INT_MIN};
#pragma unroll
    for (int y = 0; y < 8; y++) {
        const int i = x.row0 + 32 * y + lane;
        if (i < x.qn) {
            const int id = __ldg(qd + i);
            lo[y >> 2] = min(lo[y >> 2], id);
            hi[y >> 2] = max(hi[y >> 2], id);
        }
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
        lo[q] = __reduce_min_sync(0xffffffffu, lo[q]);
        hi[q] = __reduce_max_sync(0xffffffffu, hi[q]);
    }
    int t_first = x.t1, t_last = x.t0 - 1;
    for (int w = x.word0; w * 32 < x.t1; w++) {
        const int t = w * 32 + lane, j = t * KT, n = min(x.kn - j, KT);
        int klo = INT_MAX, khi = INT_MIN;
        if (t >= x.t0 && t < x.t1) document_range<KT>(kd + j, n, klo, khi);
        uint32_t either = 0;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint32_t seen = __ballot_sync(0xffffffffu, khi >= 0 && max(lo[q], 0) <= khi && klo <= hi[q]);
            const uint32_t only = __ballot_sync(0xffffffffu, lo[q] >= 0 && lo[q] == hi[q] && klo == lo[q] && khi == lo[q]);
            if (lane == 0) {
                bits[4 * (w - x.word0) + q] = seen;
                bits[4 * (w - x.word0) + 2 + q] = only;
            }
            either |= seen;
        }
        if (either) {
            t_first = min(t_first, w * 32 + __ffs(either) - 1);
            t_last = max(t_last, w * 32 + 31 - __clz(either));
        }
    }
    x.t0 = min(t_first, x.t1);
    x.t1 = t_last + 1;
}

// Every item of the block again, 16 rows in turn to each of the eight softmax warps, where the output is not
// finite (attention_odd.cuh).
template <typename T, int DP> __device__ __forceinline__ void redo_items(const TcDev &P)
{
    constexpr int KT = TcCfg<DP>::KT;
    TcWalk walk;
    TcItem it;
    walk.start(P);
    while (walk.next<KT>(P, it))
        for (int q = 0, row0 = it.row0 + (threadIdx.x >> 5) * 16; q < 2 && row0 < it.qn; q++, row0 += 128) {
            // the key tiles of this query tile
            const int from = it.before ? 0 : q ? it.from1 : it.from0, to = max(it.before, q ? it.to1 : it.to0);
            redo_rows<T, DP>(P.a, {it.b, it.h, 1, row0, it.qn, it.qn, it.kn}, from * KT, min(to * KT, it.kn));
        }
}

template <typename T, int DP, int FORM>
__global__ void __launch_bounds__(kTcThreads, TcCfg<DP>::BLOCKS)
    k_attn_tc(const __grid_constant__ TcDev P, const __grid_constant__ CUtensorMap mq,
              const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv)
{
    using C = TcCfg<DP>;
    constexpr int KT = C::KT;
    const AttnDev &p = P.a;
    extern __shared__ char sm_raw[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    char *const sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
    const uint32_t s0 = smem_u32(sm);
    const uint32_t bars = s0 + C::BARS;
    const uint32_t q_full = bars, q_empty = q_full + 16, k_full = q_empty + 16, k_empty = k_full + 8 * C::ST,
                   v_full = k_empty + 8 * C::ST, v_empty = v_full + 8 * C::ST, s_full = v_empty + 8 * C::ST,
                   p_full = s_full + 16, o_full = p_full + 16,
                   item_full = o_full + 16, item_empty = item_full + 16,
                   p_half = item_empty + 16, meet = p_half + 16;
    uint32_t *const tmem_at = (uint32_t *)(sm + C::BARS + C::NBAR * 8);
    TcItem *const items = (TcItem *)(sm + C::ITEMS);
    static_assert(sizeof(TcItem) <= 128, "");
    uint32_t *const bit_sets = (uint32_t *)(sm + C::MORE);

    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_at), C::COLUMNS);
    } else if (tid == 256) {
        tma_prefetch_desc(&mq);
        tma_prefetch_desc(&mk);
        tma_prefetch_desc(&mv);
        for (uint32_t x = bars; x < meet + 16; x += 8) {
            int arrivals = 1;
            if ((x >= k_empty && x < v_full) || (x >= v_empty && x < s_full)) arrivals = 2;        // both products warps
            if ((x >= p_full && x < o_full) || x >= p_half) arrivals = 4;                          // a query tile's softmax
            if (x >= item_empty && x < p_half) arrivals = 11;                                      // all but warp 11
            mbar_init(x, arrivals);
        }
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
    const bool documents = p.q_doc != nullptr;
    int turn = 0;  // items so far (their places in shared memory alternate)
    bool ok = true;
    // The next item, from warp 11; done() gives its place back. (A wait for an item, or for the first scores of
    // one, may be for as long as another takes: up to 2^29 keys. The other waits are for a tile.)
    TcItem x;
    auto next = [&]() {
        if (!(ok = tc_wait(item_full + 8 * (turn & 1), turn >> 1 & 1, P.err, 213, p.lk / KT))) return false;
        x = items[turn & 1];
        return x.b >= 0;
    };
    auto done = [&]() { mbar_arrive(item_empty + 8 * (turn & 1)); };
    auto bits_of = [&](int n) { return documents ? bit_sets + (n & 1) * P.words * 4 : nullptr; };

    // 384 threads of 168 registers: the softmax warps take 216 (a row of 128 scores and more), 72 stay
    // for the copies, the products and the documents.
    if (warp >= 8) {
        if (C::BLOCKS == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_REST));
        if (warp == 8) {
            // ---- copies ----
            if (elect_one()) {
                int n = 0, nq[2] = {0, 0};
                bool v_here = true;  // whether the last keys' values were asked for as well
                for (; next(); turn++) {
                    const uint32_t *bits = bits_of(turn);
                    const int g = x.h / p.group;
                    bool q_here[2] = {false, false};
                    auto queries = [&](int q) {
                        if (q_here[q] || !(ok = tc_wait(q_empty + 8 * q, (nq[q] & 1) ^ 1, P.err, 200))) return;
                        mbar_arrive_expect_tx(q_full + 8 * q, C::QTILE);
                        for (int y = 0; y < DP / 64; y++)
                            tma_load_4d(s0 + C::Q + q * C::QTILE + y * 16384, &mq, q_full + 8 * q, 64 * y, x.row0 + 128 * q, x.h,
                                        x.b);
                        q_here[q] = true;
                        nq[q]++;
                    };
                    for (int t = x.t0; t < x.t1 && ok; t++) {
                        const bool act[2] = {tc_active(x, bits, 0, t), tc_active(x, bits, 1, t)};
                        if (!act[0] && !act[1]) continue;
                        const int st = n % C::ST;
                        const uint32_t parity = ((n / C::ST) & 1) ^ 1;
                        if (act[0]) queries(0);
                        if (!ok || !(ok = tc_wait(k_empty + 8 * st, parity, P.err, 201))) break;
                        mbar_arrive_expect_tx(k_full + 8 * st, C::TILE);
                        for (int y = 0; y < DP / 64; y++)
                            tma_load_4d(s0 + C::K + st * C::TILE + y * C::HALF, &mk, k_full + 8 * st, 64 * y, t * KT, g, x.b);
                        n++;
                        v_here = false;
                        if (act[1]) queries(1);
                        if (!ok || !(ok = tc_wait(v_empty + 8 * st, parity, P.err, 202))) break;
                        mbar_arrive_expect_tx(v_full + 8 * st, C::TILE);
                        for (int y = 0; y < DP / 64; y++)
                            tma_load_4d(s0 + C::V + st * C::TILE + y * C::HALF, &mv, v_full + 8 * st, 64 * y, t * KT, g, x.b);
                        v_here = true;
                    }
                    if (!ok) break;
                    done();
                }
                // every copy has landed before the block ends, also where a wait gave up
#pragma unroll
                for (int q = 0; q < 2; q++)
                    if (nq[q]) tc_wait(q_full + 8 * q, (nq[q] - 1) & 1, P.err, 203);
                for (int i = max(0, n - C::ST); i < n; i++) {
                    tc_wait(k_full + 8 * (i % C::ST), (i / C::ST) & 1, P.err, 204);
                    if (v_here || i < n - 1) tc_wait(v_full + 8 * (i % C::ST), (i / C::ST) & 1, P.err, 205);
                }
            }
        } else if (warp < 11) {
            // ---- products of query tile q ----
            const int q = warp - 9;
            // N of P V: the components, in sixteens; k of Q K^T likewise
            const int dn = (p.d + 15) / 16 * 16;
            const uint32_t id_s = idesc_of<T>(KT, false), id_o = idesc_of<T>(dn, true);
            const uint32_t s_at = tmem + KT * q, o_at = tmem + 2 * KT + DP * q;
            const uint64_t qd = swizzled_desc(s0 + C::Q + q * C::QTILE, 16);
            uint32_t phase = 0;  // of p_full (bit 0), q_full (1) and p_half (2)
            auto wait = [&](uint32_t bar, int bit, int code) {
                const bool done = tc_wait_warp(bar + 8 * q, phase >> bit & 1, P.err, code);
                phase ^= 1u << bit;
                return done;
            };
            int n = 0;            // key tiles so far, of both query tiles
            for (; __all_sync(0xffffffffu, next()); turn++) {
                const uint32_t *bits = bits_of(turn);
                bool q_here = false, acc = false;
                int n_pend = -1, t_pend = 0;  // the key tile whose scores the softmax warps have
                // O += P V of that key tile
                auto values = [&]() {
                    const int st = n_pend % C::ST;
                    if (!tc_wait_warp(v_full + 8 * st, (n_pend / C::ST) & 1, P.err, 206)) return false;
                    const int live = x.kn - t_pend * KT;
                    if (live < KT && x.kn < p.lk) {
                        // values behind the last key may be anything: zeros (from both warps), as 0 * NaN is NaN
                        for (int i = lane; i < (KT - live) * (DP / 8); i += 32) {
                            const int r = live + i / (DP / 8), c = i % (DP / 8);
                            *reinterpret_cast<uint4 *>(sm + C::V + st * C::TILE + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16) =
                                make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    const uint64_t vd = swizzled_desc(s0 + C::V + st * C::TILE, C::HALF);
                    if (!wait(p_half, 2, 218)) return false;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < KT / 32; kk++)
                            mma_f16_ts(o_at, s_at + 8 * kk, vd + (kk * 2048 >> 4), id_o, acc || kk > 0);
                    }
                    __syncwarp();
                    if (!wait(p_full, 0, 207)) return false;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = KT / 32; kk < KT / 16; kk++)
                            mma_f16_ts(o_at, s_at + 8 * kk, vd + (kk * 2048 >> 4), id_o, 1u);
                        mma_commit(v_empty + 8 * st);
                    }
                    __syncwarp();
                    acc = true;
                    n_pend = -1;
                    return true;
                };
                for (int t = x.t0; t < x.t1 && ok; t++) {
                    const bool mine = tc_active(x, bits, q, t);
                    if (!mine && !tc_active(x, bits, 1 - q, t)) continue;
                    const int st = n % C::ST;
                    if (mine) {
                        // (the scores' columns are free once the product that reads them as probabilities is issued)
                        if (n_pend >= 0 && !(ok = values())) break;
                        if (!q_here && !(ok = wait(q_full, 1, 209))) break;
                        q_here = true;
                        if (!(ok = tc_wait_warp(k_full + 8 * st, (n / C::ST) & 1, P.err, 208))) break;
                        if (elect_one()) {
                            const uint64_t kd = swizzled_desc(s0 + C::K + st * C::TILE, 16);
#pragma unroll
                            for (int kk = 0; kk < DP / 16; kk++) {
                                const uint32_t qa = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4, ka = ((kk >> 2) * C::HALF + (kk & 3) * 32) >> 4;
                                if (kk * 16 < p.d) mma_f16(s_at, qd + qa, kd + ka, id_s, kk > 0, 0);
                            }
                            mma_commit(s_full + 8 * q);
                            mma_commit(k_empty + 8 * st);
                        }
                        __syncwarp();
                        n_pend = n;
                        t_pend = t;
                    } else {
                        // the other query tile's alone; this one's last is not held back behind it
                        if (n_pend >= 0 && !(ok = values())) break;
                        // (not ahead of the copies: an arrival a stage and turn)
                        if (!(ok = tc_wait_warp(k_full + 8 * st, (n / C::ST) & 1, P.err, 208))) break;
                        if (!(ok = tc_wait_warp(v_full + 8 * st, (n / C::ST) & 1, P.err, 206))) break;
                        if (lane == 0) {
                            mbar_arrive(k_empty + 8 * st);
                            mbar_arrive(v_empty + 8 * st);
                        }
                        __syncwarp();
                    }
                    n++;
                }
                // the queries are free when the last scores are there
                if (ok && q_here && elect_one()) mma_commit(q_empty + 8 * q);
                if (ok && n_pend >= 0) ok = values();
                if (ok && acc && elect_one()) mma_commit(o_full + 8 * q);
                if (!ok) break;
                __syncwarp();
                if (lane == 0) done();
            }
            // no product is in flight when the block ends (the softmax warps do not wait where a wait gave up)
            if (!ok) {
                if (elect_one()) mma_commit(o_full + 8 * q);
                __syncwarp();
                for (int i = 0; i < 2; i++) tc_wait_warp(o_full + 8 * q, i, P.err, 212);
            }
        } else {
            // ---- items, and documents: which key tiles hold one of a query tile's, and which nothing but its only one ----
            TcWalk walk;
            walk.start(P);
            for (;; turn++) {
                const bool more = walk.next<KT>(P, x);
                if (!more) x.b = -1;
                if (!tc_wait_warp(item_empty + 8 * (turn & 1), (turn >> 1 & 1) ^ 1, P.err, 214, p.lk / KT)) break;
                if (more && documents) document_tiles<KT>(p, x, bit_sets + (turn & 1) * P.words * 4);
                if (lane == 0) items[turn & 1] = x;
                __syncwarp();
                if (lane == 0) mbar_arrive(item_full + 8 * (turn & 1));
                if (!more) break;
            }
        }
    } else {
        // ---- softmax ----
        if (C::BLOCKS == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
        const int q = warp >> 2, r_in = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + KT * q, o_at = tmem + lanes + 2 * KT + DP * q;
        const bool grid = FORM == kFormGrid || (FORM == kFormAny && P.bias_form == kBiasGridDirect);
        const bool capped = FORM == kFormCap || (FORM == kFormAny && p.cap_out > 0.f);
        const bool scaled = FORM != kFormPlain && (FORM != kFormAny || P.scaled);
        const float sc = scaled ? 1.f : p.scale;
        const bool quads = p.grid_w % 4 == 0;
        const int table_n = grid ? P.table_st * (2 * p.reach_y + 1) : 0;
        float *const table = (float *)(sm + C::MORE + P.words * 32) + q * (table_n + 3) / 4 * 4;
        int *const places = (int *)((float *)(sm + C::MORE + P.words * 32) + 2 * ((table_n + 3) / 4 * 4));
        int table_h = -1;
        if (grid) {
            // where a key's (grids a multiple of 4 wide: four keys') entry of the table is, from its query's;
            // behind the last key: the first's, which is masked
            for (int j = tid; j < (p.lk + KT - 1) / KT * KT; j += 256) {
                const int jj = j < p.lk ? j : 0, y = jj / p.grid_w, at = y * P.table_st + jj - y * p.grid_w;
                if (!quads)
                    places[j] = at;
                else if (j % 4 == 0)
                    places[j / 4] = at;
            }
            named_bar_sync(3, 256);
        }
        // Two blocks an SM: 80 registers hold 32 scores of a row at a time, read twice. One: the whole row.
        constexpr bool TWICE = C::BLOCKS == 2;
        constexpr int CH = 32, W = TWICE ? 32 : KT;
        uint32_t phase = 0;  // of s_full (bit 0), o_full (1) and meet (2)
        bool odd_rows = false;  // whether a row of this thread came out not finite
        auto together = [&]() {  // the four warps of this query tile (bounded, unlike bar.sync)
            __syncwarp();
            if (lane == 0) mbar_arrive(meet + 8 * q);
            const bool here = tc_wait_warp(meet + 8 * q, phase >> 2, P.err, 219);
            phase ^= 4;
            return here;
        };
        // With 80 registers the item stays in shared memory: its two dozen numbers are needed now and then (2040
        // windows 550 us, in registers 596). With 216 it is copied (8192-token prompt 258 us, from shared memory 270).
        using Item = typename std::conditional<C::BLOCKS == 2, const TcItem &, const TcItem>::type;
        auto here = [&]() { return (ok = tc_wait(item_full + 8 * (turn & 1), turn >> 1 & 1, P.err, 213, p.lk / KT)) && items[turn & 1].b >= 0; };
        for (; __all_sync(0xffffffffu, here()); turn++) {
            Item x = items[turn & 1];
            if (grid && table_h != x.h) {
                if (!(ok = together())) break;  // nobody reads the last head's any more
                const float *src = p.bias_data + (int64_t)x.h * (2 * p.reach_y + 1) * (2 * p.reach_x + 1);
                for (int e = tid & 127; e < table_n; e += 128) {
                    const int y = e / P.table_st, c = e - y * P.table_st;
                    if (c <= 2 * p.reach_x) table[e] = __ldg(src + y * (2 * p.reach_x + 1) + c) * kLog2e;
                }
                if (!(ok = together())) break;
                table_h = x.h;
            }
            const uint32_t *bits = bits_of(turn);
            const int i = x.row0 + 128 * q + r_in;
            const bool there = i < x.qn;
            const Query r = query_at(p, x.doc_row, x.h, min(i, x.qn - 1), x.shift, x.pre);
            const int *const docs = documents ? p.k_doc + (int64_t)x.doc_row * p.lk : nullptr;
            const float *const mine = table + (p.reach_y - r.y) * P.table_st + p.reach_x - r.x;
            float m = -INFINITY, l = 0.f;  // m: in the units of the scores; times sc it is base 2
            bool any = false;
            for (int t = x.t0; t < x.t1; t++) {
                bool seen_here = t < x.before ? !q || x.both : t >= (q ? x.from1 : x.from0) && t < (q ? x.to1 : x.to0);
                bool all = t < x.full && (t < x.before_whole || (t >= (q ? x.whole_from1 : x.whole_from0) && t < (q ? x.whole_to1 : x.whole_to0)));
                if (bits) {
                    const uint32_t word = bits[4 * (t / 32 - x.word0) + q], whole = bits[4 * (t / 32 - x.word0) + 2 + q];
                    seen_here = seen_here && (word >> (t & 31) & 1);
                    all = all && (whole >> (t & 31) & 1);
                }
                if (!seen_here) continue;
                const int j0 = t * KT;
                if (!(ok = tc_wait_warp(s_full + 8 * q, phase & 1, P.err, 210, p.lk / KT))) break;
                phase ^= 1;
                tc_fence_after();
                // Scores that are more than a scaled product are made in a first pass, CH columns at a time (a short
                // loop: unrolled over the row its instructions are fetched anew every time), and put back.
                const bool back = scaled || !all;
                float now = -INFINITY;
                if (TWICE || back) {
#pragma unroll 1
                    for (int c0 = 0; c0 < KT; c0 += CH) {
                        float s[CH];
#pragma unroll
                        for (int c = 0; c < CH; c += 32) tmem_ld32(s_at + c0 + c, s + c);
                        tmem_wait_ld();
                        if (scaled) {
                            if (capped) {
                                // where all scores are below 0.75 of the cap the polynomial does, without the other form's exponential and
                                // reciprocal
                                float far = 0.f;
#pragma unroll
                                for (int c = 0; c < CH; c += 2) far = max3(far, fabsf(s[c]), fabsf(s[c + 1]));
                                if (__all_sync(0xffffffffu, far * fabsf(p.cap_in) <= kTanhTo)) {
                                    const F2 in = f2(p.cap_in, p.cap_in), out = f2(p.cap_out, p.cap_out);
#pragma unroll
                                    for (int c = 0; c < CH; c += 2)
                                        f2_out(f2_mul(f2_tanh(f2_mul(f2(s[c], s[c + 1]), in)), out), s[c], s[c + 1]);
                                } else {
#pragma unroll
                                    for (int c = 0; c < CH; c++) s[c] = p.cap_out * tanh_of(s[c] * p.cap_in);
                                }
                            } else if (FORM != kFormGrid && !(FORM == kFormAny && grid)) {
#pragma unroll
                                for (int c = 0; c < CH; c++) s[c] *= p.scale;
                            }
                            if (FORM == kFormSlope || (FORM == kFormAny && P.bias_form == kBiasSlope)) {
                                const float d0 = (float)(r.at - j0 - c0);
#pragma unroll
                                for (int c = 0; c < CH; c++) s[c] = fmaf(-r.slope, fabsf(d0 - (float)c), s[c]);
                            } else if (FORM == kFormAny && P.bias_form == kBiasLine) {
#pragma unroll
                                for (int c = 0; c < CH; c++) s[c] += table_bias(p, r, 0, j0 + c0 + c);
                            } else if (grid) {
                                const float f = capped ? 1.f : p.scale;
                                const F2 ff = f2(f, f);
                                if (quads) {
#pragma unroll
                                    for (int c = 0; c < CH; c += 16) {
                                        const int4 at = *reinterpret_cast<const int4 *>(places + ((j0 + c0 + c) >> 2));
#pragma unroll
                                        for (int y = 0; y < 16; y += 2) {
                                            const float *e = mine + (y < 4 ? at.x : y < 8 ? at.y : y < 12 ? at.z : at.w) + (y & 3);
                                            f2_out(f2_fma(f2(s[c + y], s[c + y + 1]), ff, f2(e[0], e[1])), s[c + y], s[c + y + 1]);
                                        }
                                    }
                                } else {
#pragma unroll
                                    for (int c = 0; c < CH; c += 4) {
                                        const int4 at = *reinterpret_cast<const int4 *>(places + j0 + c0 + c);
                                        s[c] = fmaf(s[c], f, mine[at.x]);
                                        s[c + 1] = fmaf(s[c + 1], f, mine[at.y]);
                                        s[c + 2] = fmaf(s[c + 2], f, mine[at.z]);
                                        s[c + 3] = fmaf(s[c + 3], f, mine[at.w]);
                                    }
                                }
                            }
                        }
                        if (!all) {
#pragma unroll
                            for (int w = 0; w < CH; w += 32) {
                                // a bit a key: [0, below) or [lo, hi), below end, of this query's document
                                const int j = j0 + c0 + w, lo = max(r.lo, 0) - j, hi = min(r.hi == INT_MAX ? INT_MAX : r.hi - j, 31) + 1;
                                uint32_t seen = ((bits_below(hi) & ~bits_below(lo)) | bits_below(r.pre - j)) & bits_below(x.kn - j);
                                if (docs) {
                                    // one vote for each document among the warp's queries
                                    const int key = __ldg(docs + min(j + lane, x.kn - 1));
                                    for (uint32_t left = 0xffffffffu; left;) {
                                        const int id = __shfl_sync(0xffffffffu, r.doc, __ffs(left) - 1);
                                        const bool same = r.doc == id;
                                        const uint32_t of = __ballot_sync(0xffffffffu, key == id);
                                        if (same) seen &= of;
                                        left &= ~__ballot_sync(0xffffffffu, same);
                                    }
                                }
#pragma unroll
                                for (int c = 0; c < 32; c++) s[w + c] = seen >> c & 1 ? s[w + c] : -INFINITY;
                            }
                        }
                        if (TWICE) now = fmaxf(now, row_max<CH>(s));
                        if (back) {
#pragma unroll
                            for (int c = 0; c < CH; c += 16) {
                                uint32_t w[16];
#pragma unroll
                                for (int y = 0; y < 16; y++) w[y] = __float_as_uint(s[c + y]);
                                tmem_st16(s_at + c0 + c, w);
                            }
                        }
                    }
                    if (back) tmem_wait_st();
                }
                float s[W];
                if (!TWICE) {
#pragma unroll
                    for (int c = 0; c < W; c += 32) tmem_ld32(s_at + c, s + c);
                    tmem_wait_ld();
                    now = row_max<W>(s);
                }
                // (m is -inf until a row has seen a key)
                if (__any_sync(0xffffffffu, now * sc > m * sc + 8.f || (m == -INFINITY && now > m))) {
                    const float to = fmaxf(m, now), alpha = exp2_fast((m - (to == -INFINITY ? 0.f : to)) * sc);
                    if (any) {
#pragma unroll 1
                        for (int c = 0; c < p.d; c += 16) {
                            float o[16];
                            tmem_ld16(o_at + c, o);
                            tmem_wait_ld();
                            uint32_t w[16];
#pragma unroll
                            for (int y = 0; y < 16; y++) w[y] = __float_as_uint(o[y] * alpha);
                            tmem_st16(o_at + c, w);
                        }
                    }
                    l *= m == -INFINITY ? 0.f : alpha;
                    m = to;
                }
                any = true;
                const float base = m == -INFINITY ? 0.f : m * sc;
                const F2 sc2 = f2(sc, sc), base2 = f2(-base, -base);
                F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll 1
                for (int c0 = 0; c0 < KT; c0 += W) {
                    if (TWICE) {
                        tmem_ld32(s_at + c0, s);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int c = 0; c < W; c += 2) f2_out(f2_fma(f2(s[c], s[c + 1]), sc2, base2), s[c], s[c + 1]);
#pragma unroll
                    for (int c = 0; c < W; c += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int y = 0; y < 16; y++) {
                            const float a = exp2_fast(s[c + 2 * y]), z = exp2_fast(s[c + 2 * y + 1]);
                            sum[y & 1] = f2_add(sum[y & 1], f2(a, z));
                            w[y] = MmaOp<T>::pack(a, z);
                        }
                        tmem_st16(s_at + (c0 + c) / 2, w);
                        if (c0 + c == KT / 2 - 32) {
                            // the product with the first half of the values can start
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(p_half + 8 * q);
                        }
                    }
                }
                float la, lb;
                f2_out(f2_add(sum[0], sum[1]), la, lb);
                l += la + lb;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * q);
            }
            if (!ok) break;
            T *const dst = (T *)p.out + x.b * p.ob + x.h * p.oh + (int64_t)i * p.ot;
            const bool none = q && !x.both;
            __syncwarp();
            if (lane == 0) done();

            // ---- out: a thread a row ----
            if (any) {
                if (!(ok = tc_wait_warp(o_full + 8 * q, phase >> 1 & 1, P.err, 211))) break;
                phase ^= 2;
                tc_fence_after();
            }
            if (none) continue;
            // (what a query without keys has accumulated is 0 * v: not finite only where the row is taken again)
            const float f = l == 0.f ? 0.f : 1.f / l;
            bool odd = false;
            for (int c = 0; c < p.d; c += 32) {
                float o[32];
                if (any) {
                    tmem_ld32(o_at + c, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int y = 0; y < 32; y++) o[y] = 0.f;
                }
                if (p.masked) {
                    // a sum of zeros, unless something is not finite
                    float z = 0.f;
#pragma unroll
                    for (int y = 0; y < 32; y++)
                        if (c + (y & ~15) < p.d) z = fmaf(o[y], 0.f, z);
                    odd |= z != 0.f;
                }
                uint32_t w[16];
                const F2 ff = f2(f, f);
#pragma unroll
                for (int y = 0; y < 16; y++) {
                    f2_out(f2_mul(f2(o[2 * y], o[2 * y + 1]), ff), o[2 * y], o[2 * y + 1]);
                    w[y] = MmaOp<T>::pack(o[2 * y], o[2 * y + 1]);
                }
                if (!there) continue;
                // (d is a multiple of what a store holds)
                if (P.wo == 32) {
#pragma unroll
                    for (int y = 0; y < 2; y++)
                        if (c + 16 * y < p.d)
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c + 16 * y),
                                         "r"(w[8 * y]), "r"(w[8 * y + 1]), "r"(w[8 * y + 2]), "r"(w[8 * y + 3]),
                                         "r"(w[8 * y + 4]), "r"(w[8 * y + 5]), "r"(w[8 * y + 6]), "r"(w[8 * y + 7])
                                         : "memory");
                } else if (P.wo == 16) {
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (c + 8 * y < p.d)
                            *reinterpret_cast<uint4 *>(dst + c + 8 * y) =
                                make_uint4(w[4 * y], w[4 * y + 1], w[4 * y + 2], w[4 * y + 3]);
                } else if (P.wo == 4) {
#pragma unroll
                    for (int y = 0; y < 16; y++)
                        if (c + 2 * y < p.d) *reinterpret_cast<uint32_t *>(dst + c + 2 * y) = w[y];
                } else {
#pragma unroll
                    for (int y = 0; y < 32; y++)
                        if (c + y < p.d) dst[c + y] = from_f<T>(o[y]);
                }
            }
            odd_rows |= there && odd;
        }
        // Rows that are not finite (attention_odd.cuh), when the block's items are done: nobody waits for these
        // warps any more but the barrier at the end.
        if (p.masked && named_bar_any(3, 256, odd_rows)) redo_items<T, DP>(P);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLUMNS);
    }
}

}  // namespace dev
}  // namespace ajib
