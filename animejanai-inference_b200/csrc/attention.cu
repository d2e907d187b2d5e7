/*
 * attention.cu — attention (include/aji_b200.h, ajib_attention_launch): argument checks, the choice
 * of kernel and the launches.
 */
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

#include "attention_few.cuh"
#include "attention_mma.cuh"
#include "attention_tc_run.h"
#include "cuctx.h"
#include "heads.h"

namespace ajib {

int sm_count();  // conv.cu

namespace {

using namespace dev;

constexpr int kSplitTiles = 4;   // at least this many key tiles a split
constexpr int kTcQueries = 32;  // tcgen05 from here on (queries and keys)

// How an op runs, from its sizes alone (the workspace must be known before the launch).
struct Choice {
    bool few = false;   // k_attn_few, if the tensors' layout allows TMA copies
    bool tc = false;    // k_attn_tc, likewise
    bool keys = false;  // else k_attn_mma: few queries, the warps share the keys out
    int pack = 0;       // k_attn_tc on copies of q, k and v with rows of this many components
    int row_tiles = 0, key_row_tiles = 0, nsplit = 1;  // row_tiles: of 64; key_row_tiles: of 16
    int64_t rows = 0;   // of a (sequence, key head)
    size_t space = 0;
};

// Whether the table of a grid reaches every distance on it: then it is read without clamps.
bool grid_reached(const ajib_attn *op)
{
    return op->reach_x >= op->grid_w - 1 && op->reach_y >= (std::max(op->lq, op->lk) - 1) / op->grid_w;
}

size_t packed_bytes(const ajib_attn *op, int dp, int tensor)
{
    return (size_t)op->batch * (tensor ? (size_t)op->lk * op->hk : (size_t)op->lq * op->hq) * dp * 2;
}

// Whether the copies are of a size that a device may hold (of repeated sequences they need not be, and the
// number of their bytes may pass 64 bits).
bool packable(const ajib_attn *op, int dp)
{
    const __int128 most = std::max((__int128)op->lk * op->hk, (__int128)op->lq * op->hq);
    return most * op->batch * dp * 2 <= (__int128)1 << 42;
}

// Which kernel. Measured (us, 8 heads, causal; k_attn_mma / few / tc):
//   64 components, 200 tokens 12.3 / 9.0 / 14.4, 800 26 / 18 / 27; 16 sequences of 150 20 / 23 / 14
//   128 components, 500 tokens 27 / 14 / 19, 800 39 / 27 / 21
// so few while all its blocks run at once, then tc: 600 windows of 144 tokens of 6 heads 303 / 723 / 169, 464
// windows of 64 of 3 heads - / 97 / 27 (below kTcQueries few again, whose blocks hold 16 rows).
// Heads of a size that TMA cannot copy (d not a multiple of 8) are copied to padded rows for tc.
// With few queries the keys are also split until there is a block an SM, or a split has only kSplitTiles tiles of
// all the keys (a window leaves it fewer, and some splits none). Three blocks an SM where lengths are given: caches
// are then uneven as a rule, 8 of 9 to 16 thousand keys take 78 / 79 / 75 us with one / two / three and five tokens
// over them 102 / 97 / 89, but even ones lose by it (2 x 16384 keys of 8 heads of 128 33 / 37 / 39). With at least 4 / 8
// tiles a split: 4000 keys 14.2 / 16.4 us, 1500 keys 12.4 / 13.9.
bool choose(const ajib_attn *op, Choice &c)
{
    const int64_t group = op->hq / op->hk, base = (int64_t)op->batch * op->hk;
    c.rows = op->lq * group;
    if (c.rows > 1 << 30) return false;
    c.row_tiles = (int)((c.rows + 63) / 64);
    c.key_row_tiles = (int)((c.rows + 15) / 16);
    const int64_t few_blocks = base * c.key_row_tiles;
    if (base * c.row_tiles > 0x7fffffff) return false;
    c.keys = c.rows <= 64;
    const int fit = sm_count() * (op->d <= 64 ? FewCfg<64>::BLOCKS : op->d <= 128 ? FewCfg<128>::BLOCKS : FewCfg<256>::BLOCKS);
    const bool tma = op->lk && !op->q_doc && op->d % 8 == 0 && few_blocks <= 0x7fffffff;
    c.few = tma && few_blocks <= fit;
    if (!c.few && op->lq >= kTcQueries && op->lk >= kTcQueries && op->d <= 128) {
        const bool grid = op->bias == AJIB_BIAS_TABLE && op->grid_w;
        c.tc = (!grid || grid_reached(op)) && (int64_t)op->batch * op->hq * ((op->lq + 255) / 256) <= 0x7fffffff &&
               (op->d <= 64 ? TcCfg<64>::smem(op) : TcCfg<128>::smem(op)) <= kMaxSmem;
        const int dp = (op->d + 7) / 8 * 8;
        c.tc = c.tc && (op->d == dp || packable(op, dp));
        if (c.tc && op->d != dp) {
            c.pack = dp;
            for (int i = 0; i < 3; i++) c.space += packed_bytes(op, c.pack, i);
        }
    }
    if (!c.tc && c.keys) c.few = tma;  // few queries of many sequences
    if (!c.tc && (c.few || c.keys) && few_blocks) {
        const int tiles = (op->lk + kMmaKeys - 1) / kMmaKeys;
        const int64_t want = ((op->k_len ? 3 : 1) * (int64_t)sm_count() + few_blocks - 1) / few_blocks;
        c.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, tiles / kSplitTiles), kMaxSplits));
        if (few_blocks * c.nsplit > 0x7fffffff) return false;
        if (c.nsplit > 1) c.space = (size_t)(base * c.rows * c.nsplit) * (8 + (size_t)op->d * 4);
    }
    return true;
}

template <typename T, int DP, bool KEYS>
cudaError_t run_mma(const MmaDev &p, cudaStream_t s)
{
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(k_attn_mma<T, DP, KEYS>, kMaxSmem, done);
    if (e != cudaSuccess) return e;
    const int64_t blocks = (int64_t)p.a.batch * p.a.hk * p.row_tiles * (KEYS ? p.nsplit : 1);
    k_attn_mma<T, DP, KEYS><<<(unsigned)blocks, kMmaThreads, MmaCfg<DP, KEYS>::smem(p.a), s>>>(p);
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t run_few(const MmaDev &p, const CUtensorMap (&m)[3], cudaStream_t s)
{
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(k_attn_few<T, DP>, kMaxSmem, done);
    if (e != cudaSuccess) return e;
    int *const err = status_word();
    if (!err) return cudaErrorUnknown;
    const int64_t blocks = (int64_t)p.a.batch * p.a.hk * p.row_tiles * p.nsplit;
    k_attn_few<T, DP><<<(unsigned)blocks, kFewThreads, FewCfg<DP>::SMEM, s>>>(p, m[1], m[2], err);
    return cudaGetLastError();
}

struct PackDev {
    const void *src[3];
    void *dst[3];
    int64_t sb[3], st[3], sh[3], chunks[3];  // chunks: of 8 components
    int tokens[3], heads[3], d, width;
};

// Rows of d components copied to 16-byte aligned rows padded with zeros: a thread a chunk of 8.
__global__ void __launch_bounds__(256) k_pack_heads(const __grid_constant__ PackDev p)
{
    const int x = blockIdx.y, per = (p.d + 7) / 8;
    const uint16_t *src = (const uint16_t *)p.src[x];
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < p.chunks[x]; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / per, bt = row / p.heads[x];
        const int c = (int)(at - row * per) * 8, h = (int)(row - bt * p.heads[x]);
        const int64_t b = bt / p.tokens[x];
        const uint16_t *s = src + b * p.sb[x] + (bt - b * p.tokens[x]) * p.st[x] + h * p.sh[x] + c;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = 0;
            if (p.width >= 4 && c + 2 * i < p.d)
                w[i] = __ldg(reinterpret_cast<const unsigned int *>(s + 2 * i));
            else if (p.width < 4)
                w[i] = (c + 2 * i < p.d ? s[2 * i] : 0u) | (c + 2 * i + 1 < p.d ? (uint32_t)s[2 * i + 1] << 16 : 0u);
        }
        reinterpret_cast<uint4 *>(p.dst[x])[at] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// maps: of the keys and values, where k_attn_few runs
template <typename T>
cudaError_t run(MmaDev &p, const Choice &c, const CUtensorMap (*maps)[3], cudaStream_t s)
{
    const int d = p.a.d;
    cudaError_t e;
    p.row_tiles = maps || c.keys ? c.key_row_tiles : c.row_tiles;
    p.nsplit = maps || c.keys ? c.nsplit : 1;
    if (maps)
        e = d <= 64 ? run_few<T, 64>(p, *maps, s) : d <= 128 ? run_few<T, 128>(p, *maps, s) : run_few<T, 256>(p, *maps, s);
    else if (c.keys)
        e = d <= 32 ? run_mma<T, 32, true>(p, s) : d <= 64 ? run_mma<T, 64, true>(p, s)
            : d <= 128 ? run_mma<T, 128, true>(p, s) : run_mma<T, 256, true>(p, s);
    else
        e = d <= 32 ? run_mma<T, 32, false>(p, s) : d <= 64 ? run_mma<T, 64, false>(p, s)
            : d <= 128 ? run_mma<T, 128, false>(p, s) : run_mma<T, 256, false>(p, s);
    if (e != cudaSuccess || p.nsplit == 1) return e;
    const int64_t rows = (int64_t)p.a.batch * p.a.hk * p.rows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_attn_join<T>, p);
}

// A tensor map of tiles of `rows` tokens, 64 components of one head (128-byte swizzle; zeros outside).
// False if the layout does not allow one (16-byte aligned, no repeated dimension).
bool map_of(CUtensorMap *m, const ajib_heads *x, int batch, int tokens, int heads, int d, int dtype, int rows)
{
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? (Encode)fn : nullptr;
    }();
    if (!encode || heads_width(x, batch, tokens, heads, d) != 16) return false;
    const int n[3] = {tokens, heads, batch};
    const int64_t st[3] = {x->st, x->sh, x->sb};
    cuuint64_t dims[4] = {(cuuint64_t)d, 0, 0, 0}, strides[3];
    for (int i = 0; i < 3; i++) {
        if (n[i] > 1 && (st[i] <= 0 || st[i] >= 1ll << 38)) return false;
        dims[i + 1] = (cuuint64_t)n[i];
        strides[i] = n[i] > 1 ? (cuuint64_t)st[i] * 2 : 16;  // (never used)
    }
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, one[4] = {1, 1, 1, 1};
    return encode(m, dtype == AJIB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, x->p, dims,
                  strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool misaligned4(const void *p) { return ((uintptr_t)p & 3) != 0; }

// Everything but the tensors.
bool check(const ajib_attn *op)
{
    if (!op || (op->dtype != AJIB_F16 && op->dtype != AJIB_BF16)) return false;
    if (op->batch < 0 || op->lq < 0 || op->lk < 0 || op->hq < 1 || op->hk < 1 || op->hq % op->hk) return false;
    if (op->d < 1 || op->d > kMaxHeadDim) return false;
    if (op->batch > kMaxCount || op->lq > kMaxCount || op->lk > kMaxCount || op->hq > kMaxCount) return false;
    if (!std::isfinite(op->scale * dev::kLog2e) || !std::isfinite(op->cap * dev::kLog2e) || op->cap < 0) return false;
    if (op->cap > 0 && !std::isfinite(op->scale / op->cap)) return false;
    if (op->left < -1 || op->right < -1) return false;
    if (misaligned4(op->q_len) || misaligned4(op->k_len) || misaligned4(op->prefix)) return false;
    if (misaligned4(op->q_doc) || misaligned4(op->k_doc) || misaligned4(op->bias_data)) return false;
    if (op->lk && !op->q_doc != !op->k_doc) return false;  // (no keys: no ids of theirs)
    if (op->q_doc && (op->doc_rows < 1 || op->lk > 1 << 22)) return false;
    if (op->bias < AJIB_BIAS_NONE || op->bias > AJIB_BIAS_TABLE) return false;
    if (op->bias != AJIB_BIAS_NONE && !op->bias_data) return false;
    if (op->bias == AJIB_BIAS_TABLE) {
        if (op->reach_x < 0 || op->reach_y < 0 || op->grid_w < 0) return false;
        if (op->reach_x > 1 << 20 || op->reach_y > 1 << 20) return false;
        if (op->grid_w ? op->align_end != 0 : op->reach_y != 0) return false;
        if ((int64_t)(2 * op->reach_x + 1) * (2 * op->reach_y + 1) > 1 << 24) return false;
    }
    return true;
}

}  // namespace
}  // namespace ajib

using namespace ajib;

extern "C" size_t ajib_attention_workspace(const ajib_attn *op)
{
    Choice c;
    return check(op) && choose(op, c) ? c.space : 0;
}

extern "C" int ajib_attention_launch(const ajib_attn *op, const ajib_heads *q, const ajib_heads *k, const ajib_heads *v,
                                     const ajib_heads *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!check(op)) return AJIB_ERR_ARGS;
    if (!op->batch || !op->lq) return AJIB_OK;
    const int b = op->batch, d = op->d;
    if (!heads_ok(q, b, op->lq, op->hq, d) || !heads_ok(out, b, op->lq, op->hq, d)) return AJIB_ERR_ARGS;
    if (!heads_distinct(out, b, op->lq, op->hq, d) || out->p == q->p) return AJIB_ERR_ARGS;
    if (op->lk) {
        if (!heads_ok(k, b, op->lk, op->hk, d) || !heads_ok(v, b, op->lk, op->hk, d)) return AJIB_ERR_ARGS;
        if (out->p == k->p || out->p == v->p) return AJIB_ERR_ARGS;
    }
    ajib_attn uncapped;
    if (op->cap > 0 && std::fabs(op->scale / op->cap) < FLT_MIN) {  // (a subnormal loses bits; tanh is its argument here)
        uncapped = *op;
        uncapped.cap = 0;
        op = &uncapped;
    }
    Choice c;
    if (!choose(op, c)) return AJIB_ERR_UNSUPPORTED;
    if (c.space && (!workspace || workspace_bytes < c.space || ((uintptr_t)workspace & 15))) return AJIB_ERR_ARGS;
    MmaDev m{};
    AttnDev &p = m.a;
    p.q = q->p;
    p.out = out->p;
    p.qb = q->sb, p.qt = q->st, p.qh = q->sh;
    p.ob = out->sb, p.ot = out->st, p.oh = out->sh;
    if (op->lk) {
        p.k = k->p;
        p.v = v->p;
        p.kb = k->sb, p.kt = k->st, p.kh = k->sh;
        p.vb = v->sb, p.vt = v->st, p.vh = v->sh;
    }
    p.batch = b;
    p.lq = op->lq;
    p.lk = op->lk;
    p.hq = op->hq;
    p.hk = op->hk;
    p.group = op->hq / op->hk;
    p.d = d;
    p.scale = op->scale * dev::kLog2e;
    if (op->cap > 0) {
        p.cap_in = op->scale / op->cap;
        p.cap_out = op->cap * dev::kLog2e;
    }
    // (a reach that passes every distance is none; sums of a place and a reach then fit an int)
    const int far = INT_MAX / 2, most = op->lq + op->lk;
    p.left = op->left < 0 || op->left >= most ? far : op->left;
    p.right = op->causal ? 0 : op->right < 0 || op->right >= most ? far : op->right;
    p.align_end = op->align_end != 0;
    p.q_len = op->q_len;
    p.k_len = op->k_len;
    p.prefix = op->prefix;
    p.q_doc = op->q_doc;
    p.k_doc = op->k_doc;
    p.doc_rows = op->doc_rows;
    p.bias = op->bias;
    p.bias_data = op->bias_data;
    p.grid_w = op->grid_w;
    p.reach_y = op->reach_y;
    p.reach_x = op->reach_x;
    p.masked = p.left != far || p.right != far || p.q_doc;
    m.rows = (int)c.rows;
    auto copies = [&](const ajib_heads *x, int tokens, int heads) {  // of 16, 4 or 2 bytes
        const int w = heads_width(x, b, tokens, heads, d);
        return w == 8 ? 4 : w;
    };
    m.wq = copies(q, op->lq, op->hq);
    m.wo = copies(out, op->lq, op->hq);
    m.wkv = op->lk ? std::min(copies(k, op->lk, op->hk), copies(v, op->lk, op->hk)) : 16;
    const int64_t slots = (int64_t)b * op->hk * c.rows * c.nsplit;
    m.part_ml = (float2 *)workspace;
    m.part = (float *)workspace + 2 * slots;
    m.bias_form = op->bias == AJIB_BIAS_SLOPE ? kBiasSlope : kBiasNone;
    if (op->bias == AJIB_BIAS_TABLE) {
        m.bias_form = !op->grid_w ? kBiasLine : grid_reached(op) ? kBiasGridDirect : kBiasGrid;
    }
    CUtensorMap maps[3];
    const int key_tile = d <= 64 ? TcCfg<64>::KT : TcCfg<128>::KT;
    ajib_heads packed[3] = {*q, op->lk ? *k : *q, op->lk ? *v : *q};
    if (c.pack) {
        PackDev w{};
        char *to = (char *)workspace;
        int64_t most = 0;
        for (int i = 0; i < 3; i++) {
            w.src[i] = packed[i].p;
            w.dst[i] = to;
            w.sb[i] = packed[i].sb, w.st[i] = packed[i].st, w.sh[i] = packed[i].sh;
            w.tokens[i] = i ? op->lk : op->lq;
            w.heads[i] = i ? op->hk : op->hq;
            w.chunks[i] = (int64_t)b * w.tokens[i] * w.heads[i] * (c.pack / 8);
            most = std::max(most, w.chunks[i]);
            const int64_t row = (int64_t)w.heads[i] * c.pack;
            packed[i] = {to, row * w.tokens[i], row, c.pack};
            to += packed_bytes(op, c.pack, i);
        }
        w.d = d;
        w.width = std::min(m.wq, m.wkv);
        const unsigned blocks = (unsigned)std::min<int64_t>((most + 255) / 256, 16 * sm_count());
        k_pack_heads<<<dim3(blocks, 3), 256, 0, (cudaStream_t)stream>>>(w);
        if (cudaGetLastError() != cudaSuccess) return AJIB_ERR_CUDA;
    }
    const int md = c.pack ? c.pack : d;
    if (c.tc && map_of(&maps[0], &packed[0], b, op->lq, op->hq, md, op->dtype, 128) &&
        map_of(&maps[1], &packed[1], b, op->lk, op->hk, md, op->dtype, key_tile) &&
        map_of(&maps[2], &packed[2], b, op->lk, op->hk, md, op->dtype, key_tile)) {
        TcDev t{};
        t.a = p;
        t.tiles = (op->lq + 255) / 256;
        t.items = (int64_t)b * op->hq * t.tiles;
        t.bias_form = m.bias_form;
        t.head_major = m.bias_form == kBiasGridDirect;
        t.scaled = op->cap > 0 || op->bias != AJIB_BIAS_NONE || !(op->scale > 0);
        const uint64_t rows = (uint64_t)(uintptr_t)out->p | (uint64_t)d * 2 | (uint64_t)(b > 1 ? out->sb : 0) * 2 |
                              (uint64_t)out->st * 2 | (uint64_t)(op->hq > 1 ? out->sh : 0) * 2;
        t.wo = rows % 32 == 0 ? 32 : m.wo;
        t.err = status_word();
        if (!t.err) return AJIB_ERR_CUDA;
        const cudaError_t e = op->dtype == AJIB_F16 ? attn_tc_f16(t, op, maps, (cudaStream_t)stream)
                                                    : attn_tc_bf16(t, op, maps, (cudaStream_t)stream);
        return e == cudaSuccess ? AJIB_OK : AJIB_ERR_CUDA;
    }
    m.plain = m.bias_form == kBiasNone && !(op->cap > 0);
    const bool few = c.few && map_of(&maps[1], k, b, op->lk, op->hk, d, op->dtype, kMmaKeys) &&
                     map_of(&maps[2], v, b, op->lk, op->hk, d, op->dtype, kMmaKeys);
    const cudaError_t e = op->dtype == AJIB_F16 ? run<__half>(m, c, few ? &maps : nullptr, (cudaStream_t)stream)
                                                : run<__nv_bfloat16>(m, c, few ? &maps : nullptr, (cudaStream_t)stream);
    return e == cudaSuccess ? AJIB_OK : AJIB_ERR_CUDA;
}
