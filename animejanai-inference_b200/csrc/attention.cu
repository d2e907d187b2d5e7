/*
 * attention.cu — attention (include/aji_b200.h, ajib_attention_launch): argument checks, the choice
 * of kernel and the launches.
 */
#include <cuda_runtime.h>

#include <cmath>

#include "attention.cuh"
#include "heads.h"

namespace ajib {
namespace {

using namespace dev;

constexpr int kRowWarps = 8;

// One warp per query of a head: any d, alignment and stride.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) k_attn_rows(const __grid_constant__ AttnDev p, int64_t rows)
{
    __shared__ float qs[kRowWarps][kMaxHeadDim];
    const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int64_t bh = row / p.lq;
    const int i = (int)(row - bh * p.lq), b = (int)(bh / p.hq), h = (int)(bh - (int64_t)b * p.hq);
    const int qn = q_count(p, b), kn = k_count(p, b);
    if (i >= qn) return;
    float m, l, o[8];
    attend_row<T>(p, b, h, i, qn, kn, 0, kn, qs[threadIdx.x >> 5], m, l, o);
    T *out = (T *)p.out + b * p.ob + i * p.ot + h * p.oh;
    const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int c = (threadIdx.x & 31) + 32 * e;
        if (c < p.d) out[c] = from_f<T>(l == 0.f ? 0.f : o[e] * f);
    }
}

template <typename T>
cudaError_t run(const AttnDev &p, cudaStream_t s)
{
    const int64_t rows = (int64_t)p.batch * p.hq * p.lq, blocks = (rows + kRowWarps - 1) / kRowWarps;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    k_attn_rows<T><<<(unsigned)blocks, kRowWarps * 32, 0, s>>>(p, rows);
    return cudaGetLastError();
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
    if (!op->q_doc != !op->k_doc) return false;
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
    if (!check(op)) return 0;
    return 0;
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
    AttnDev p{};
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
    const int far = INT_MAX / 2;
    p.left = op->left < 0 || op->left > kMaxCount * 2 ? far : op->left;
    p.right = op->causal ? 0 : op->right < 0 || op->right > kMaxCount * 2 ? far : op->right;
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
    const cudaError_t e = op->dtype == AJIB_F16 ? run<__half>(p, (cudaStream_t)stream)
                                                : run<__nv_bfloat16>(p, (cudaStream_t)stream);
    if (e == cudaErrorInvalidConfiguration) return AJIB_ERR_UNSUPPORTED;
    return e == cudaSuccess ? AJIB_OK : AJIB_ERR_CUDA;
}
