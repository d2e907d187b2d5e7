/*
 * attention_tc_run.h — launches of the tcgen05 attention kernel, one translation unit a type
 * (attention_tc_f16.cu, attention_tc_bf16.cu).
 */
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "attention_tc.cuh"

namespace ajib {

int sm_count();      // conv.cu
int *status_word();  // conv.cu

constexpr int kMaxSmem = 227 * 1024;

template <typename K>
cudaError_t allow_smem(K kernel, int smem, std::atomic<uint64_t> &done)
{
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return cudaErrorInvalidDevice;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load() & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

cudaError_t attn_tc_f16(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s);
cudaError_t attn_tc_bf16(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s);

template <typename T, int DP, int FORM>
cudaError_t run_tc(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s)
{
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(dev::k_attn_tc<T, DP, FORM>, kMaxSmem, done);
    if (e != cudaSuccess) return e;
    p.words = TcCfg<DP>::bit_words(op);
    p.table_st = TcCfg<DP>::table_stride(op);
    const unsigned blocks = (unsigned)std::min<int64_t>(p.items, sm_count() * TcCfg<DP>::BLOCKS);
    dev::k_attn_tc<T, DP, FORM><<<blocks, kTcThreads, (int)TcCfg<DP>::smem(op), s>>>(p, m[0], m[1], m[2]);
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t run_tc_form(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s)
{
    const bool cap = op->cap > 0;
    if (!p.scaled) return run_tc<T, DP, kFormPlain>(p, op, m, s);
    if (cap && p.bias_form == kBiasNone) return run_tc<T, DP, kFormCap>(p, op, m, s);
    if (!cap && p.bias_form == kBiasSlope) return run_tc<T, DP, kFormSlope>(p, op, m, s);
    if (!cap && p.bias_form == kBiasGridDirect) return run_tc<T, DP, kFormGrid>(p, op, m, s);
    return run_tc<T, DP, kFormAny>(p, op, m, s);
}

template <typename T>
cudaError_t run_tc_any(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s)
{
    return op->d <= 64 ? run_tc_form<T, 64>(p, op, m, s) : run_tc_form<T, 128>(p, op, m, s);
}

}  // namespace ajib
