/* attention_tc_f16.cu — the tcgen05 attention kernels of one type (attention_tc.cuh). */
#include "attention_tc_run.h"

cudaError_t ajib::attn_tc_f16(TcDev &p, const ajib_attn *op, const CUtensorMap (&m)[3], cudaStream_t s)
{
    return run_tc_any<__half>(p, op, m, s);
}
