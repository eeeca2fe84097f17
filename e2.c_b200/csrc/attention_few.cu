// attention_few.cu — the attention kernels for entries of few rows (attention_few.cuh) over pages of 16 bits.
#include "attention_few.cuh"

int e2c_attn_few(const e2c_attn_args &a, const void *q, int64_t ldq, int sms, cudaStream_t st) {
    return a.q_type == E2C_BF16 ? few_of<__nv_bfloat16, false>(a, q, ldq, sms, st) : few_of<__half, false>(a, q, ldq, sms, st);
}
