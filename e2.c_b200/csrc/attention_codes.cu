// attention_codes.cu — the attention kernels (attention_pages.cuh) over pages of 8 bits, whatever the rows see.
#include "attention_pages.cuh"

int e2c_attn_codes(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    return run_kind<SIGHT | CODES>(a, q, ldq, prefix, sms, st);
}
