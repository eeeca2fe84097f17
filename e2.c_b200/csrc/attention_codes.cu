#include "attention_pages.cuh"
int e2c_attn_codes(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    e2c_set_msg("pages_attention: pages of 8 bits");
    return -1;
}
