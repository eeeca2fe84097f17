// attention_sight.cu — the attention kernels (attention_pages.cuh) of rows that see a window and the first
// tokens of their text, or a tree of drafted tokens behind it.
#include "attention_pages.cuh"

int e2c_attn_sight(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    return run_kind<SIGHT>(a, q, ldq, prefix, sms, st);
}
