// pages_codes.h — a store's arguments, and the store into pages of 8 bits (host side, C++).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.h"

struct e2c_store_args {
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;
    void *q_out;
    int64_t ldo;
    const float *cs, *sn;
    int positions, half, inter;
    const int32_t *pos;  // rotary positions, or null: the rows' places
    const int32_t *seqs, *q_start;
    int n, T, H;
    e2c_pages pc;  // k and v at the layer
    int *status;
};

int e2c_store_codes(const e2c_store_args &a, int x_type, int q_type, cudaStream_t st);
