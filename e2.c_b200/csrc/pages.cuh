// pages.cuh — what the kernels over a paged key/value cache share.
#pragma once
#include <stdint.h>

#include "launch.h"
#include "ptx.cuh"

// The batch entry whose query tokens hold row t (q_start[i] <= t < q_start[i + 1]), or -1; `last` gets
// q_start[i + 1]. Entries of equal length (a decode step, uniform prompts) are found at the first
// guess, others by bisection.
E2C_DEV int e2c_token_seq(const int32_t *q_start, int n, int T, int t, int &last) {
    int i = (int)((int64_t)t * n / T);
    last = q_start[i + 1];
    if (q_start[i] <= t && t < last) return i;
    int lo = 0, hi = n;  // q_start[lo] <= t < q_start[hi], if any
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (q_start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    last = q_start[lo + 1];
    return q_start[lo] <= t && t < last ? lo : -1;
}
