// attention_pages.cu — attention of query tokens over the cached keys of their sequences.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "devstate.cuh"
#include "launch.h"
#include "pages.cuh"
#include "pdl.h"
#include "ptx.cuh"

namespace {

struct Args {
    e2c_pages pc;
    const void *q;
    int64_t ldq;
    const int32_t *seqs, *q_start;
    int n, T, H, causal, window;
    float scale;
    void *out;
    int64_t ldo;
    float *lse;
    int *status;
};

template <typename T>
E2C_DEV float f32(T x);
template <>
E2C_DEV float f32(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <>
E2C_DEV float f32(__half x) {
    return __half2float(x);
}

// one warp per (token, head): the running maximum and sum of the softmax, a key at a time
template <typename T, int D>
__global__ void __launch_bounds__(128) k_attention_pages(const Args p) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(u / p.H), h = (int)(u - (int64_t)t * p.H);
    if (t >= p.T) return;
    constexpr int PER = D / 32;
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
    const int seq = i < 0 ? -1 : p.seqs[i];
    const bool ok = (unsigned)seq < (unsigned)p.pc.max_seqs;
    if (!ok && lane == 0) record_status(p.status, E2C_ERR_BAD_SEQ);
    const int len = ok ? min(p.pc.len[seq], p.pc.max_blocks * p.pc.page) : 0, pos = len - (last - t);
    int lo = 0, hi = len;
    if (p.causal) hi = min(hi, pos + 1);
    if (p.window >= 0) {
        lo = max(lo, pos - p.window);
        hi = (int)min((int64_t)hi, (int64_t)pos + p.window + 1);
    }
    const T *q = static_cast<const T *>(p.q) + t * p.ldq + h * D;
    float x[PER], o[PER] = {};
#pragma unroll
    for (int e = 0; e < PER; e++) x[e] = f32(q[lane + 32 * e]) * p.scale;
    float m = -INFINITY, l = 0.f;
    const int kvh = h / (p.H / p.pc.KV);
    for (int j = lo; j < hi; j++) {
        const int page = p.pc.table[(int64_t)seq * p.pc.max_blocks + j / p.pc.page];
        if ((unsigned)page >= (unsigned)p.pc.n_pages) continue;
        const int64_t row = (((int64_t)page * p.pc.page + j % p.pc.page) * p.pc.KV + kvh) * D;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) s += x[e] * f32(static_cast<const T *>(p.pc.k)[row + lane + 32 * e]);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float mn = fmaxf(m, s);
        const float a = m == -INFINITY ? 0.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(s - mn);
        l = l * a + w;
        m = mn;
#pragma unroll
        for (int e = 0; e < PER; e++) o[e] = o[e] * a + w * f32(static_cast<const T *>(p.pc.v)[row + lane + 32 * e]);
    }
    T *y = static_cast<T *>(p.out) + t * p.ldo + h * D;
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < PER; e++) y[lane + 32 * e] = T(o[e] * inv);
    if (p.lse && lane == 0) p.lse[(int64_t)t * p.H + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

template <typename T>
void launch(const Args &a, int D, cudaStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.T * a.H + 3) / 4));
    if (D == 64) e2c_launch(k_attention_pages<T, 64>, grid, dim3(128), 0, st, a);
    if (D == 128) e2c_launch(k_attention_pages<T, 128>, grid, dim3(128), 0, st, a);
    if (D == 256) e2c_launch(k_attention_pages<T, 256>, grid, dim3(128), 0, st, a);
}

}  // namespace

extern "C" size_t e2c_pages_attention_ws_bytes(int n, int T, int max_q, int H, int KV, int D, int shared) { return 0; }

extern "C" int e2c_pages_attention(const e2c_pages *pc, const void *q, int64_t ldq, const int32_t *seqs, const int32_t *q_start, int n,
                                   int T, int max_q, int H, int shared, int causal, int window, float scale, void *out, int64_t ldo,
                                   float *lse, void *ws, size_t ws_bytes, int *status, void *stream) {
    if (T <= 0) return 0;
    const Args a = {*pc, q, ldq, seqs, q_start, n, T, H, causal, window, scale, out, ldo, lse, status};
    if (pc->type == E2C_BF16)
        launch<__nv_bfloat16>(a, pc->D, (cudaStream_t)stream);
    else
        launch<__half>(a, pc->D, (cudaStream_t)stream);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        e2c_set_msg("pages_attention launch: %s", cudaGetErrorString(e));
        return -2;
    }
    return 0;
}
