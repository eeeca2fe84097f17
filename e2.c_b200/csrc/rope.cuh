// rope.cuh — what the kernels over the heads of token rows share (rope.cu, pages_codes.cu): which elements of a
// head a thread owns, their loads and stores as they lie in memory, and the rotation of its pairs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.h"
#include "ptx.cuh"

namespace {

constexpr int HPT = 4;      // heads per thread
constexpr int BLOCK = 128;  // threads per block: decode-sized calls spread over more SMs than with 256

template <typename T>
E2C_DEV float to_f(T x);
template <>
E2C_DEV float to_f(float x) {
    return x;
}
template <>
E2C_DEV float to_f(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <>
E2C_DEV float to_f(__half x) {
    return __half2float(x);
}
template <typename T>
E2C_DEV T from_f(float x);
template <>
E2C_DEV float from_f(float x) {
    return x;
}
template <>
E2C_DEV __nv_bfloat16 from_f(float x) {
    return __float2bfloat16_rn(x);
}
template <>
E2C_DEV __half from_f(float x) {
    return __float2half_rn(x);
}

// N consecutive values; N * sizeof(T) is a multiple of 16 with 16-byte alignment, or N = 1
template <typename T, int N>
E2C_DEV void store(T *p, const float (&r)[N]) {
    if constexpr (N == 1) {
        *p = from_f<T>(r[0]);
    } else {
        constexpr int PER = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += PER) {
            uint4 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int j = 0; j < PER; j++) e[j] = from_f<T>(r[i + j]);
            *reinterpret_cast<uint4 *>(p + i) = w;
        }
    }
}

// N values as they lie in memory
template <typename T, int N>
struct Raw {
    static constexpr int WORDS = N == 1 ? 0 : N * sizeof(T) / 16;
    uint4 w[WORDS ? WORDS : 1];
    T one;
    E2C_DEV void get(const T *p) {
        if constexpr (N == 1) {
            one = *p;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) w[i] = reinterpret_cast<const uint4 *>(p)[i];
        }
    }
    E2C_DEV void floats(float (&r)[N]) const {
        if constexpr (N == 1) {
            r[0] = to_f<T>(one);
        } else {
            const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
            for (int i = 0; i < N; i++) r[i] = to_f<T>(e[i]);
        }
    }
    // to y: bit for bit where the types are the same
    template <typename TO>
    E2C_DEV void copy(TO *y) const {
        if constexpr (std::is_same<T, TO>::value && N > 1) {
#pragma unroll
            for (int i = 0; i < WORDS; i++) reinterpret_cast<uint4 *>(y)[i] = w[i];
        } else {
            float r[N];
            floats(r);
            store<TO, N>(y, r);
        }
    }
};

// u / d for u < 2^31 by a multiplication
struct Div {
    uint32_t d, mul, shift;
};
E2C_DEV uint32_t div_by(uint32_t u, const Div &v) { return v.d == 1 ? u : (uint32_t)(__umulhi(u, v.mul) >> v.shift); }

// A thread's part of each of its heads: V elements from e0 on and V from e1 on, which neighbouring threads
// continue; together V pairs, or some of the dimensions that pass through.
struct Part {
    int e0, e1;
    bool two, turn;  // there is a second run; it is rotated
};
template <int V>
E2C_DEV Part part_of(int j, int half, int units, int D, bool inter) {
    const int nrot = half / V;
    if (j < nrot && V == 1 && inter) return {2 * j, 2 * j + 1, true, true};
    if (j < nrot) return {j * V, half + j * V, true, true};
    const int e0 = 2 * half + (j - nrot) * V, e1 = e0 + (units - nrot) * V;
    return {e0, e1, e1 < D, false};
}
// the angles of unit j's V pairs: those of its first run and those of its second
template <int V>
E2C_DEV void angles(const float *t, int j, int half, bool inter, float (&r)[V]) {
    if constexpr (V == 1) {
        r[0] = t[j];
    } else {
        const float *a = t + (inter ? j * V / 2 : j * V), *b = inter ? a + half / 2 : a + V / 2;
        using Half = std::conditional_t<V == 8, float4, float2>;
        static_assert(sizeof(Half) * 2 == sizeof r, "16-bit or 32-bit results");
        reinterpret_cast<Half *>(r)[0] = *reinterpret_cast<const Half *>(a);
        reinterpret_cast<Half *>(r)[1] = *reinterpret_cast<const Half *>(b);
    }
}
template <typename TI, typename TO, int V>
E2C_DEV void turn(const Raw<TI, V> &x0, const Raw<TI, V> &x1, TO *y0, TO *y1, bool inter, const float (&c)[V],
                  const float (&s)[V]) {
    float a[V], b[V], u[V], w[V];
    x0.floats(a);
    x1.floats(b);
    if (!inter || V == 1) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            u[i] = a[i] * c[i] - b[i] * s[i];
            w[i] = b[i] * c[i] + a[i] * s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) {
            u[i] = a[i] * c[i / 2] - a[i + 1] * s[i / 2];
            u[i + 1] = a[i + 1] * c[i / 2] + a[i] * s[i / 2];
            w[i] = b[i] * c[(V + i) / 2] - b[i + 1] * s[(V + i) / 2];
            w[i + 1] = b[i + 1] * c[(V + i) / 2] + b[i] * s[(V + i) / 2];
        }
    }
    store<TO, V>(y0, u);
    store<TO, V>(y1, w);
}

int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 0;
    e2c_set_msg("%s launch: %s", what, cudaGetErrorString(e));
    return -2;
}

Div divide_by(int d) {
    int s = 0;
    while ((1ll << s) < d) s++;
    // ceil(2^(31 + s) / d) < 2^32: right for every u < 2^31
    return {(uint32_t)d, (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), (uint32_t)(s ? s - 1 : 0)};
}

bool fits16(const void *p, int64_t ld, int bytes) { return ((uintptr_t)p & 15) == 0 && (ld * bytes) % 16 == 0; }

}  // namespace
