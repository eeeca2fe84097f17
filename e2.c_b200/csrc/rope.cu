// rope.cu — rotary positions on the heads of token rows, and the same fused with the write of a
// token's key and value into its page of the cache.
//
// A pair (a, b) of a head at position p with the angle's cos c and sin s becomes
//   a' = a c - b s,  b' = b c + a s          (its transpose, the gradient: s -> -s)
// for the rot / 2 pairs (i, i + rot/2), or (2i, 2i+1) interleaved; dimensions past rot pass through.
//
// Bound: memory. One thread owns two runs of V elements (16 bytes of the output type) at the same place of up
// to four heads of one token: the two halves of V pairs, or dimensions that pass through. A pair's cos
// and sin are read once for four heads; every access of neighbouring threads is contiguous, whatever
// is rotated in it; and loads come before the branch on what to do with them, as they lie in memory (as
// floats they took twice the registers, and with a thread's runs side by side half sectors were written:
// 16384 x 40 heads of 128 in bf16 92 us, now 57; 24000 tokens of 48 heads into pages 160, now 86).
// Further: fp32, the same heads, 106 us, 97% of the copy rate; 24000 rows of 8 heads of 256 from fp32 into pages
// 53 us; a quarter of 24 heads of 64 rotated, 20011 tokens, 29 us. Decode-sized calls are bound by
// their launch (4 us). All arithmetic is in 32 bits with one rounding at the store. Rows
// that 16-byte accesses do not fit (an odd stride, a rot whose halves are not multiples of V, an
// unaligned base) take V = 1.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.h"
#include "pages.cuh"
#include "pages_codes.h"
#include "pdl.h"
#include "ptx.cuh"
#include "rope.cuh"

namespace {

struct RopeArgs {
    const void *x;
    void *y;
    int64_t ldx, ldy;
    const float *cs, *sn;
    const int32_t *pos;
    int positions, half, T, H, D, inter, copy_rest;
    float sign;
    int *status;
};

// One thread: unit j of heads 4 hg .. 4 hg + 3, of V pairs, or past them of 2 V elements passed through
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(BLOCK) k_rope(const RopeArgs p, const Div per_token, const Div units) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t u = blockIdx.x * BLOCK + threadIdx.x;
    const int t = (int)div_by(u, per_token);
    if (t >= p.T) return;
    const uint32_t rem = u - t * per_token.d;
    const int hg = (int)div_by(rem, units), j = (int)(rem - hg * units.d);
    const int h0 = hg * HPT, nh = min(HPT, p.H - h0);
    const TI *x = static_cast<const TI *>(p.x) + t * p.ldx + (int64_t)h0 * p.D;
    TO *y = static_cast<TO *>(p.y) + t * p.ldy + (int64_t)h0 * p.D;
    const Part at = part_of<V>(j, p.half, (int)units.d, p.D, p.inter);
    Raw<TI, V> a[HPT], b[HPT];
#pragma unroll
    for (int h = 0; h < HPT; h++)
        if (h < nh) {
            a[h].get(x + h * p.D + at.e0);
            if (at.two) b[h].get(x + h * p.D + at.e1);
        }
    if (at.turn) {
        int pos = p.pos ? p.pos[t] : t;
        if ((unsigned)pos >= (unsigned)p.positions) {
            record_status(p.status, E2C_ERR_BAD_POSITION);
            pos = 0;
        }
        alignas(16) float c[V], s[V];
        angles<V>(p.cs + (int64_t)pos * p.half, j, p.half, p.inter, c);
        angles<V>(p.sn + (int64_t)pos * p.half, j, p.half, p.inter, s);
#pragma unroll
        for (int i = 0; i < V; i++) s[i] *= p.sign;
#pragma unroll
        for (int h = 0; h < HPT; h++)
            if (h < nh) turn<TI, TO, V>(a[h], b[h], y + h * p.D + at.e0, y + h * p.D + at.e1, p.inter, c, s);
    } else {
#pragma unroll
        for (int h = 0; h < HPT; h++)
            if (h < nh) {
                a[h].copy(y + h * p.D + at.e0);
                if (at.two) b[h].copy(y + h * p.D + at.e1);
            }
    }
}


// One thread: unit j of up to four heads of one token, as k_rope; the heads are H query heads and KV
// key heads (rotated) and KV value heads (passed through). The input loads are issued before the
// chain of lookups (token -> sequence -> length -> page) that the stores wait for.
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(BLOCK) k_pages_store(const e2c_store_args p, const Div per_token, const Div units, const Div vunits, int qgroups, int kgroups) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t u = blockIdx.x * BLOCK + threadIdx.x;
    const int t = (int)div_by(u, per_token);
    if (t >= p.T) return;
    const uint32_t rem = u - t * per_token.d, rot_units = units.d * (qgroups + kgroups);
    const int D = p.pc.D, KV = p.pc.KV;
    const bool is_v = rem >= rot_units;
    const uint32_t r2 = is_v ? rem - rot_units : rem;
    int hg = (int)div_by(r2, is_v ? vunits : units);
    const int j = (int)(r2 - hg * (is_v ? vunits.d : units.d));
    const bool is_q = !is_v && hg < qgroups;
    if (!is_v && !is_q) hg -= qgroups;
    const int h0 = hg * HPT, nh = min(HPT, (is_q ? p.H : KV) - h0);
    const TI *x = is_q ? static_cast<const TI *>(p.q) + t * p.ldq
                       : is_v ? static_cast<const TI *>(p.v) + t * p.ldv : static_cast<const TI *>(p.k) + t * p.ldk;
    x += (int64_t)h0 * D;
    const Part part = is_v ? part_of<V>(j, 0, (int)vunits.d, D, false) : part_of<V>(j, p.half, (int)units.d, D, p.inter);
    Raw<TI, V> a[HPT], b[HPT];
#pragma unroll
    for (int h = 0; h < HPT; h++)
        if (h < nh) {
            a[h].get(x + h * D + part.e0);
            if (part.two) b[h].get(x + h * D + part.e1);
        }
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
    const int seq = i < 0 ? -1 : p.seqs[i];
    const bool ok = (unsigned)seq < (unsigned)p.pc.max_seqs;
    const int at = ok ? p.pc.len[seq] - (last - t) : -1;
    // a token without a place (its sequence is not in the cache, or is shorter than its queries, or
    // longer than the table or the rotary table) is not written
    const int turn_at = p.pos && at >= 0 ? p.pos[t] : at;
    if (at < 0 || (unsigned)turn_at >= (unsigned)p.positions) {
        record_status(p.status, at < 0 ? E2C_ERR_BAD_SEQ : E2C_ERR_BAD_POSITION);
        return;
    }
    TO *y;
    if (is_q) {
        y = static_cast<TO *>(p.q_out) + t * p.ldo;
    } else {
        const int blk = at / p.pc.page, page = blk < p.pc.max_blocks ? p.pc.table[(int64_t)seq * p.pc.max_blocks + blk] : -1;
        if ((unsigned)page >= (unsigned)p.pc.n_pages) {
            record_status(p.status, E2C_ERR_BAD_SEQ);
            return;
        }
        const int64_t row = (int64_t)page * p.pc.page + (at - blk * p.pc.page);
        y = static_cast<TO *>(is_v ? p.pc.v : p.pc.k) + row * (KV * D);
    }
    y += (int64_t)h0 * D;
    if (part.turn) {
        alignas(16) float c[V], s[V];
        angles<V>(p.cs + (int64_t)turn_at * p.half, j, p.half, p.inter, c);
        angles<V>(p.sn + (int64_t)turn_at * p.half, j, p.half, p.inter, s);
#pragma unroll
        for (int h = 0; h < HPT; h++)
            if (h < nh) turn<TI, TO, V>(a[h], b[h], y + h * D + part.e0, y + h * D + part.e1, p.inter, c, s);
    } else {
#pragma unroll
        for (int h = 0; h < HPT; h++)
            if (h < nh) {
                a[h].copy(y + h * D + part.e0);
                if (part.two) b[h].copy(y + h * D + part.e1);
            }
    }
}

struct Freqs {
    double f[256];
};

// cos and sin of position * frequency, in 64 bits: at position 10^6 a 32-bit product would be off by
// 0.06 radians. That arithmetic is what bounds it (32768 positions of 64 pairs 22.5 us, 262144 135 us, where
// writing them takes 2.6 and 21); a program makes its table once.
__global__ void __launch_bounds__(256) k_rope_table(float *cs, float *sn, int64_t total, int half, const __grid_constant__ Freqs fr,
                                                    double gain) {
    griddep_launch_dependents();
    griddep_wait();
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= total) return;
    const int64_t p = u / half;
    double s, c;
    sincos((double)p * fr.f[u - p * half], &s, &c);
    cs[u] = (float)(c * gain);
    sn[u] = (float)(s * gain);
}

template <typename TI, typename TO>
int rope_as(const RopeArgs &a, bool vec, cudaStream_t st) {
    constexpr int VV = 16 / sizeof(TO);
    const int V = vec ? VV : 1;
    const int rest = a.copy_rest ? (a.D - 2 * a.half) / V : 0;
    const int units = a.half / V + (rest + 1) / 2, hgroups = (a.H + HPT - 1) / HPT;
    const int64_t total = (int64_t)a.T * units * hgroups;
    if (total == 0) return 0;
    const int64_t blocks = (total + BLOCK - 1) / BLOCK;
    if (total > 0x7fffffff - BLOCK) {
        e2c_set_msg("rope: %d tokens of %d heads are too many for one call", a.T, a.H);
        return -1;
    }
    const Div per = divide_by(units * hgroups), by = divide_by(units);
    if (vec)
        e2c_launch_as(true, k_rope<TI, TO, VV>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, by);
    else
        e2c_launch_as(true, k_rope<TI, TO, 1>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, by);
    return launched("rope");
}

template <typename TI, typename TO>
int store_as(const e2c_store_args &a, bool vec, cudaStream_t st) {
    constexpr int VV = 16 / sizeof(TO);
    const int V = vec ? VV : 1, D = a.pc.D;
    const int units = a.half / V + ((D - 2 * a.half) / V + 1) / 2, vunits = (D / V + 1) / 2;
    const int qg = (a.H + HPT - 1) / HPT, kg = (a.pc.KV + HPT - 1) / HPT, per_token = units * (qg + kg) + vunits * kg;
    const int64_t total = (int64_t)a.T * per_token, blocks = (total + BLOCK - 1) / BLOCK;
    if (total > 0x7fffffff - BLOCK) {
        e2c_set_msg("pages_store: %d tokens of %d heads are too many for one call", a.T, a.H);
        return -1;
    }
    const Div per = divide_by(per_token), by = divide_by(units), vby = divide_by(vunits);
    if (vec)
        e2c_launch_as(true, k_pages_store<TI, TO, VV>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, by, vby, qg, kg);
    else
        e2c_launch_as(true, k_pages_store<TI, TO, 1>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, by, vby, qg, kg);
    return launched("pages_store");
}

}  // namespace

extern "C" int e2c_rope_table(float *cs, float *sn, int positions, int half, const double *freq, double gain, void *stream) {
    Freqs fr;
    for (int i = 0; i < half; i++) fr.f[i] = freq[i];
    const int64_t total = (int64_t)positions * half;
    e2c_launch_as(true, k_rope_table, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (cudaStream_t)stream, cs, sn, total, half, fr,
               gain);
    return launched("rope_table");
}

extern "C" int e2c_rope(const void *x, int64_t ldx, int x_type, void *y, int64_t ldy, int y_type, const float *cs, const float *sn,
                        int positions, int half, const int32_t *pos, int T, int H, int D, int inter, int transpose, int *status,
                        void *stream) {
    RopeArgs a = {x, y, ldx, ldy, cs, sn, pos, positions, half, T, H, D, inter, x != y, transpose ? -1.f : 1.f, status};
    const int xb = x_type == E2C_F32 ? 4 : 2, yb = y_type == E2C_F32 ? 4 : 2, V = 16 / yb;
    const bool vec = half % V == 0 && D % V == 0 && fits16(x, ldx, xb) && fits16(y, ldy, yb) && fits16(cs, 0, 4) && fits16(sn, 0, 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (x_type == E2C_F32 && y_type == E2C_F32) return rope_as<float, float>(a, vec, st);
    if (x_type == E2C_F32 && y_type == E2C_BF16) return rope_as<float, __nv_bfloat16>(a, vec, st);
    if (x_type == E2C_F32 && y_type == E2C_F16) return rope_as<float, __half>(a, vec, st);
    if (x_type == E2C_BF16 && y_type == E2C_BF16) return rope_as<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
    if (x_type == E2C_F16 && y_type == E2C_F16) return rope_as<__half, __half>(a, vec, st);
    e2c_set_msg("rope: types %d -> %d", x_type, y_type);
    return -1;
}

extern "C" int e2c_pages_store(const e2c_pages *pc, int x_type, const void *q, int64_t ldq, const void *k, int64_t ldk,
                               const void *v, int64_t ldv, void *q_out, int q_type, int64_t ldo, const float *cs,
                               const float *sn, int positions, int half, int inter, const int32_t *pos, const int32_t *seqs, const int32_t *q_start, int n, int T, int H,
                               int *status, void *stream) {
    e2c_store_args a = {q, k, v, ldq, ldk, ldv, q_out, ldo, cs, sn, positions, half, inter, pos, seqs, q_start, n, T, H, *pc, status};
    const int xb = x_type == E2C_F32 ? 4 : 2;
    const bool vec = half % 8 == 0 && fits16(q, ldq, xb) && fits16(k, ldk, xb) && fits16(v, ldv, xb) && fits16(q_out, ldo, 2) &&
                     fits16(cs, 0, 4) && fits16(sn, 0, 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (pc->type == E2C_I8) return e2c_store_codes(a, x_type, q_type, st);
    if (pc->type == E2C_BF16)
        return x_type == E2C_F32 ? store_as<float, __nv_bfloat16>(a, vec, st) : store_as<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
    return x_type == E2C_F32 ? store_as<float, __half>(a, vec, st) : store_as<__half, __half>(a, vec, st);
}
