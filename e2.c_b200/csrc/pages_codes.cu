// pages_codes.cu — pages of 8 bits: a token's rotated key and its value quantised as they are written, and
// read back; and the reading back of 16-bit pages.
//
// A head x of D values becomes codes c = round(127 x / amax) and a scale s = amax / 127, and stands for s c. D / 16
// neighbouring threads hold a head, 16 values each in registers: the largest magnitude is a maximum over their lanes,
// and every value is read and every code written once. Rotation and quantisation are rounded step by step, without
// contraction, so that a code depends on nothing but its head (a value between two codes goes to the even one).
//
// Bound: memory, and the chain of lookups (row -> sequence -> length -> page) for a few rows. As in rope.cu a thread takes
// four heads, whose loads come before the lookups.
#include "pages_codes.h"

#include "pages.cuh"
#include "pdl.h"
#include "rope.cuh"
#include "rowmath.cuh"

namespace {

// 2^-100: below it 127 / amax would leave fp32's range; a head that small is held as zeros
constexpr float kLeast = 0x1p-100f;

// Sixteen values of a head: the two runs of part_of (VEC), or every (D / 16)-th value from j on.
template <typename TI, bool VEC>
struct Sixteen {
    Raw<TI, VEC ? 8 : 1> a[VEC ? 1 : 16], b[VEC ? 1 : 16];
    E2C_DEV static int element(const Part &at, int j, int lanes, int i) { return VEC ? (i < 8 ? at.e0 + i : at.e1 + i - 8) : j + lanes * i; }
    E2C_DEV void get(const TI *x, const Part &at, int j, int lanes, int half, bool inter) {
        if constexpr (VEC) {
            a[0].get(x + at.e0);
            b[0].get(x + at.e1);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int e = j + lanes * i;
                a[i].get(x + e);
                // the other value of its pair
                if (e < 2 * half) b[i].get(x + (inter ? e ^ 1 : e < half ? e + half : e - half));
            }
        }
    }
    // the values, rotated where they are part of the first 2 half ones
    E2C_DEV void floats(float (&r)[16], const Part &at, int j, int lanes, int half, bool inter, const float *cs, const float *sn) const {
        if constexpr (VEC) {
            float u[8], w[8];
            a[0].floats(u);
            b[0].floats(w);
            if (!at.turn) {
#pragma unroll
                for (int i = 0; i < 8; i++) r[i] = u[i], r[8 + i] = w[i];
                return;
            }
            alignas(16) float c[8], s[8];
            angles<8>(cs, j, half, inter, c);
            angles<8>(sn, j, half, inter, s);
            if (!inter) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    r[i] = __fsub_rn(__fmul_rn(u[i], c[i]), __fmul_rn(w[i], s[i]));
                    r[8 + i] = __fadd_rn(__fmul_rn(w[i], c[i]), __fmul_rn(u[i], s[i]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    r[i] = __fsub_rn(__fmul_rn(u[i], c[i / 2]), __fmul_rn(u[i + 1], s[i / 2]));
                    r[i + 1] = __fadd_rn(__fmul_rn(u[i + 1], c[i / 2]), __fmul_rn(u[i], s[i / 2]));
                    r[8 + i] = __fsub_rn(__fmul_rn(w[i], c[4 + i / 2]), __fmul_rn(w[i + 1], s[4 + i / 2]));
                    r[9 + i] = __fadd_rn(__fmul_rn(w[i + 1], c[4 + i / 2]), __fmul_rn(w[i], s[4 + i / 2]));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int e = j + lanes * i;
                float x[1], y[1];
                a[i].floats(x);
                if (e >= 2 * half) {
                    r[i] = x[0];
                    continue;
                }
                b[i].floats(y);
                const int pair = inter ? e >> 1 : e < half ? e : e - half;
                const bool second = inter ? e & 1 : e >= half;
                const float c = cs[pair], s = sn[pair];
                r[i] = second ? __fadd_rn(__fmul_rn(x[0], c), __fmul_rn(y[0], s)) : __fsub_rn(__fmul_rn(x[0], c), __fmul_rn(y[0], s));
            }
        }
    }
};

E2C_DEV uint32_t four(const float *r, float inv) {
    return (uint32_t)(qround(r[0], inv) & 255) | (uint32_t)(qround(r[1], inv) & 255) << 8 | (uint32_t)(qround(r[2], inv) & 255) << 16 |
           (uint32_t)(qround(r[3], inv) & 255) << 24;
}

// One thread: lane j of D / 16 of up to four heads of one token, as k_pages_store
template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(BLOCK) k_store_codes(const e2c_store_args p, const Div per_token, int shift, int qgroups, int kgroups) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t u = blockIdx.x * BLOCK + threadIdx.x;
    const int t = (int)div_by(u, per_token);
    if (t >= p.T) return;
    const int lanes = 1 << shift, D = p.pc.D, KV = p.pc.KV;
    const uint32_t rem = u - t * per_token.d;
    const int j = (int)(rem & (lanes - 1));
    int hg = (int)(rem >> shift);
    const bool is_q = hg < qgroups, is_v = hg >= qgroups + kgroups;
    if (!is_q) hg -= is_v ? qgroups + kgroups : qgroups;
    const int h0 = hg * HPT, nh = min(HPT, (is_q ? p.H : KV) - h0);
    const TI *x = is_q ? static_cast<const TI *>(p.q) + t * p.ldq
                       : is_v ? static_cast<const TI *>(p.v) + t * p.ldv : static_cast<const TI *>(p.k) + t * p.ldk;
    x += (int64_t)h0 * D;
    const int half = is_v ? 0 : p.half;
    const Part part = VEC ? part_of<8>(j, half, lanes, D, p.inter) : Part{};
    Sixteen<TI, VEC> in[HPT];
#pragma unroll
    for (int h = 0; h < HPT; h++)
        if (h < nh) in[h].get(x + h * D, part, j, lanes, half, p.inter);
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
    const int seq = i < 0 ? -1 : p.seqs[i];
    const int at = (unsigned)seq < (unsigned)p.pc.max_seqs ? p.pc.len[seq] - (last - t) : -1;
    const int turn_at = p.pos && at >= 0 ? p.pos[t] : at;
    if (at < 0 || (unsigned)turn_at >= (unsigned)p.positions) {
        record_status(p.status, at < 0 ? E2C_ERR_BAD_SEQ : E2C_ERR_BAD_POSITION);
        return;
    }
    const int blk = at / p.pc.page, slot = at - blk * p.pc.page;
    int page = 0;
    if (!is_q) {
        page = blk < p.pc.max_blocks ? p.pc.table[(int64_t)seq * p.pc.max_blocks + blk] : -1;
        if ((unsigned)page >= (unsigned)p.pc.n_pages) {
            record_status(p.status, E2C_ERR_BAD_SEQ);
            return;
        }
    }
    const float *cs = p.cs + (int64_t)turn_at * p.half, *sn = p.sn + (int64_t)turn_at * p.half;
    const uint32_t group = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
#pragma unroll
    for (int h = 0; h < HPT; h++) {
        if (h >= nh) break;
        float r[16];
        in[h].floats(r, part, j, lanes, half, p.inter, cs, sn);
        if (is_q) {
            TO *y = static_cast<TO *>(p.q_out) + t * p.ldo + (int64_t)(h0 + h) * D;
            if constexpr (VEC) {
                store<TO, 8>(y + part.e0, reinterpret_cast<const float(&)[8]>(r[0]));
                store<TO, 8>(y + part.e1, reinterpret_cast<const float(&)[8]>(r[8]));
            } else {
                // in place, a value is also read as the other of its pair: all lanes' loads are done
                __syncwarp(group);
#pragma unroll
                for (int k = 0; k < 16; k++) y[j + lanes * k] = from_f<TO>(r[k]);
            }
            continue;
        }
        // magnitudes as their bits: those of a NaN are above all others
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 16; k++) top = max(top, __float_as_uint(r[k]) & 0x7fffffffu);
        for (int d = 1; d < lanes; d <<= 1) top = max(top, __shfl_xor_sync(group, top, d));
        const float amax = __uint_as_float(top);
        const bool bad = top >= 0x7f800000u, some = !bad && amax >= kLeast;
        const float inv = some ? __fdiv_rn(127.0f, amax) : 0.f;
        if (!some) {
#pragma unroll
            for (int k = 0; k < 16; k++) r[k] = 0.f;
        }
        int8_t *y = static_cast<int8_t *>(is_v ? p.pc.v : p.pc.k) + (((int64_t)page * p.pc.page + slot) * KV + h0 + h) * D;
        if constexpr (VEC) {
            *reinterpret_cast<uint2 *>(y + part.e0) = make_uint2(four(r, inv), four(r + 4, inv));
            *reinterpret_cast<uint2 *>(y + part.e1) = make_uint2(four(r + 8, inv), four(r + 12, inv));
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++) y[j + lanes * k] = (int8_t)qround(r[k], inv);
        }
        if (j == 0)
            (is_v ? p.pc.vs : p.pc.ks)[((int64_t)page * KV + h0 + h) * p.pc.page + slot] = bad ? NAN : some ? __fmul_rn(amax, kInv127) : 1.0f;
    }
}

template <typename TI, typename TO>
int store_as(const e2c_store_args &a, bool vec, cudaStream_t st) {
    const int shift = a.pc.D == 64 ? 2 : a.pc.D == 128 ? 3 : 4;
    const int qg = (a.H + HPT - 1) / HPT, kg = (a.pc.KV + HPT - 1) / HPT;
    const int64_t per_token = (int64_t)(qg + 2 * kg) << shift, total = a.T * per_token, blocks = (total + BLOCK - 1) / BLOCK;
    if (total > 0x7fffffff - BLOCK) {
        e2c_set_msg("pages_store: %d tokens of %d heads are too many for one call", a.T, a.H);
        return -1;
    }
    const Div per = divide_by((int)per_token);
    if (vec)
        e2c_launch_as(true, k_store_codes<TI, TO, true>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, shift, qg, kg);
    else
        e2c_launch_as(true, k_store_codes<TI, TO, false>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, a, per, shift, qg, kg);
    return launched("pages_store");
}
template <typename TO>
int store_to(const e2c_store_args &a, int x_type, bool vec, cudaStream_t st) {
    return x_type == E2C_F32 ? store_as<float, TO>(a, vec, st)
           : x_type == E2C_BF16 ? store_as<__nv_bfloat16, TO>(a, vec, st) : store_as<__half, TO>(a, vec, st);
}

struct LoadArgs {
    e2c_pages pc;
    const int32_t *seqs, *first, *q_start;
    int n, T;
    void *k, *v;
    int *status;
};

// eight values of a token's head as floats
E2C_DEV void eight(const uint4 &w, __nv_bfloat16, float (&r)[8]) {
    const __nv_bfloat16 *e = reinterpret_cast<const __nv_bfloat16 *>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = __bfloat162float(e[i]);
}
E2C_DEV void eight(const uint4 &w, __half, float (&r)[8]) {
    const __half *e = reinterpret_cast<const __half *>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = __half2float(e[i]);
}
E2C_DEV void eight(const uint2 &w, int8_t, float (&r)[8]) {
    const int8_t *e = reinterpret_cast<const int8_t *>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = (float)e[i];
}

// One thread: eight values of k and of v at the same places of up to four heads of one token. TC: what a page holds.
template <typename TC, typename TO>
__global__ void __launch_bounds__(BLOCK) k_load_pages(const LoadArgs p, const Div per_token, const Div units) {
    using Vec = std::conditional_t<sizeof(TC) == 1, uint2, uint4>;
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t u = blockIdx.x * BLOCK + threadIdx.x;
    const int t = (int)div_by(u, per_token);
    if (t >= p.T) return;
    const uint32_t rem = u - t * per_token.d;
    const int hg = (int)div_by(rem, units), j = (int)(rem - hg * units.d);
    const int D = p.pc.D, KV = p.pc.KV, h0 = hg * HPT, nh = min(HPT, KV - h0);
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
    const int seq = i < 0 ? -1 : p.seqs[i];
    int at = -1;
    if ((unsigned)seq < (unsigned)p.pc.max_seqs) {
        const int len = p.pc.len[seq];
        // a row of no token: before the first, or past the last
        const int64_t tok = p.first ? (int64_t)p.first[i] + (t - p.q_start[i]) : (int64_t)len - (last - t);
        if (tok >= 0 && tok < len && tok < (int64_t)p.pc.max_blocks * p.pc.page) at = (int)tok;
    }
    const int blk = at / p.pc.page, slot = at - blk * p.pc.page;
    const int page = at < 0 ? -1 : p.pc.table[(int64_t)seq * p.pc.max_blocks + blk];
    if ((unsigned)page >= (unsigned)p.pc.n_pages) {
        record_status(p.status, E2C_ERR_BAD_SEQ);
        return;
    }
    const int64_t from = (((int64_t)page * p.pc.page + slot) * KV + h0) * D + 8 * j, to = ((int64_t)t * KV + h0) * D + 8 * j;
    Vec a[HPT], b[HPT];
    float ka[HPT], vb[HPT];
#pragma unroll
    for (int h = 0; h < HPT; h++)
        if (h < nh) {
            a[h] = *reinterpret_cast<const Vec *>(static_cast<const TC *>(p.pc.k) + from + h * D);
            b[h] = *reinterpret_cast<const Vec *>(static_cast<const TC *>(p.pc.v) + from + h * D);
            if (sizeof(TC) == 1) {
                const int64_t s = ((int64_t)page * KV + h0 + h) * p.pc.page + slot;
                ka[h] = p.pc.ks[s];
                vb[h] = p.pc.vs[s];
            }
        }
#pragma unroll
    for (int h = 0; h < HPT; h++)
        if (h < nh) {
            float r[8], w[8];
            eight(a[h], TC(), r);
            eight(b[h], TC(), w);
            if (sizeof(TC) == 1) {
#pragma unroll
                for (int k = 0; k < 8; k++) r[k] *= ka[h], w[k] *= vb[h];
            }
            store<TO, 8>(static_cast<TO *>(p.k) + to + h * D, r);
            store<TO, 8>(static_cast<TO *>(p.v) + to + h * D, w);
        }
}

template <typename TC>
int load_from(const LoadArgs &a, int y_type, cudaStream_t st) {
    const int units = a.pc.D / 8, hgroups = (a.pc.KV + HPT - 1) / HPT;
    const int64_t total = (int64_t)a.T * units * hgroups, blocks = (total + BLOCK - 1) / BLOCK;
    if (total > 0x7fffffff - BLOCK) {
        e2c_set_msg("pages_load: %d tokens of %d heads are too many for one call", a.T, a.pc.KV);
        return -1;
    }
    const Div per = divide_by(units * hgroups), by = divide_by(units);
    const dim3 grid((unsigned)blocks), block(BLOCK);
    if (y_type == E2C_F32)
        e2c_launch_as(true, k_load_pages<TC, float>, grid, block, 0, st, a, per, by);
    else if (y_type == E2C_BF16)
        e2c_launch_as(true, k_load_pages<TC, __nv_bfloat16>, grid, block, 0, st, a, per, by);
    else
        e2c_launch_as(true, k_load_pages<TC, __half>, grid, block, 0, st, a, per, by);
    return launched("pages_load");
}

}  // namespace

int e2c_store_codes(const e2c_store_args &a, int x_type, int q_type, cudaStream_t st) {
    const int xb = x_type == E2C_F32 ? 4 : 2;
    const bool vec = a.half % 8 == 0 && fits16(a.q, a.ldq, xb) && fits16(a.k, a.ldk, xb) && fits16(a.v, a.ldv, xb) &&
                     fits16(a.q_out, a.ldo, 2) && fits16(a.cs, 0, 4) && fits16(a.sn, 0, 4);
    return q_type == E2C_BF16 ? store_to<__nv_bfloat16>(a, x_type, vec, st) : store_to<__half>(a, x_type, vec, st);
}

extern "C" int e2c_pages_load(const e2c_pages *pc, const int32_t *seqs, const int32_t *first, const int32_t *q_start, int n, int T,
                              void *k_out, void *v_out, int y_type, int *status, void *stream) {
    const LoadArgs a = {*pc, seqs, first, q_start, n, T, k_out, v_out, status};
    cudaStream_t st = (cudaStream_t)stream;
    if (pc->type == E2C_I8) return load_from<int8_t>(a, y_type, st);
    return pc->type == E2C_BF16 ? load_from<__nv_bfloat16>(a, y_type, st) : load_from<__half>(a, y_type, st);
}
