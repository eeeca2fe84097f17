// attention_pages.cu — attention of query tokens over the cached keys of their sequences, on the
// sm_100a tensor cores (tcgen05.mma kind::f16).
//
// Work is cut into ITEMS: one key head, up to 128 query rows that share its keys, and a run of key
// tiles of 128. Rows are (token, query head of the group) pairs, token-major, so the G query heads that
// read one key head fill a tile together.
//   - A sequence item has the rows of one sequence's tokens and reads that sequence's pages.
//   - With a shared prefix, a prefix item packs the rows of the whole batch, whatever their sequence,
//     and reads the prefix's pages once for all of them; sequence items then begin past the prefix.
// All lengths are on the device: every block adds up the items' tiles itself and takes an equal share
// of the tiles, in order (its first and last item may be parts of one). An item that lies in one block
// and has no prefix is written to the output; other parts leave their normalised sums and log-sum-exps in
// the workspace, and a second kernel joins them in a fixed order. No atomics: results do not depend
// on timing.
//
// Per key tile j of an item, with the online softmax of attention.cu:
//   S = Q K_j^T     fp32 in tensor memory, N rounded up to 16 keys in an item's last tile
//   P = exp2(S scale log2 e - m)  16 bits over S's columns; m moves only when it grows by 2^8, then O is rescaled
//   O += P V_j      fp32 in tensor memory; V is read as it lies in the cache (its head dim contiguous)
// Two S buffers: the two softmax warpgroups take alternate tiles, handing the running maximum on as
// soon as a tile's maximum is known, so their exponentials overlap.
//
// K and V tiles share one ring of stages in the order the products need them; pages arrive one TMA box
// each (a page's rows land as consecutive rows of the tile). Rows of V past the sequence's last key
// are zeroed in shared memory up to the product's 16-key granularity: what a page holds there is
// arbitrary, and 0 x NaN would not vanish. Keys past it are masked in S by a select.
//
// Warps: 0 = items and TMA, 1 = MMA issue (and zeroing), 4..11 = softmax, 12..15 = epilogue.
#include <cuda.h>
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
#include "tmap.h"

namespace {

constexpr int TR = 128;  // rows of an item
constexpr int TK = 128;  // keys of a tile
constexpr int NTHREADS = 512;
constexpr int NI = 8;  // item descriptors in flight
constexpr float kRescaleLog2 = 8.0f;
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

template <int D>
struct Cfg {
    static constexpr int NQ = D == 256 ? 1 : 2;                 // Q buffers
    static constexpr int NO = D == 256 ? 1 : 2;                 // O buffers in tensor memory
    static constexpr int PANELS = D / 64;                       // 64 of the head's dimensions each
    // a stage: one panel of a K tile (128 keys x 64), or VROWS keys of a V tile (VROWS x D)
    static constexpr int STAGE = 16384;
    static constexpr int NST = D == 64 ? 10 : 9;
    static constexpr int VROWS = STAGE / (2 * D);
    static constexpr bool CROSS = NQ == 2;  // an item's first QK is issued before the last PV of the one before
    static constexpr int Q_BYTES = TR * D * 2;
    static constexpr int RING = NQ * Q_BYTES;
    static constexpr int XM = RING + NST * STAGE;               // running maxima handed on [2][128]
    static constexpr int ML = XM + 2 * TR * 4;                  // item's (m, l) [2 items][2 groups][128] x 2
    static constexpr int ITEMS = ML + 2 * 2 * TR * 8;
    static constexpr int SCAN = ITEMS + NI * 64;
    static constexpr int BARS = SCAN + 256;
};
enum { SCAN_INTS = 64 };

enum {
    B_QF,
    B_QE = B_QF + 2,
    B_SF = B_QE + 2,
    B_PF = B_SF + 2,
    B_PV = B_PF + 2,
    B_MX = B_PV + 2,  // [2][4 lane quadrants]
    B_OF = B_MX + 8,
    B_OE = B_OF + 2,
    B_MLF = B_OE + 2,
    B_MLE = B_MLF + 2,
    B_ITF = B_MLE + 2,
    B_ITE = B_ITF + NI,
    B_DRAIN = B_ITE + NI,
    B_STF,
    B_STE = B_STF + 10,
    B_NUM = B_STE + 10
};
template <int D>
constexpr int smem_bytes() {
    return Cfg<D>::BARS + B_NUM * 8 + 16;
}
static_assert(smem_bytes<64>() <= 232448 && smem_bytes<128>() <= 232448 && smem_bytes<256>() <= 232448, "shared memory");

struct Args {
    e2c_pages pc;
    const int32_t *seqs, *q_start;
    int n, T, max_q, H, G, tpt;  // tpt: tokens of an item
    int shared, causal, window;
    float c;                     // |scale| log2 e
    uint32_t neg;                // scale < 0: the products negate Q
    void *out;
    int64_t ldo;
    float *lse;
    // workspace
    int4 *split;       // [blocks][2]: the item a block's first part belongs to, if the block is to report it
    int64_t *before;   // [n + 1] tiles of the sequence items before entry i; [n]: of the prefix items
    float *po, *pl;    // parts: [2 * blocks][128][D], [2 * blocks][128]
    float *dpo, *dpl;  // undivided parts with a prefix: [2][T][H][D], [2][T][H] (0: prefix, 1: own)
    int *status;
};

enum { TO_OUT = 0, TO_SLOT = 1, TO_DENSE = 2 };
struct __align__(16) Item {
    int t0, ntok;     // first token row and tokens; ntok < 0: no more items
    int kvh, nt;      // key head, key tiles of this part
    int k0, klim;     // first key of the first tile; keys from klim on are not there
    int base, len;    // sequence items: keys before base belong to the prefix; the sequence's length
    int pos0;         // position of token t0
    int masked;       // prefix items: rows differ in what they see
    int prefix, dst;  // dst: TO_*
    int slot;
    int pad[3];
};
static_assert(sizeof(Item) == 64, "descriptor");

// What one block of a grid of `blocks` does: tiles [begin(c), begin(c + 1)) of W. The number of blocks
// at work is at most W, so every one of them has a tile.
E2C_DEV int64_t begin_of(int64_t c, int64_t W, int64_t blocks) { return c * W / blocks; }
E2C_DEV int block_of(int64_t x, int64_t W, int64_t blocks) { return (int)(((x + 1) * blocks - 1) / W); }

struct Entry {
    int seq, len, q0, nq;
};
E2C_DEV Entry entry_of(const Args &p, int i, bool report) {
    Entry e;
    e.seq = p.seqs[i];
    e.q0 = p.q_start[i];
    e.nq = p.q_start[i + 1] - e.q0;
    bool bad = (unsigned)e.seq >= (unsigned)p.pc.max_seqs;
    e.len = 0;
    if (!bad) {
        e.len = p.pc.len[e.seq];
        const int most = p.pc.max_blocks * p.pc.page;
        if (e.len < 0 || e.len > most) {
            bad = true;
            e.len = e.len < 0 ? 0 : most;
        }
    }
    if (e.q0 < 0 || e.nq < 0 || e.nq > p.max_q || e.q0 > p.T - e.nq) {  // rows outside the call's: left out
        e.nq = 0;
        e.q0 = 0;
        bad = true;
    }
    if (bad && report) record_status(p.status, E2C_ERR_BAD_SEQ);
    return e;
}

// the keys that row tile r of an entry sees, past `base`: tiles of 128 from k0 on, up to klim. A tile of
// rows that sees nothing still has one tile (its rows are masked), so that its output is written.
E2C_DEV int span_of(const Args &p, int len, int nq, int r, int base, int &k0, int &klim) {
    const int a = r * p.tpt, b = min(nq, a + p.tpt);
    const int pa = len - nq + a, pb = len - nq + b - 1;
    int lo = base, hi = p.causal ? min(len, pb + 1) : len;
    if (p.window >= 0) {
        lo = max(lo, pa - p.window);
        hi = min(hi, pb + p.window + 1);
    }
    if (hi <= lo) {
        k0 = 0;
        klim = 1;
        return 1;
    }
    k0 = base + (lo - base) / TK * TK;
    klim = hi;
    return (hi - k0 + TK - 1) / TK;
}
// tiles of all of an entry's row tiles, for one key head
E2C_DEV int64_t tiles_of(const Args &p, const Entry &e, int base) {
    if (e.nq <= 0) return 0;
    const int nr = (e.nq + p.tpt - 1) / p.tpt;
    int k0, klim;
    if (!p.causal && p.window < 0) return (int64_t)nr * span_of(p, e.len, e.nq, 0, base, k0, klim);
    int64_t s = 0;
    for (int r = 0; r < nr; r++) s += span_of(p, e.len, e.nq, r, base, k0, klim);
    return s;
}

// the batch's totals, the same in every block
struct Plan {
    int64_t W, Wp;   // tiles in all; of prefix items
    int ptiles, plo; // tiles of a prefix item, its first key
    int pseq, pmax;  // the sequence whose table maps the prefix, and its tokens there
    int masked;      // some row does not see every key of the prefix
    int npt;         // row tiles of the batch
    int first;       // the entry of this block's first sequence item,
    int64_t first_before;  // and the tiles before it
};

// every thread of the block; sums, mins and maxima over the entries
E2C_DEV void make_plan(const Args &p, Plan &pl, int64_t *s64) {
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    int *s32 = reinterpret_cast<int *>(s64 + 18);
    int64_t mine = 0, total = 0;
    int best = -1, best_seq = 0, least = 0x7fffffff, flag = 0;
    Entry e = {};
    for (int base = 0; base < p.n; base += NTHREADS) {
        const int i = base + tid;
        if (i < p.n) {
            e = entry_of(p, i, blockIdx.x == 0);
            const int64_t t = tiles_of(p, e, p.shared) * p.pc.KV;
            mine = base == 0 ? t : mine;
            total += t;
            if (e.nq > 0) {
                if (e.len > best) {
                    best = e.len;
                    best_seq = e.seq;
                }
                least = min(least, e.len - e.nq);
                flag |= e.len < p.shared || (p.causal && e.len - e.nq < p.shared - 1);
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, d);
        least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
        flag |= __shfl_xor_sync(0xffffffffu, flag, d);
        const int b = __shfl_xor_sync(0xffffffffu, best, d), bs = __shfl_xor_sync(0xffffffffu, best_seq, d);
        if (b > best || (b == best && bs < best_seq)) {
            best = b;
            best_seq = bs;
        }
    }
    // 16 warps: totals in s64[0..15]; the rest in 4 rows of s32
    if (lane == 0) {
        s64[w] = total;
        s32[w] = best;
    }
    __syncthreads();
    int64_t Ws = 0;
    for (int i = 0; i < 16; i++) {
        Ws += s64[i];
        best = max(best, s32[i]);
    }
    __syncthreads();
    // the longest sequence's id, the least first position and the flag, one round each (the scratch is small)
    if (lane == 0) {
        s32[w] = least;
    }
    __syncthreads();
    for (int i = 0; i < 16; i++) least = min(least, s32[i]);
    __syncthreads();
    if (lane == 0) s32[w] = flag;
    __syncthreads();
    for (int i = 0; i < 16; i++) flag |= s32[i];
    pl.pmax = min(p.shared, max(best, 0));
    pl.masked = flag || p.window >= 0;
    pl.npt = (p.T + p.tpt - 1) / p.tpt;
    pl.plo = 0;
    pl.ptiles = 0;
    pl.pseq = -1;
    if (p.shared > 0 && best > 0) {
        if (p.window >= 0) pl.plo = max(0, least - p.window) / TK * TK;
        pl.ptiles = pl.plo < pl.pmax ? (pl.pmax - pl.plo + TK - 1) / TK : 0;
    }
    pl.Wp = (int64_t)pl.ptiles * pl.npt * p.pc.KV;
    pl.W = pl.Wp + Ws;
    // second pass: the longest sequence, the entry that this block's share begins in, and the tiles before
    // each entry for the joining kernel
    const int64_t blocks = min((int64_t)gridDim.x, pl.W);
    const int64_t at = (int64_t)blockIdx.x < blocks ? max((int64_t)0, begin_of(blockIdx.x, pl.W, blocks) - pl.Wp) : -1;
    int64_t run = 0;
    __syncthreads();
    if (tid == 0) {
        s32[0] = -1;
        s32[1] = 0x7fffffff;
    }
    for (int base = 0; base < p.n; base += NTHREADS) {
        const int i = base + tid;
        int64_t t = 0;
        if (i < p.n) {
            if (p.n > NTHREADS) {
                e = entry_of(p, i, false);
                mine = tiles_of(p, e, p.shared) * p.pc.KV;
            }
            t = mine;
        }
        int64_t x = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 31) s64[w] = x;
        __syncthreads();
        int64_t pre = run, all = 0;
        for (int k = 0; k < 16; k++) {
            if (k < w) pre += s64[k];
            all += s64[k];
        }
        pre += x - t;
        run += all;
        if (i < p.n) {
            if (t > 0 && at >= pre && at < pre + t) {
                s32[0] = i;
                s64[16] = pre;
            }
            if (e.nq > 0 && e.len == best) atomicMin(&s32[1], e.seq);
            if (blockIdx.x == 0 && p.shared > 0) p.before[i] = pre;
        }
    }
    __syncthreads();
    pl.first = s32[0];
    pl.first_before = s64[16];
    if (pl.ptiles) pl.pseq = s32[1];
    if (blockIdx.x == 0 && tid == 0) {
        p.before[p.n] = pl.Wp;
        p.before[p.n + 1] = pl.W;
        p.before[p.n + 2] = pl.ptiles;
    }
    __syncthreads();
}

E2C_DEV float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
E2C_DEV uint32_t pack2(float a, float b);
template <>
E2C_DEV uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
E2C_DEV uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__host__ __device__ constexpr uint32_t type_bits() {  // A and B formats of the instruction descriptor
    return sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? (1u << 7) | (1u << 10) : 0u;
}

// one producer step: a tile's place in its item and where its pages lie
struct Tile {
    int item;       // running item number; -1: no more tiles
    int kvh, kk, nk, row;
    int t0, prefix;
    bool first;
};

template <typename T, int D>
__global__ void __launch_bounds__(NTHREADS, 1)
    k_attention_pages(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQp,
                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args p,
                      const int q_box, const int qp_box) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    if (smem_u32(smem) & 1023) {
        griddep_wait();
        if (threadIdx.x == 0) record_status(p.status, E2C_ERR_SMEM_ALIGN);
        return;
    }
    const uint32_t sbase = smem_u32(smem);
    auto bar = [&](int i) { return sbase + C::BARS + 8u * i; };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + C::BARS + B_NUM * 8);
    Item *items = reinterpret_cast<Item *>(smem + C::ITEMS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(B_QF + i), 1);
            mbar_init(bar(B_QE + i), 1);
            mbar_init(bar(B_SF + i), 1);
            mbar_init(bar(B_PF + i), 4);
            mbar_init(bar(B_PV + i), 1);
            mbar_init(bar(B_OF + i), 1);
            mbar_init(bar(B_OE + i), 4);
            mbar_init(bar(B_MLF + i), 8);
            mbar_init(bar(B_MLE + i), 4);
        }
        for (int i = 0; i < 8; i++) mbar_init(bar(B_MX + i), 1);
        for (int i = 0; i < NI; i++) {
            mbar_init(bar(B_ITF + i), 1);
            mbar_init(bar(B_ITE + i), 13);  // MMA, 8 softmax and 4 epilogue warps
        }
        for (int i = 0; i < C::NST; i++) {
            mbar_init(bar(B_STF + i), 1);
            mbar_init(bar(B_STE + i), 1);
        }
        mbar_init(bar(B_DRAIN), 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(sbase + C::BARS + B_NUM * 8, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = *tmem_slot;  // S buffer i: columns 128 i .. +127; O buffer i: 256 + D i ..

    Plan pl;
    make_plan(p, pl, reinterpret_cast<int64_t *>(smem + C::SCAN));
    const int64_t blocks = min((int64_t)gridDim.x, pl.W);
    const int64_t L0 = (int64_t)blockIdx.x < blocks ? begin_of(blockIdx.x, pl.W, blocks) : 0;
    const int64_t L1 = (int64_t)blockIdx.x < blocks ? begin_of(blockIdx.x + 1, pl.W, blocks) : 0;

    // a consumer's copy of the next item; false after the last (or a failure). The slot is released at once.
    auto take = [&](int &n, Item &it) -> bool {
        const int s = n & (NI - 1);
        if (!__all_sync(0xffffffffu, mbar_wait(bar(B_ITF + s), (uint32_t)((n / NI) & 1), p.status, E2C_ERR_WAIT_ATTN))) return false;
        const int4 *d = reinterpret_cast<const int4 *>(items + s);
        int4 *o = reinterpret_cast<int4 *>(&it);
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = d[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_ITE + s));
        n++;
        return it.ntok >= 0;
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- items, Q, K and V loads
        bool ok = true;
        int ni = 0;                // items published
        int64_t pos = L0;
        // sequence entries, 32 at a time, one per lane
        int ebase = -1;
        Entry e = {};
        int64_t etiles = 0;
        int ei = pl.first, kvh = 0, r = 0;
        bool placed = false;  // kvh, r and left are valid for entry ei
        // the part being walked
        Item it = {};
        int seq = -1, j = 0;
        it.nt = 0;
        const int PB = min(p.pc.page, C::VROWS), NB = TK / PB;
        const int row_blk = lane < NB ? lane : 0;

        auto entry = [&](int i) {
            if (ebase < 0 || i >= ebase + 32) {
                ebase = i;
                const int k = i + lane;
                e = {};
                etiles = 0;
                if (k < p.n) {
                    e = entry_of(p, k, false);
                    etiles = tiles_of(p, e, p.shared);
                }
            }
        };
        auto publish = [&]() -> bool {
            const int s = ni & (NI - 1);
            if (!__all_sync(0xffffffffu,
                            mbar_wait(bar(B_ITE + s), (uint32_t)(((ni / NI) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER)))
                return false;
            if (lane == 0) {
                const int4 *d = reinterpret_cast<const int4 *>(&it);
                int4 *o = reinterpret_cast<int4 *>(items + s);
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = d[k];
                mbar_arrive(bar(B_ITF + s));
            }
            __syncwarp();
            ni++;
            return true;
        };
        // where a part goes: [s, s + nt) are the item's tiles, `undivided` where it goes whole
        auto destination = [&](int64_t s, int64_t end, int undivided) {
            if (s >= L0 && end <= L1) {
                it.dst = undivided;
                return;
            }
            it.dst = TO_SLOT;
            it.slot = 2 * blockIdx.x + (s > L0 ? 1 : 0);
            // an item's second block reports it to the joining kernel
            if (p.shared == 0 && s < L0 && block_of(s, pl.W, blocks) == (int)blockIdx.x - 1 && lane == 0) {
                const int c0 = blockIdx.x - 1, c1 = block_of(end - 1, pl.W, blocks);
                p.split[2 * blockIdx.x] = make_int4(it.t0, it.ntok, it.kvh, 2 * c0 + (s > begin_of(c0, pl.W, blocks) ? 1 : 0));
                p.split[2 * blockIdx.x + 1] = make_int4(c1, 0, 0, 0);
            }
        };
        if (p.shared == 0 && lane == 0 && pos < L1) p.split[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        __syncwarp();

        // the next tile, its pages asked for; publishes an item at its first tile
        auto advance = [&](Tile &t) -> bool {
            if (j == it.nt) {
                if (pos >= L1) {
                    t.item = -1;
                    return true;
                }
                if (pos < pl.Wp) {
                    const int64_t q = pos / pl.ptiles;
                    const int j0 = (int)(pos - q * pl.ptiles);
                    it.prefix = 1;
                    it.kvh = (int)(q / pl.npt);
                    it.t0 = (int)(q - (int64_t)it.kvh * pl.npt) * p.tpt;
                    it.ntok = min(p.tpt, p.T - it.t0);
                    it.nt = (int)(min((q + 1) * pl.ptiles, L1) - pos);
                    it.k0 = pl.plo + j0 * TK;
                    it.klim = pl.pmax;
                    it.masked = pl.masked;
                    it.slot = 0;
                    seq = pl.pseq;
                    destination(q * pl.ptiles, (q + 1) * pl.ptiles, TO_DENSE);
                } else {
                    int nq, len, q0;
                    int64_t skip = 0;  // tiles of the item before this block's share
                    if (!placed) {
                        entry(ei);
                        const int64_t c = __shfl_sync(0xffffffffu, etiles, ei - ebase);
                        int64_t off = pos - pl.Wp - pl.first_before;
                        kvh = (int)(off / c);
                        skip = off - kvh * c;
                        r = 0;
                    } else if (r * p.tpt >= __shfl_sync(0xffffffffu, e.nq, ei - ebase)) {
                        r = 0;
                        if (++kvh == p.pc.KV) {
                            kvh = 0;
                            do {
                                ei++;
                                if (ei >= p.n) break;  // cannot happen: pos < L1 <= W
                                entry(ei);
                            } while (__shfl_sync(0xffffffffu, e.nq, ei - ebase) == 0);
                            if (ei >= p.n) {
                                t.item = -1;
                                return true;
                            }
                        }
                    }
                    const int src = ei - ebase;
                    seq = __shfl_sync(0xffffffffu, e.seq, src);
                    len = __shfl_sync(0xffffffffu, e.len, src);
                    q0 = __shfl_sync(0xffffffffu, e.q0, src);
                    nq = __shfl_sync(0xffffffffu, e.nq, src);
                    int k0, klim, nt = span_of(p, len, nq, r, p.shared, k0, klim);
                    if (!placed) {
                        while (skip >= nt) {
                            skip -= nt;
                            nt = span_of(p, len, nq, ++r, p.shared, k0, klim);
                        }
                        placed = true;
                    }
                    if (len == 0) seq = -1;  // its table says nothing
                    const int64_t s = pos - skip;
                    it.prefix = 0;
                    it.kvh = kvh;
                    it.t0 = q0 + r * p.tpt;
                    it.ntok = min(p.tpt, nq - r * p.tpt);
                    it.nt = (int)(min(s + nt, L1) - pos);
                    it.k0 = k0 + (int)skip * TK;
                    it.klim = klim;
                    it.base = p.shared;
                    it.len = len;
                    it.pos0 = len - nq + r * p.tpt;
                    it.masked = 1;
                    it.slot = 0;
                    destination(s, s + nt, p.shared > 0 ? TO_DENSE : TO_OUT);
                    r++;
                }
                if (!publish()) return false;
                pos += it.nt;
                j = 0;
            }
            t.item = ni - 1;
            t.kvh = it.kvh;
            t.kk = it.k0 + j * TK;
            t.nk = min(TK, it.klim - t.kk);
            t.t0 = it.t0;
            t.prefix = it.prefix;
            t.first = j == 0;
            const int key = t.kk + row_blk * PB;
            int page = 0;
            if (seq >= 0 && key < it.klim) page = p.pc.table[(int64_t)seq * p.pc.max_blocks + key / p.pc.page];
            t.row = ((unsigned)page < (unsigned)p.pc.n_pages ? page : 0) * p.pc.page + (key & (p.pc.page - 1));
            j++;
            return true;
        };
        int st = 0;  // stages filled
        auto stage = [&](uint32_t bytes, uint32_t &dst, uint32_t &b) -> bool {
            const int s = st % C::NST;
            if (!__all_sync(0xffffffffu,
                            mbar_wait(bar(B_STE + s), (uint32_t)(((st / C::NST) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER)))
                return false;
            dst = sbase + C::RING + s * C::STAGE;
            b = bar(B_STF + s);
            if (lane == 0) mbar_arrive_expect_tx(b, bytes);
            __syncwarp();
            st++;
            return true;
        };
        int nq_loads = 0;
        auto push_k = [&](const Tile &t) -> bool {
            if (t.first) {
                const int qb = t.item % C::NQ;
                if (!__all_sync(0xffffffffu, mbar_wait(bar(B_QE + qb), (uint32_t)(((t.item / C::NQ) & 1) ^ 1), p.status,
                                                       E2C_ERR_WAIT_PRODUCER)))
                    return false;
                if (lane == 0) {
                    const int box = t.prefix ? qp_box : q_box;
                    mbar_arrive_expect_tx(bar(B_QF + qb), (uint32_t)(C::PANELS * box * p.G * 128));
                    for (int i = 0; i < C::PANELS; i++)
                        tma_load_3d(sbase + qb * C::Q_BYTES + i * (TR * 128), t.prefix ? &tmQp : &tmQ, 64 * i, t.kvh * p.G, t.t0,
                                    bar(B_QF + qb));
                }
                __syncwarp();
                nq_loads = t.item + 1;
            }
            const int nb = (t.nk + PB - 1) / PB;
            for (int h = 0; h < C::PANELS; h++) {
                uint32_t dst, b;
                if (!stage((uint32_t)(nb * PB * 128), dst, b)) return false;
                if (lane < nb) tma_load_2d(dst + lane * (PB * 128), &tmK, t.kvh * D + 64 * h, t.row, b);
                __syncwarp();
            }
            return true;
        };
        auto push_v = [&](const Tile &t) -> bool {
            const int nb = (t.nk + PB - 1) / PB;
            constexpr int per = C::VROWS;
            for (int h = 0; h * per < t.nk; h++) {
                const int b0 = h * per / PB, bn = min(nb, (h + 1) * per / PB);
                uint32_t dst, b;
                if (!stage((uint32_t)((bn - b0) * PB * 128 * C::PANELS), dst, b)) return false;
                if (lane >= b0 && lane < bn)
                    for (int i = 0; i < C::PANELS; i++)
                        tma_load_2d(dst + i * (per * 128) + (lane - b0) * (PB * 128), &tmV, t.kvh * D + 64 * i, t.row, b);
                __syncwarp();
            }
            return true;
        };

        Tile cur, nxt, nn;
        ok = advance(cur);
        if (ok && cur.item >= 0) {
            ok = advance(nxt) && push_k(cur);
            while (ok) {
                if (nxt.item >= 0)
                    ok = advance(nn);
                else
                    nn.item = -1;
                if (!ok) break;
                if (nxt.item >= 0 && (C::CROSS || !nxt.first)) ok = push_k(nxt);
                ok = ok && push_v(cur);
                if (ok && nxt.item >= 0 && !(C::CROSS || !nxt.first)) ok = push_k(nxt);
                if (nxt.item < 0) break;
                cur = nxt;
                nxt = nn;
            }
        }
        if (ok) {
            it.ntok = -1;
            publish();
        }
        // every load that was issued has landed before the block may end
        for (int i = nq_loads - C::NQ < 0 ? 0 : nq_loads - C::NQ; i < nq_loads; i++)
            mbar_wait(bar(B_QF + i % C::NQ), (uint32_t)((i / C::NQ) & 1), nullptr, E2C_ERR_WAIT_DRAIN);
        for (int i = st - C::NST < 0 ? 0 : st - C::NST; i < st; i++)
            mbar_wait(bar(B_STF + i % C::NST), (uint32_t)((i / C::NST) & 1), nullptr, E2C_ERR_WAIT_DRAIN);
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issue
        // QK of the next tile, then PV of this one (across items too, with two Q buffers)
        const uint32_t idesc = (1u << 4) | type_bits<T>() | ((uint32_t)(128 >> 4) << 24);
        bool ok = true;
        int n = 0, st = 0;
        Item it = {};
        int left = 0, item = -1, kk = 0;  // of the tile that `step` gave last
        struct Step {
            int item, nk, g;
            bool first, last;
        };
        int g = 0;
        auto step = [&](Step &s) -> bool {
            if (left == 0) {
                if (!take(n, it)) {
                    s.item = -1;
                    return it.ntok < 0;
                }
                left = it.nt;
                item++;
                kk = it.k0;
                s.first = true;
            } else {
                s.first = false;
            }
            s.item = item;
            s.nk = min(TK, it.klim - kk);
            s.g = g++;
            kk += TK;
            left--;
            s.last = left == 0;
            return true;
        };
        auto full = [&](int s) {
            return __all_sync(0xffffffffu, mbar_wait(bar(B_STF + s % C::NST), (uint32_t)((s / C::NST) & 1), p.status, E2C_ERR_WAIT_MMA));
        };
        auto qk = [&](const Step &s) -> bool {
            const int qb = s.item % C::NQ;
            if (s.first && !__all_sync(0xffffffffu, mbar_wait(bar(B_QF + qb), (uint32_t)((s.item / C::NQ) & 1), p.status,
                                                              E2C_ERR_WAIT_MMA)))
                return false;
            const uint32_t id = idesc | (p.neg << 13) | (uint32_t)(((s.nk + 15) >> 4) << 1) << 17;
            const uint32_t d = tmem + (uint32_t)((s.g & 1) * 128);
            for (int h = 0; h < C::PANELS; h++, st++) {
                if (!full(st)) return false;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t kb = sbase + C::RING + (st % C::NST) * C::STAGE;
                    const uint32_t qa = sbase + qb * C::Q_BYTES + h * (TR * 128);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_bf16(d, smem_desc_sw128(qa + k * 32), smem_desc_sw128(kb + k * 32), id, h != 0 || k != 0);
                    mma_commit(bar(B_STE + st % C::NST));
                }
                __syncwarp();
            }
            if (lane == 0) {
                mma_commit(bar(B_SF + (s.g & 1)));
                if (s.last) mma_commit(bar(B_QE + qb));
            }
            __syncwarp();
            return true;
        };
        auto pv = [&](const Step &s) -> bool {
            const int ob = s.item % C::NO;
            const uint32_t id = idesc | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // B: N contiguous
            const uint32_t d = tmem + 256u + (uint32_t)(ob * D), a = tmem + (uint32_t)((s.g & 1) * 128);
            const int nk16 = (s.nk + 15) & ~15;
            bool waited = false;
            for (int h = 0; h * C::VROWS < s.nk; h++, st++) {
                if (!full(st)) return false;
                const uint32_t vb = sbase + C::RING + (st % C::NST) * C::STAGE;
                const int r0 = h * C::VROWS, here = min(C::VROWS, nk16 - r0);
                if (s.nk < r0 + here) {
                    // rows nk .. nk16 - 1 of every panel, 16 bytes a lane
                    const int rows = r0 + here - s.nk;
                    uint8_t *v = smem + C::RING + (st % C::NST) * C::STAGE + (s.nk - r0) * 128;
                    for (int x = lane; x < C::PANELS * rows * 8; x += 32) {
                        const int panel = x / (rows * 8), y = x - panel * (rows * 8);
                        *reinterpret_cast<uint4 *>(v + panel * (C::VROWS * 128) + y * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (!waited) {
                    waited = true;
                    if (!__all_sync(0xffffffffu, mbar_wait(bar(B_PF + (s.g & 1)), (uint32_t)((s.g >> 1) & 1), p.status,
                                                           E2C_ERR_WAIT_MMA)))
                        return false;
                    if (s.first && !__all_sync(0xffffffffu, mbar_wait(bar(B_OE + ob), (uint32_t)(((s.item / C::NO) & 1) ^ 1),
                                                                      p.status, E2C_ERR_WAIT_MMA)))
                        return false;
                }
                tc_fence_after();
                if (lane == 0) {
                    for (int k = 0; k < here / 16; k++)
                        mma_bf16_ts(d, a + (uint32_t)((r0 / 16 + k) * 8), smem_desc_sw128_mn(vb + k * 2048, C::VROWS * 128), id,
                                    !s.first || h != 0 || k != 0);
                    mma_commit(bar(B_STE + st % C::NST));
                }
                __syncwarp();
            }
            if (lane == 0) {
                mma_commit(bar(B_PV + (s.g & 1)));
                if (s.last) mma_commit(bar(B_OF + ob));
            }
            __syncwarp();
            return true;
        };
        Step cur, nxt;
        ok = step(cur);
        if (ok && cur.item >= 0) {
            ok = qk(cur);
            while (ok) {
                ok = step(nxt);
                if (!ok) break;
                if (nxt.item >= 0 && (C::CROSS || !nxt.first)) ok = qk(nxt);
                ok = ok && pv(cur);
                if (ok && nxt.item >= 0 && !(C::CROSS || !nxt.first)) ok = qk(nxt);
                if (nxt.item < 0) break;
                cur = nxt;
            }
        }
        // all products are done before the block frees tensor memory or ends
        if (lane == 0) mma_commit(bar(B_DRAIN));
        __syncwarp();
        mbar_wait(bar(B_DRAIN), 0, nullptr, E2C_ERR_WAIT_DRAIN);
    } else if (warp >= 4 && warp < 12) {
        // ---------------------------------------------------------------- softmax
        const int quad = warp & 3, group = (warp - 4) >> 2, row = quad * 32 + lane;
        const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16);
        float *xm = reinterpret_cast<float *>(smem + C::XM);
        float2 *ml = reinterpret_cast<float2 *>(smem + C::ML);
        const int tok = row / p.G;
        bool ok = true;
        int n = 0, g = 0;
        Item it;
        for (int item = 0; take(n, it); item++) {
            const bool live = tok < it.ntok;
            const bool busy = quad * 32 < it.ntok * p.G;  // some row of this warp is live
            int lo = 0, hi = it.klim;
            if (live && it.masked) {
                int pos, len;
                if (it.prefix) {
                    int last;
                    const int t = it.t0 + tok, i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
                    const int seq = i < 0 ? -1 : p.seqs[i];
                    len = (unsigned)seq < (unsigned)p.pc.max_seqs ? min(max(p.pc.len[seq], 0), p.pc.max_blocks * p.pc.page) : 0;
                    pos = len - (last - t);
                } else {
                    len = it.len;
                    pos = it.pos0 + tok;
                    lo = it.base;
                }
                hi = min(hi, len);
                if (p.causal) hi = min(hi, pos + 1);
                if (p.window >= 0) {
                    lo = max(lo, pos - p.window);
                    hi = min(hi, pos + p.window + 1);
                }
            }
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < it.nt; j++, g++) {
                if ((g & 1) != group) continue;
                const int b = g & 1, kk = it.k0 + j * TK, nk = min(TK, it.klim - kk);
                if (!__all_sync(0xffffffffu, mbar_wait(bar(B_SF + b), (uint32_t)((g >> 1) & 1), p.status, E2C_ERR_WAIT_ATTN))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t ts = ta + (uint32_t)(b * 128);
                const int chunks = (nk + 31) >> 5;
                const int ra = lo - kk, rb = max(hi - kk, ra);  // columns [ra, rb) are seen
                const bool mask = __any_sync(0xffffffffu, live && (ra > 0 || rb < TK));
                float mx = -INFINITY;
                if (busy) {
#pragma unroll 1
                    for (int c = 0; c < chunks; c++) {
                        uint32_t s[32];
                        tmem_ld32(ts + 32 * c, s);
                        tmem_wait_ld();
                        if (mask) {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if ((unsigned)(32 * c + i - ra) >= (unsigned)(rb - ra)) s[i] = 0xff800000u;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) mx = fmaxf(mx, __uint_as_float(s[i]));
                    }
                }
                mx *= p.c;
                // the running maximum, from the tile before
                float before = -INFINITY;
                if (g > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(bar(B_MX + (b ^ 1) * 4 + quad), (uint32_t)(((g - 1) >> 1) & 1), p.status,
                                                           E2C_ERR_WAIT_ATTN))) {
                        ok = false;
                        break;
                    }
                    if (j > 0) before = xm[(b ^ 1) * TR + row];
                }
                float now = before, alpha = 1.f;
                if (live && (mx > before + kRescaleLog2 || (before == -INFINITY && mx > -INFINITY))) {
                    now = mx;
                    alpha = before == -INFINITY ? 0.f : exp2f(before - mx);
                }
                xm[b * TR + row] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_MX + b * 4 + quad));
                if (busy) {
                    if (now != m) {
                        l = m == -INFINITY ? 0.f : l * exp2f(m - now);
                        m = now;
                    }
                    if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // O holds the tiles before this one once their products are done
                        if (!__all_sync(0xffffffffu, mbar_wait(bar(B_PV + (b ^ 1)), (uint32_t)(((g - 1) >> 1) & 1), p.status,
                                                               E2C_ERR_WAIT_ATTN))) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t to = ta + 256u + (uint32_t)((item % C::NO) * D);
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            tmem_ld32(to + 32 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st32(to + 32 * c, o);
                        }
                        tmem_wait_st();
                    }
                    const float cc = p.c, mneg = -m;
                    const bool any = m != -INFINITY;
                    float sum = 0.f;
#pragma unroll 1
                    for (int c = 0; c < chunks; c++) {
                        uint32_t s[32], pk[16];
                        tmem_ld32(ts + 32 * c, s);
                        tmem_wait_ld();
                        if (mask) {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if ((unsigned)(32 * c + i - ra) >= (unsigned)(rb - ra)) s[i] = 0xff800000u;
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float e0 = any ? ex2_approx(__fmaf_rn(__uint_as_float(s[2 * i]), cc, mneg)) : 0.f;
                            const float e1 = any ? ex2_approx(__fmaf_rn(__uint_as_float(s[2 * i + 1]), cc, mneg)) : 0.f;
                            sum += e0 + e1;
                            pk[i] = pack2<T>(e0, e1);
                        }
                        tmem_st16(ts + 16 * c, pk);
                    }
                    l += sum;
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PF + b));
            }
            if (!ok) break;
            // the slot's last reader was the epilogue two items ago
            if (!__all_sync(0xffffffffu, mbar_wait(bar(B_MLE + (item & 1)), (uint32_t)(((item >> 1) & 1) ^ 1), p.status,
                                                   E2C_ERR_WAIT_ATTN)))
                break;
            ml[((item & 1) * 2 + group) * TR + row] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_MLF + (item & 1)));
        }
    } else if (warp >= 12) {
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3, row = quad * 32 + lane;
        const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16);
        const float2 *ml = reinterpret_cast<const float2 *>(smem + C::ML);
        const int tok = row / p.G, hd = row - tok * p.G;
        int n = 0;
        Item it;
        for (int item = 0; take(n, it); item++) {
            const int ob = item % C::NO;
            if (!__all_sync(0xffffffffu, mbar_wait(bar(B_MLF + (item & 1)), (uint32_t)((item >> 1) & 1), p.status, E2C_ERR_WAIT_EPI)))
                break;
            const float2 a = ml[(item & 1) * 2 * TR + row], b = ml[((item & 1) * 2 + 1) * TR + row];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_MLE + (item & 1)));
            const float m = fmaxf(a.x, b.x);
            float l = 0.f;
            if (a.x > -INFINITY) l += a.y * exp2f(a.x - m);
            if (b.x > -INFINITY) l += b.y * exp2f(b.x - m);
            const bool some = l > 0.f;
            const float inv = some ? __fdiv_rn(1.0f, l) : 0.f;
            if (!__all_sync(0xffffffffu, mbar_wait(bar(B_OF + ob), (uint32_t)((item / C::NO) & 1), p.status, E2C_ERR_WAIT_EPI))) break;
            tc_fence_after();
            const bool live = tok < it.ntok;
            const int64_t t = it.t0 + tok;
            const int h = it.kvh * p.G + hd;
            if (quad * 32 < it.ntok * p.G) {
                const float sums = some ? m + log2f(l) : -INFINITY;
                T *out = nullptr;
                float *part = nullptr;
                if (it.dst == TO_OUT) {
                    out = static_cast<T *>(p.out) + t * p.ldo + (int64_t)h * D;
                    if (live && p.lse) p.lse[t * p.H + h] = sums * LN2;
                } else if (it.dst == TO_SLOT) {
                    part = p.po + ((int64_t)it.slot * TR + row) * D;
                    if (live) p.pl[(int64_t)it.slot * TR + row] = sums;
                } else {
                    const int64_t at = ((int64_t)(it.prefix ? 0 : 1) * p.T + t) * p.H + h;
                    part = p.dpo + at * D;
                    if (live) p.dpl[at] = sums;
                }
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[32];
                    tmem_ld32(ta + 256u + (uint32_t)(ob * D + 32 * c), o);
                    tmem_wait_ld();
                    // a row that saw nothing may have met a page's NaN: its zeros are not a product
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = some ? __float_as_uint(__uint_as_float(o[i]) * inv) : 0u;
                    if (live && out) {
                        uint4 *y = reinterpret_cast<uint4 *>(out + 32 * c);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint4 v;
                            v.x = pack2<T>(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1]));
                            v.y = pack2<T>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]));
                            v.z = pack2<T>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]));
                            v.w = pack2<T>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
                            y[i] = v;
                        }
                    } else if (live) {
                        uint4 *y = reinterpret_cast<uint4 *>(part + 32 * c);
#pragma unroll
                        for (int i = 0; i < 8; i++) y[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_OE + ob));
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of a row: out = sum_k w_k o_k / sum_k w_k with w_k = 2^(lse_k - max). D / 4 threads a row.
constexpr int JOIN = 256;
template <typename T, int D>
struct Join {
    static constexpr int LANES = D / 4, ROWS = JOIN / LANES;
    float4 acc = {0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;
    E2C_DEV void add(const float *o, float s, int x) {
        if (s == -INFINITY) return;
        const float4 v = *reinterpret_cast<const float4 *>(o + 4 * x);
        const float mn = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - mn);
        acc.x = acc.x * a + w * v.x;
        acc.y = acc.y * a + w * v.y;
        acc.z = acc.z * a + w * v.z;
        acc.w = acc.w * a + w * v.w;
        l = l * a + w;
        m = mn;
    }
    E2C_DEV void put(const Args &p, int64_t t, int h, int x) {
        const float inv = l > 0.f ? __fdiv_rn(1.0f, l) : 0.f;
        T *y = static_cast<T *>(p.out) + t * p.ldo + (int64_t)h * D + 4 * x;
        uint2 v;
        v.x = pack2<T>(acc.x * inv, acc.y * inv);
        v.y = pack2<T>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2 *>(y) = v;
        if (p.lse && x == 0) p.lse[t * p.H + h] = l > 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
    }
};

// without a prefix: the items that blocks share, one grid row per reporting block
template <typename T, int D>
__global__ void __launch_bounds__(JOIN) k_join_split(const Args p, int grid) {
    using J = Join<T, D>;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t W = p.before[p.n + 1];
    if ((int64_t)blockIdx.x >= min((int64_t)grid, W)) return;
    const int4 a = p.split[2 * blockIdx.x];
    if (a.y == 0) return;
    const int c1 = p.split[2 * blockIdx.x + 1].x;
    const int x = threadIdx.x % J::LANES, rows = a.y * p.G;
    for (int row = blockIdx.y * J::ROWS + threadIdx.x / J::LANES; row < rows; row += gridDim.y * J::ROWS) {
        J j;
        j.add(p.po + ((int64_t)a.w * TR + row) * D, p.pl[(int64_t)a.w * TR + row], x);
        for (int c = blockIdx.x; c <= c1; c++) j.add(p.po + ((int64_t)(2 * c) * TR + row) * D, p.pl[(int64_t)(2 * c) * TR + row], x);
        const int tok = row / p.G;
        j.put(p, a.x + tok, a.z * p.G + (row - tok * p.G), x);
    }
}

// with a prefix: every row's prefix parts and its own
template <typename T, int D>
__global__ void __launch_bounds__(JOIN) k_join_prefix(const Args p, int grid) {
    using J = Join<T, D>;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t u = (int64_t)blockIdx.x * J::ROWS + threadIdx.x / J::LANES;
    const int64_t t = u / p.H;
    if (t >= p.T) return;
    const int h = (int)(u - t * p.H), kvh = h / p.G, hd = h - kvh * p.G, x = threadIdx.x % J::LANES;
    const int64_t Wp = p.before[p.n], W = p.before[p.n + 1];
    const int ptiles = (int)p.before[p.n + 2];
    const int64_t blocks = min((int64_t)grid, W);
    J j;
    auto parts = [&](int64_t s, int64_t end, int which, int row) {
        const int c0 = block_of(s, W, blocks), c1 = block_of(end - 1, W, blocks);
        if (c0 == c1) {
            const int64_t at = ((int64_t)which * p.T + t) * p.H + h;
            j.add(p.dpo + at * D, p.dpl[at], x);
            return;
        }
        for (int c = c0; c <= c1; c++) {
            const int slot = 2 * c + (c == c0 && s > begin_of(c0, W, blocks) ? 1 : 0);
            j.add(p.po + ((int64_t)slot * TR + row) * D, p.pl[(int64_t)slot * TR + row], x);
        }
    };
    if (ptiles) {
        const int npt = (p.T + p.tpt - 1) / p.tpt, rt = (int)(t / p.tpt);
        const int64_t s = ((int64_t)kvh * npt + rt) * ptiles;
        parts(s, s + ptiles, 0, (int)(t - (int64_t)rt * p.tpt) * p.G + hd);
    }
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, (int)t, last);
    if (i < 0) return;
    const Entry e = entry_of(p, i, false);
    if (e.nq == 0) return;
    // an entry has one row tile here
    int k0, klim;
    const int nt = span_of(p, e.len, e.nq, 0, p.shared, k0, klim);
    const int64_t s = Wp + p.before[i] + (int64_t)kvh * nt;
    parts(s, s + nt, 1, (int)(t - e.q0) * p.G + hd);
    j.put(p, t, h, x);
}

// Sequences of few query tokens fill a small part of a 128-row tile each; packed, the batch reads the
// prefix once per 128 rows instead of once per sequence. From half a tile on they gain nothing.
bool use_prefix(int max_q, int G, int shared) { return shared > 0 && 2 * max_q * G <= TR; }

struct Layout {
    size_t split, before, po, pl, dpo, dpl, bytes;
};
Layout layout(int blocks, int n, int T, int H, int D, bool prefix) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    l.split = take(sizeof(int4) * 2 * blocks);
    l.before = take(sizeof(int64_t) * (prefix ? (size_t)n + 3 : (size_t)n + 3));
    l.pl = take(sizeof(float) * 2 * blocks * TR);
    l.po = take(sizeof(float) * 2 * blocks * TR * D);
    l.dpl = take(prefix ? sizeof(float) * 2 * (size_t)T * H : 0);
    l.dpo = take(prefix ? sizeof(float) * 2 * (size_t)T * H * D : 0);
    l.bytes = at;
    return l;
}

int launch_error(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 0;
    e2c_set_msg("%s launch: %s", what, cudaGetErrorString(e));
    return -2;
}

template <typename T, int D>
int run(const Args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    using C = Cfg<D>;
    static E2cPerDev attr;
    const int dev = e2c_device();
    if (!attr.get(dev)) {
        if (cudaFuncSetAttribute(k_attention_pages<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D>()) !=
            cudaSuccess) {
            cudaGetLastError();
            e2c_set_msg("pages_attention: cannot reserve %d bytes of shared memory", smem_bytes<D>());
            return -2;
        }
        attr.set(dev, 1);
    }
    const CUtensorMapDataType dt = __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int q_box = a.tpt < a.max_q ? a.tpt : a.max_q, qp_box = a.tpt < a.T ? a.tpt : a.T;
    const uint64_t rows = (uint64_t)a.pc.n_pages * a.pc.page, width = (uint64_t)a.pc.KV * D;
    const uint32_t box = a.pc.page < C::VROWS ? a.pc.page : C::VROWS;
    CUtensorMap tq, tqp, tk, tv;
    if (e2c_tmap_3d(&tq, q, dt, 2, D, a.H, a.T, D * 2, (uint64_t)ldq * 2, 64, a.G, q_box) ||
        e2c_tmap_3d(&tqp, q, dt, 2, D, a.H, a.T, D * 2, (uint64_t)ldq * 2, 64, a.G, qp_box) ||
        e2c_tmap_2d(&tk, a.pc.k, dt, 2, width, rows, width * 2, 64, box) ||
        e2c_tmap_2d(&tv, a.pc.v, dt, 2, width, rows, width * 2, 64, box))
        return -3;
    e2c_launch(k_attention_pages<T, D>, dim3(sms), dim3(NTHREADS), smem_bytes<D>(), st, tq, tqp, tk, tv, a, q_box, qp_box);
    if (launch_error("pages_attention")) return -2;
    using J = Join<T, D>;
    if (prefix)
        e2c_launch(k_join_prefix<T, D>, dim3((unsigned)(((int64_t)a.T * a.H + J::ROWS - 1) / J::ROWS)), dim3(JOIN), 0, st, a, sms);
    else
        e2c_launch(k_join_split<T, D>, dim3(sms, 8), dim3(JOIN), 0, st, a, sms);
    return launch_error("pages_attention join");
}

}  // namespace

extern "C" size_t e2c_pages_attention_ws_bytes(int n, int T, int max_q, int H, int KV, int D, int shared) {
    const int sms = e2c_sm_count(e2c_device());
    return sms ? layout(sms, n, T, H, D, use_prefix(max_q, H / KV, shared)).bytes : 0;
}

extern "C" int e2c_pages_attention(const e2c_pages *pc, const void *q, int64_t ldq, const int32_t *seqs, const int32_t *q_start, int n,
                                   int T, int max_q, int H, int shared, int causal, int window, float scale, void *out, int64_t ldo,
                                   float *lse, void *ws, size_t ws_bytes, int *status, void *stream) {
    const int sms = e2c_sm_count(e2c_device());
    if (!sms) {
        e2c_set_msg("pages_attention: no CUDA device");
        return -2;
    }
    const int G = H / pc->KV;
    const bool prefix = use_prefix(max_q, G, shared);
    const Layout l = layout(sms, n, T, H, pc->D, prefix);
    if (ws_bytes < l.bytes) {
        e2c_set_msg("pages_attention: workspace");
        return -1;
    }
    Args a;
    a.pc = *pc;
    a.seqs = seqs;
    a.q_start = q_start;
    a.n = n;
    a.T = T;
    a.max_q = max_q;
    a.H = H;
    a.G = G;
    a.tpt = TR / G;
    a.shared = prefix ? shared : 0;
    a.causal = causal != 0;
    a.window = window < 0 || window >= 1 << 30 ? -1 : window;  // lengths are at most 2^30
    // a scale of zero keeps masked logits (-inf) apart from the others (0)
    a.c = scale == 0.f ? 1e-30f : fabsf(scale) * LOG2E;
    a.neg = scale < 0.f;
    a.out = out;
    a.ldo = ldo;
    a.lse = lse;
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.split = reinterpret_cast<int4 *>(w + l.split);
    a.before = reinterpret_cast<int64_t *>(w + l.before);
    a.po = reinterpret_cast<float *>(w + l.po);
    a.pl = reinterpret_cast<float *>(w + l.pl);
    a.dpo = reinterpret_cast<float *>(w + l.dpo);
    a.dpl = reinterpret_cast<float *>(w + l.dpl);
    a.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = pc->type == E2C_BF16;
    if (pc->D == 64) return bf ? run<__nv_bfloat16, 64>(a, q, ldq, prefix, sms, st) : run<__half, 64>(a, q, ldq, prefix, sms, st);
    if (pc->D == 128) return bf ? run<__nv_bfloat16, 128>(a, q, ldq, prefix, sms, st) : run<__half, 128>(a, q, ldq, prefix, sms, st);
    return bf ? run<__nv_bfloat16, 256>(a, q, ldq, prefix, sms, st) : run<__half, 256>(a, q, ldq, prefix, sms, st);
}
