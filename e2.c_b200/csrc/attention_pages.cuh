// attention_pages.cuh — attention of query tokens over the cached keys of their sequences, on the
// sm_100a tensor cores (tcgen05.mma kind::f16).
//
// Work is cut into ITEMS: one key head, up to 128 query rows that share its keys, and a run of key
// tiles of 128. Rows are (token, query head of the group) pairs, token-major, so the G query heads that
// read one key head fill a tile together.
//   - A sequence item has the rows of one sequence's tokens and reads that sequence's pages.
//   - With a shared prefix, a prefix item packs the rows of the whole batch, whatever their sequence,
//     and reads the prefix's pages once for all of them; sequence items then begin past the prefix.
// All lengths are on the device: every block adds up the items' tiles itself and takes its share (Share).
// A sequence item that lies in one block and has no prefix is written to the output; other parts leave
// their normalised sums and log-sum-exps in the workspace, and a second kernel joins them in a fixed
// order. No floating-point atomics: results do not depend on timing.
//
// Per key tile j of an item, with the online softmax of attention.cu:
//   S = Q K_j^T     fp32 in tensor memory, N rounded up to 16 keys in an item's last tile
//   P = exp2(S scale log2 e - m)  16 bits over S's columns; m moves only when it grows by 2^8, then O is rescaled
//   O += P V_j      fp32 in tensor memory; V is read as it lies in the cache (its head dim contiguous)
// P is rounded to the cache's type, the tensor cores' operand (against 64 bits the output is then off by 0.0018 to
// 0.0023 of its size in bf16, where 32-bit arithmetic rounded once at the end is off by 0.0017; an fp32 P would
// take a second product for its low bits); its sum, m and O are held in 32 bits. The
// softmax warpgroups take the tiles in turn, handing the running maximum on as soon as a tile's is known, so
// that their exponentials overlap.
//
// K and V have a ring of stages and a loading warp each; pages arrive one TMA box each (a page's rows land as
// consecutive rows of the tile). Rows of V past the sequence's last key are zeroed in shared memory up
// to the product's 16-key granularity: what a page holds there is arbitrary, and 0 x NaN would not
// vanish. Keys past it are masked in S by a select.
//
// What bounds it (one B200, CUDA events): long single-token batches the memory (64 sequences of 5470 to 8192
// tokens, 429425 in all, 32 heads of 128 over 8 key heads, 1.76 GB: 280 us, 96% of the copy rate); whole prompts
// the chain from S to P in the softmax warps and the products' issue, some 1800 (heads of 64), 1980 (of 128)
// and 3100 cycles (of 256) a tile of 128 rows by 128 keys where the products take 512, 1024 and 2048 (4 prompts of
// 4096, 3007, 3284 and 3561 tokens, every key: 16 heads of 128 over 4 388 us, 63% of the measured bf16 rate; 8 heads
// of 256 over 4 315 us, 78%; 16 heads of 64 over 4 338 us); short sequences an item's set-up and output, some
// 3500 cycles (512 sequences of 11 to 16 tokens, 8 key heads: 60 us). The rings' depth (2 to 5 stages) moves a tile's time by less than 2%; so does a thread
// for each of the two products, except that heads of 256 lose 10%.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "devstate.cuh"
#include "launch.h"
#include "pages.cuh"
#include "pdl.h"
#include "ptx.cuh"
#include "tmap.h"

// An attention call, as its kernels take it.
struct e2c_attn_args {
    e2c_pages pc;
    int q_type;  // of q and out
    const int32_t *seqs, *q_start;
    int n, T, max_q, H, G, tpt;  // tpt: tokens of an item
    int shared, causal, window;
    int sinks, words;            // SIGHT: first tokens that a window leaves visible (0 without a window);
    int align;                   // FEW: what a window's first key is rounded down to,
    int hs;                      // blocks side by side that take a share's items of one key head each (1: all of them),
    int whole;                   // an item a block, undivided
    const uint32_t *tree;        // rows' bits among their entry's drafted tokens [T][words], or null
    float c;                     // |scale| log2 e
    uint32_t neg;                // scale < 0: the products negate Q
    void *out;
    int64_t ldo;
    float *lse;
    // workspace
    int4 *split;       // [blocks][2]: the item a block's first part belongs to, if the block is to report it
    int *before;       // [n + 2] the cost of the sequence items before entry i; of all; tiles of the prefix
    float *po, *pl;    // parts: [slots][128][D], [slots][128]; two a block, then one a prefix item
    float *dpo, *dpl;  // with a prefix, the undivided sequence items: [T][H][D], [T][H]
    int *status;
};

// What a call has beside causal order and a window: sinks or a tree (SIGHT), pages of 8 bits (CODES), few rows an
// entry (FEW, attention_few.cuh)
enum { SIGHT = 1, CODES = 2, FEW = 4 };
// The kernels of one kind over 16-bit pages: launches them for heads of a.pc.D, and their join.
int e2c_attn_plain(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st);
int e2c_attn_sight(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st);
// The same over pages of 8 bits, with SIGHT.
int e2c_attn_codes(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st);
// The same over pages of 16 and of 8 bits, for entries of at most FEW_ROWS rows (tokens by the heads of a key head), without a prefix:
// two N tiles, beyond which O alone is 32 registers more a tile (heads of 128). us a call with 9 to 16 rows, here and by tiles of 128 rows: 8 bits,
// 64 sequences of 5461 to 8192 tokens, heads of 64 291 and 345, of 128 236 and 363, of 256 243 and 367, 4 of 700 15.9 and 17.6; 16 bits,
// 128 windows of 2047 and sinks, heads of 64 131 and 141, of 128 194 and 190, of 256 192 and 188, 40 windows of 300 30.6 and 29.0, 3 of 511 15.0 and
// 16.4, 4 trees behind 300 tokens 12.9 and 15.5.
constexpr int FEW_ROWS = 16;
int e2c_attn_few(const e2c_attn_args &a, const void *q, int64_t ldq, int sms, cudaStream_t st);
int e2c_attn_few_codes(const e2c_attn_args &a, const void *q, int64_t ldq, int sms, cudaStream_t st);

namespace {

using Args = e2c_attn_args;

constexpr int TR = 128;  // rows of an item
constexpr int TK = 128;  // keys of a tile
constexpr int NI = 8;  // item descriptors in flight
// What a sequence item costs beside its tiles, in tiles: its set-up and its output
constexpr int ITEM_COST = 1;
constexpr int PREFIX_TILES = 13;  // use_prefix
constexpr float kRescaleLog2 = 8.0f;

// A wait of a whole warp, bounded by its number of tries, each of which sleeps for kTryNs at most: it gives up
// after 1.3 s at the latest, sooner where tries return early. It is small on
// purpose: with ptx.cuh's mbar_wait inlined at every wait the kernel was 234 KB of code, whose
// instruction fetches took most of a tile's time (heads of 128, the 4 prompts above: 905 us a call).
constexpr uint32_t kTryNs = 10000, kTries = 1u << 17;
E2C_DEV bool wait_warp(uint32_t bar, uint32_t parity, int *status, int code) {
    bool ok = false;
#pragma unroll 1
    for (uint32_t i = 0; i < kTries && !ok; i++) ok = mbar_try_wait_sleep(bar, parity, kTryNs);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) record_status(status, code);
    return ok;
}

constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

template <int D, int KIND>
struct Cfg {
    static constexpr bool CODE = KIND & CODES;
    // warps: NG softmax groups of four, the epilogue's four, then one each. A third softmax group hides more
    // of a tile's latencies where its products are shortest (heads of 64, us with two and with three: the 4 prompts
    // above 366 and 338, single tokens behind 700 of their own 55.4 and 52.1, behind 16 42.3 and 43.5); with wider
    // heads it gives less and costs batches of short items (128: 385 and 374, 92.9 and 94.1 for 128
    // tokens behind a shared prefix; 256: 312 and 314)
    static constexpr int NG = D == 64 && !CODE ? 3 : 2;
    static constexpr int W_EPI = 4 * NG, W_ITEMS = W_EPI + 4, W_MMA = W_ITEMS + 1, W_K = W_MMA + 1, W_V = W_K + 1;
    static constexpr int W_CONVERT = W_V + 1;  // CODES: four warps for K, then four for V
    static constexpr int WARPS = W_CONVERT + (CODE ? 8 : 0), NTHREADS = 32 * WARPS;
    // CODES: registers of a thread by role, and of the block
    static constexpr int R_SOFTMAX = 104, R_OTHERS = 72, R_CONVERT = 64;
    static constexpr int REGISTERS = 32 * (W_EPI * R_SOFTMAX + (W_CONVERT - W_EPI) * R_OTHERS + (WARPS - W_CONVERT) * R_CONVERT);
    static constexpr int PANELS = D / 64;  // 64 of the head's dimensions each, 128 bytes a row
    static constexpr int NQ = D == 64 ? 2 : 1;  // Q buffers
    // K and V have a ring of stages each: of a tile, or for D = 256 of half a one (K: half of the
    // head's dimensions, V: half of the keys)
    static constexpr int KPARTS = D == 256 ? 2 : 1, VROWS = TK / KPARTS;
    static constexpr int STAGE = TK * D * 2 / KPARTS;
    static constexpr int NKS = CODE ? (D == 64 ? 3 : D == 128 ? 2 : 1) : D == 64 ? 5 : D == 128 ? 3 : 2;
    static constexpr int NVS = CODE ? (D == 64 ? 3 : 1) : D == 64 ? 5 : 2;
    // CODES: stages as the pages hold them, rows of ROW bytes in panels; K's with the scales of both behind its codes
    static constexpr int ROW = D == 64 ? 64 : 128, CSTAGE = STAGE / 2, KCSTAGE = CSTAGE + 1024;  // (swizzled: multiples of 1024)
    static constexpr int NKC = !CODE ? 0 : D == 64 ? 4 : 3, NVC = !CODE ? 0 : D == 64 ? 4 : 2;
    static constexpr int NC = 4;  // tiles whose scales are in shared memory
    // tensor memory: NS buffers of S (128 columns each), then NO of O (D columns each), 512 columns
    static constexpr int NS = D == 256 ? 2 : 3;
    static constexpr int NO = D == 64 ? 2 : 1;
    static constexpr int O_COL = NS * 128;
    // QK runs NS - 1 tiles ahead of PV, across items too; with half tiles in the rings an item's first QK
    // follows the last PV of the item before
    static constexpr bool CROSS = KPARTS == 1;
    static constexpr int Q_BYTES = TR * D * 2;
    static constexpr int K_OFF = NQ * Q_BYTES;
    static constexpr int V_OFF = K_OFF + NKS * STAGE;
    static constexpr int KC_OFF = V_OFF + NVS * STAGE, VC_OFF = KC_OFF + NKC * KCSTAGE;
    static constexpr int SC_OFF = VC_OFF + NVC * CSTAGE;        // [NC]: K's times c; V's, their log2 and they themselves
    static constexpr int SC = 3 * TK;
    static constexpr int XM = SC_OFF + (CODE ? NC * SC * 4 : 0);  // running maxima handed on [NG][128]
    static constexpr int ML = XM + NG * TR * 4;                 // item's (m, l) [2 items][NG][128] x 2
    static constexpr int ITEMS = ML + 2 * NG * TR * 8;
    static constexpr int SCAN = ITEMS + NI * 64;
    static constexpr int BARS = SCAN + 256;
};

enum {
    B_QF,
    B_QE = B_QF + 2,
    B_SF = B_QE + 2,
    B_PF = B_SF + 3,
    B_PV = B_PF + 3,
    B_MX = B_PV + 2,  // [NG][4 lane quadrants]
    B_OF = B_MX + 12,
    B_OE = B_OF + 2,
    B_MLF = B_OE + 2,
    B_MLE = B_MLF + 2,
    B_ITF = B_MLE + 2,
    B_ITE = B_ITF + NI,
    B_DRAIN = B_ITE + NI,
    B_KF,
    B_KE = B_KF + 5,
    B_VF = B_KE + 5,
    B_VE = B_VF + 5,
    B_KCF = B_VE + 5,  // CODES: codes of K and V, and scales
    B_KCE = B_KCF + 4,
    B_VCF = B_KCE + 4,
    B_VCE = B_VCF + 4,
    B_SCF = B_VCE + 4,
    B_SCE = B_SCF + 4,
    B_NUM = B_SCE + 4
};
template <int D, int KIND>
constexpr int smem_bytes() {
    return Cfg<D, KIND>::BARS + B_NUM * 8 + 16;
}
template <int KIND>
constexpr bool fits = smem_bytes<64, KIND>() <= 232448 && smem_bytes<128, KIND>() <= 232448 && smem_bytes<256, KIND>() <= 232448;
static_assert(fits<0> && fits<SIGHT | CODES>, "shared memory");

enum { TO_OUT = 0, TO_SLOT = 1, TO_DENSE = 2 };
struct __align__(16) Item {
    int t0, ntok;     // first token row and tokens; ntok < 0: no more items
    int kvh, nt;      // key head, key tiles of this part
    int k0, klim;     // first key of the first tile; keys from klim on are not there
    int base, len;    // sequence items: keys before base belong to the prefix; the sequence's length
                      // (SIGHT: base is the first of the entry's rows' own keys instead)
    int pos0;         // position of token t0
    int masked;       // prefix items: rows differ in what they see
    int prefix, dst;  // dst: TO_*
    int slot, seq;    // seq: whose table maps the keys; -1: none (a page that is masked is read)
    int ns, gap;      // SIGHT: the first ns tiles hold sinks; after them gap keys are skipped
};
static_assert(sizeof(Item) == 64, "descriptor");

// What each of `grid` blocks does.
//
// Prefix items: a key head's prefix is cut into as many runs of `chunk` tiles as there are blocks for its row
// tiles, and the row tiles of one run go to neighbouring blocks, which read its keys at the same time: then one
// of them fetches a tile from memory and the others find it near in the L2 cache. (Shares that divide
// items anywhere had each row tile read the prefix at a time of its own, and took twice as long.) Item
// i goes to block i mod grid, whole.
//
// Sequence items: their tiles, in order, are divided so that all blocks have about the same to do; block
// c does tiles [begin(c), begin(c + 1)), and items are divided where a share ends.
struct Share {
    int items, splits, chunk;  // prefix items, runs of a key head's prefix, tiles of a run
    int n1, s1, each1, rest1;  // the first n1 blocks have a prefix item more; s1 tiles are theirs
    int each2, rest2;          // the other blocks' shares: each2, the first rest2 of them one more
    E2C_DEV void set(int rows, int ptiles, int tiles, int grid) {
        items = splits = chunk = n1 = s1 = each1 = rest1 = 0;
        if (ptiles <= 0) {
            each2 = tiles / grid;
            rest2 = tiles - each2 * grid;
            return;
        }
        const int s = max(1, grid / rows);
        chunk = (ptiles + s - 1) / s;
        splits = (ptiles + chunk - 1) / chunk;
        items = rows * splits;
        const int cost = chunk + 2 * ITEM_COST, k = items / grid;
        n1 = items - k * grid;
        const int64_t target = ((int64_t)items * cost + tiles) / grid;
        const int64_t room = target - (int64_t)(k + 1) * cost;  // for a block with k + 1 prefix items
        s1 = room > 0 ? (int)min((int64_t)tiles, room * n1) : 0;
        each1 = n1 > 0 ? s1 / n1 : 0;
        rest1 = s1 - each1 * n1;
        const int n2 = grid - n1;
        each2 = (tiles - s1) / n2;
        rest2 = tiles - s1 - each2 * n2;
    }
    E2C_DEV int begin(int c) const {
        return c <= n1 ? c * each1 + min(c, rest1) : s1 + (c - n1) * each2 + min(c - n1, rest2);
    }
    static E2C_DEV int part(int x, int each, int rest) {
        const int c = (int)((unsigned)x / (unsigned)(each + 1));
        return c < rest ? c : rest + (int)((unsigned)(x - rest * (each + 1)) / (unsigned)each);
    }
    E2C_DEV int block(int x) const { return x < s1 ? part(x, each1, rest1) : n1 + part(x - s1, each2, rest2); }
};

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

// A window's first tile begins at a multiple of it (past the prefix): of what one load brings, at least
template <int KIND>
E2C_DEV int aligned(const Args &p, int x) {
    return KIND & FEW ? x & -p.align : x / TK * TK;
}
// the blocks side by side that have the same share of the entries' tiles, for a key head each
template <int KIND>
E2C_DEV int hs_of(const Args &p) {
    return KIND & FEW ? p.hs : 1;
}
template <int KIND>
constexpr int SLOT = KIND & FEW ? FEW_ROWS : TR;  // rows of a part in the workspace
// A run of key tiles: nt of them from k0 on, keys before klim; gap keys are skipped after the first ns.
struct Span {
    int nt, k0, klim, ns, gap;
    // the part of nt tiles from tile off on, in an item's fields
    E2C_DEV void cut(const Args &p, int off, int n, Item &it) const {
        const bool past = off >= ns;
        it.nt = n;
        it.k0 = k0 + off * TK + (past ? gap : 0);
        it.klim = past || off + n > ns ? klim : min(klim, p.sinks);
        it.ns = past || off + n <= ns ? 0 : ns - off;
        it.gap = it.ns > 0 ? gap : 0;
    }
};
// first key of tile j of an item, and the keys' end in it
template <int KIND>
E2C_DEV int tile_key(const Item &it, int j) {
    return it.k0 + j * TK + (KIND & SIGHT && j >= it.ns ? it.gap : 0);
}
template <int KIND>
E2C_DEV int tile_end(const Args &p, const Item &it, int j) {
    return KIND & SIGHT && j < it.ns ? p.sinks : it.klim;
}
// the sinks [base, se) and a window's keys [lo, hi) as one run of tiles from base on; those in neither are skipped
template <int KIND>
E2C_DEV Span with_sinks(const Args &p, int base, int se, int lo, int hi) {
    const int ns = se > base ? (se - base + TK - 1) / TK : 0;
    if (hi <= lo) {
        if (ns == 0) return {1, 0, 1, 0, 0};
        return {ns, base, se, 0, 0};
    }
    const int kw = base + aligned<KIND>(p, lo - base), end = base + ns * TK;
    if (ns > 0 && kw > end) return {ns + (hi - kw + TK - 1) / TK, base, hi, ns, kw - end};
    const int k0 = ns > 0 ? base : kw, klim = max(hi, se);
    return {(klim - k0 + TK - 1) / TK, k0, klim, 0, 0};
}

// the keys that row tile r of an entry sees, past `base`: tiles of 128 from k0 on, up to klim. A tile of
// rows that sees nothing still has one tile (its rows are masked), so that its output is written.
template <int KIND>
E2C_DEV Span span_of(const Args &p, int len, int nq, int r, int base) {
    const int a = r * p.tpt, b = min(nq, a + p.tpt);
    int pa = len - nq + a, pb = len - nq + b - 1;
    if (KIND & SIGHT) {
        int text = p.causal ? min(len, pb + 1) : len;
        int lo = base, hi = text;
        if (p.tree) {  // a drafted token's position is the text's end or past it, or one before for a row without bits
            text = min(len, len - nq);
            pa = len - nq - 1;
            hi = len;
        }
        if (p.window >= 0) {
            lo = max(lo, pa - p.window);
            if (!p.tree) hi = min(hi, pb + p.window + 1);
        }
        return with_sinks<KIND>(p, base, min(p.sinks, text), lo, hi);
    }
    int lo = base, hi = p.causal ? min(len, pb + 1) : len;
    if (p.window >= 0) {
        lo = max(lo, pa - p.window);
        hi = min(hi, pb + p.window + 1);
    }
    if (hi <= lo) return {1, 0, 1, 0, 0};
    const int k0 = base + (lo - base) / TK * TK;
    return {(hi - k0 + TK - 1) / TK, k0, hi, 0, 0};
}

// What row t of an entry sees, whose rows' own keys begin at `first`: the keys [lo, hi), the sinks [0, se), and of the
// drafted ones [first, len) those whose bit is set. A drafted token's position is that of the text's end and its
// ancestors.
struct Seen {
    int lo, hi, se, first, len;
    const uint32_t *bits;
    E2C_DEV uint32_t word(int i, int words) const { return (unsigned)i < (unsigned)words ? bits[i] : 0u; }
    E2C_DEV void set(const Args &p, int64_t t, int pos, int n, int own) {
        first = own;
        len = n;
        bits = p.tree ? p.tree + t * p.words : nullptr;
        int text = p.causal ? min(n, pos + 1) : n;
        if (bits) {
            text = min(n, own);
            if (p.window >= 0) {
                pos = own - 1;
#pragma unroll 1
                for (int i = 0; i < (n - own + 31) / 32; i++) pos += __popc(word(i, p.words) & below(n - own - 32 * i));
            }
        }
        lo = 0;
        hi = text;
        se = min(p.sinks, text);
        if (p.window >= 0) {
            lo = max(lo, pos - p.window);
            hi = min(hi, pos + p.window + 1);
        }
    }
    // 32 bits of which the first n are set
    static E2C_DEV uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
    static E2C_DEV uint32_t between(int a, int b) { return below(b) & ~below(a); }
    // keys [key, key + 32) that it sees, as bits
    E2C_DEV uint32_t keys(const Args &p, int key) const {
        uint32_t s = between(lo - key, hi - key) | below(se - key);
        if (bits && key + 32 > first && key < len) {
            const int at = key - first, i = at >> 5;
            s |= __funnelshift_r(word(i, p.words), word(i + 1, p.words), at & 31) & between(max(first, 0) - key, len - key);
        }
        return s;
    }
    E2C_DEV bool any(const Args &p) const {
        if (lo < hi || se > 0) return true;
        if (bits)
            for (int key = max(first, 0); key < len; key += 32)
                if (keys(p, key)) return true;
        return false;
    }
};
// whether row t, at position pos of a sequence of len tokens whose rows begin at `first`, sees any key
template <int KIND>
E2C_DEV bool sees_keys(const Args &p, int64_t t, int pos, int len, int first) {
    if (KIND & SIGHT) {
        Seen s;
        s.set(p, t, pos, len, first);
        return s.any(p);
    }
    int lo = 0, hi = p.causal ? min(len, pos + 1) : len;
    if (p.window >= 0) {
        lo = max(lo, pos - p.window);
        hi = min(hi, pos + p.window + 1);
    }
    return lo < hi;
}
// the cost of all of an entry's row tiles, for one key head
template <int KIND>
E2C_DEV int64_t tiles_of(const Args &p, int len, int nq, int base) {
    if (nq <= 0) return 0;
    const int nr = (nq + p.tpt - 1) / p.tpt;
    // every row tile sees every key, or a tree's rows are not told apart
    const bool same = (!p.causal && p.window < 0) || (KIND & SIGHT && p.tree);
    int64_t s = 0;
#pragma unroll 1
    for (int r = 0; r < nr; r++) {
        s += span_of<KIND>(p, len, nq, r, base).nt + ITEM_COST;
        if (same) return s * nr;
    }
    return s;
}

// the batch's totals, the same in every block
struct Plan {
    Share share;
    int ptiles;      // tiles of the prefix
    Span pspan;      // their keys
    int pseq;        // the sequence whose table maps the prefix
    int masked;      // some row does not see every key of the prefix
    int npt;         // row tiles of the batch
    int tiles;       // cost of the sequence items
    int first;       // the entry of this block's first sequence item,
    int first_before;  // and the tiles before it
};

// Every thread of the block: sums over the entries, the longest of them, and the entry in which this
// block's share begins (block 0 leaves the joining kernel the cost before each entry). Up to NTHREADS
// entries are read once, more of them twice.
template <int WARPS>
struct PlanScratch {
    int64_t sum[WARPS];  // by warp
    int at;              // cost before the block's first entry
    int longest, least, masked, first, seq;
};
template <int WARPS, int KIND>
E2C_DEV void make_plan(const Args &p, Plan &pl, PlanScratch<WARPS> &s) {
    constexpr int NTHREADS = 32 * WARPS;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    if (tid == 0) {
        s.longest = -1;
        s.least = 0x7fffffff;
        s.masked = 0;
        s.first = -1;
        s.seq = 0x7fffffff;
    }
    pl.npt = (p.T + p.tpt - 1) / p.tpt;
    const int rounds = p.n > NTHREADS ? 2 : 1;
    int at = -1;
#pragma unroll 1
    for (int round = 0; round < rounds; round++) {
        const bool last = round == rounds - 1;
        int64_t run = 0;
#pragma unroll 1
        for (int base = 0; base < p.n; base += NTHREADS) {
            const int i = base + tid;
            Entry e = {};
            int64_t mine = 0;
            if (i < p.n) {
                e = entry_of(p, i, round == 0 && blockIdx.x == 0);
                mine = tiles_of<KIND>(p, e.len, e.nq, p.shared) * (p.pc.KV / hs_of<KIND>(p));
            }
            int64_t x = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            __syncthreads();  // the scratch is set, the sums of the step before have been read
            if (lane == 31) s.sum[w] = x;
            if (p.shared > 0 && round == 0) {
                const int longest = __reduce_max_sync(0xffffffffu, e.nq > 0 ? e.len : -1);
                const int least = __reduce_min_sync(0xffffffffu, e.nq > 0 ? e.len - e.nq : 0x7fffffff);
                const bool masked = __any_sync(0xffffffffu, e.nq > 0 && (e.len < p.shared || (p.causal && e.len - e.nq < p.shared - 1) ||
                                                                                 (KIND & SIGHT && p.tree && e.len - e.nq < p.shared)));
                if (lane == 0) {
                    atomicMax(&s.longest, longest);
                    atomicMin(&s.least, least);
                    if (masked) s.masked = 1;
                }
            }
            __syncthreads();
            // every warp adds up the warps' sums
            int64_t y = lane < WARPS ? s.sum[lane] : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t z = __shfl_up_sync(0xffffffffu, y, d);
                if (lane >= d) y += z;
            }
            const int64_t all = __shfl_sync(0xffffffffu, y, 31), here = __shfl_sync(0xffffffffu, y, w > 0 ? w - 1 : 0);
            const int64_t before = run + (w > 0 ? here : 0) + x - mine;
            run += all;
            if (round == 0 && base + NTHREADS >= p.n) {
                const int pmax = min(p.shared, max(s.longest, 0));
                int lo = 0;
                pl.masked = s.masked || p.window >= 0;
                if (p.window >= 0) lo = max(0, s.least - (KIND & SIGHT && p.tree ? 1 : 0) - p.window);
                if (KIND & SIGHT) {
                    const int se = min(p.sinks, pmax);
                    pl.pspan = with_sinks<KIND>(p, 0, se, lo, pmax);
                    pl.ptiles = lo < pmax || se > 0 ? pl.pspan.nt : 0;
                } else {
                    const int k0 = lo / TK * TK;
                    pl.ptiles = k0 < pmax ? (pmax - k0 + TK - 1) / TK : 0;
                    pl.pspan = {pl.ptiles, k0, pmax, 0, 0};
                }
                const bool fits = run < 1ll << 30;
                if (!fits && tid == 0) record_status(p.status, E2C_ERR_TOO_LARGE);
                pl.tiles = fits ? (int)run : 0;
                if (!fits) pl.ptiles = 0;
                pl.share.set(p.pc.KV * pl.npt, pl.ptiles, pl.tiles, gridDim.x / hs_of<KIND>(p));
                at = pl.share.begin(blockIdx.x / hs_of<KIND>(p));
            }
            if (last && i < p.n) {
                if (at >= before && at < before + mine) {
                    s.first = i;
                    s.at = (int)before;
                }
                if (p.shared > 0) {
                    if (e.nq > 0 && e.len == s.longest) atomicMin(&s.seq, e.seq);
                    if (blockIdx.x == 0) p.before[i] = (int)before;
                }
            }
        }
    }
    __syncthreads();
    pl.first = s.first;
    pl.first_before = s.at;
    pl.pseq = s.seq;
    if (blockIdx.x == 0 && tid == 0) {
        p.before[p.n] = pl.tiles;
        p.before[p.n + 1] = pl.ptiles;
    }
}

// One warp: the parts of sequence items in a block's share, in order. Entries are read 32 at a time, one a lane.
template <int KIND>
struct Walk {
    int pos, end, off;      // the share left; tiles before pos of the entry
    int i, base, kvh, r;    // the entry, the first of those read; the next key head and row tile
    Entry e;                // the lane's entry and its tiles for one key head
    int etiles;
    bool inside;            // an entry has been begun: its tokens, rows and first row
    int len, nq, q0, seq;
    E2C_DEV void begin(const Plan &pl, int L0, int L1) {
        pos = L0;
        end = L1;
        off = L0 - pl.first_before;
        i = pl.first;
        base = -32;
        inside = false;
    }
    // the next part, in the fields of `it` that do not hold for all of them; false after the last
    E2C_DEV bool next(const Args &p, const Plan &pl, Item &it, int lane) {
        const int hs = hs_of<KIND>(p), share = blockIdx.x / hs, head = blockIdx.x - share * hs, heads = p.pc.KV / hs;
        for (;;) {
            if (!inside) {
                if (pos >= end || i >= p.n) return false;
                if (i >= base + 32) {
                    base = i;
                    e = {};
                    etiles = 0;
                    if (i + lane < p.n) {
                        e = entry_of(p, i + lane, false);
                        etiles = (int)tiles_of<KIND>(p, e.len, e.nq, p.shared);
                    }
                }
                const int src = i - base, c = __shfl_sync(0xffffffffu, etiles, src);
                nq = __shfl_sync(0xffffffffu, e.nq, src);
                if (nq == 0) {
                    i++;
                    continue;
                }
                len = __shfl_sync(0xffffffffu, e.len, src);
                q0 = __shfl_sync(0xffffffffu, e.q0, src);
                seq = __shfl_sync(0xffffffffu, e.seq, src);
                if (len == 0) seq = -1;  // its table says nothing
                kvh = r = 0;
                if (off >= c) {
                    kvh = off / c;
                    off -= kvh * c;
                }
                inside = true;
            }
#pragma unroll 1
            while (pos < end && kvh < heads) {
                const Span sp = span_of<KIND>(p, len, nq, r, p.shared);
                const int nt = sp.nt, cost = nt + ITEM_COST;
                bool found = false;
                if (off >= cost) {
                    off -= cost;
                } else if (off >= nt) {  // the share begins past the item's tiles
                    pos = min(pos + cost - off, end);
                    off = 0;
                } else {
                    const int s = pos - off, stop = s + nt, first = pl.share.begin(share);
                    it.seq = seq;
                    it.len = len;
                    if (KIND & SIGHT) it.base = len - nq;
                    it.kvh = kvh + head;
                    it.t0 = q0 + r * p.tpt;
                    it.ntok = min(p.tpt, nq - r * p.tpt);
                    sp.cut(p, off, min(stop, end) - pos, it);
                    it.pos0 = len - nq + r * p.tpt;
                    it.dst = p.shared > 0 ? TO_DENSE : TO_OUT;
                    if (off > 0 || stop > end) {  // a part of an item
                        it.dst = TO_SLOT;
                        it.slot = 2 * blockIdx.x + (s > first ? 1 : 0);
                        // an item's second block reports it to the joining kernel
                        const int c0 = pl.share.block(s);
                        if (p.shared == 0 && off > 0 && c0 == share - 1 && lane == 0) {
                            p.split[2 * blockIdx.x] = make_int4(it.t0, it.ntok, it.kvh, 2 * (c0 * hs + head) + (s > pl.share.begin(c0) ? 1 : 0));
                            p.split[2 * blockIdx.x + 1] = make_int4(pl.share.block(stop - 1), 0, 0, 0);
                        }
                    }
                    pos = min(s + cost, end);
                    off = 0;
                    found = true;
                }
                if (++r * p.tpt >= nq) {
                    r = 0;
                    kvh++;
                }
                if (found) return true;
            }
            inside = false;
            i++;
        }
    }
};

E2C_DEV float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
E2C_DEV float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maxima that a NaN stays in. A row whose largest logit is NaN or +infinity has no softmax: its running maximum
// keeps that value to the end, and the result is NaN whatever the sums became meanwhile.
E2C_DEV float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
E2C_DEV float max2(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
E2C_DEV bool no_softmax(float m) { return !(m < INFINITY); }
// two fp32 operations in one instruction
E2C_DEV float2 fma2(float2 a, float2 b, float2 c) {
    float2 y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(y))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return y;
}
E2C_DEV float2 add2(float2 a, float2 b) {
    float2 y;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(y))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return y;
}
E2C_DEV float2 mul2(float2 a, float2 b) {
    float2 y;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(y))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return y;
}
// 2^x of two values on the FMA pipe, for x <= 125: x = n + f with |f| <= 1/2 (adding 1.5 * 2^23 rounds to
// the whole number n and leaves it in the low bits), a polynomial of degree 4 in f fitted to the
// least relative error (2.7e-6 in fp32), and n added to the exponent. Below 2^-125 the result stays there.
// One exponential in kPoly pairs takes this way: the exponential unit's 16 a cycle are what
// bounds 64-wide heads, and nearly bound 128-wide ones (us with and without: the 4 prompts above, heads of
// 128 388 and 392, of 256 314 and 319; ragged prompts in a window, heads of 64 172 and 175).
constexpr int kPoly = 4;
E2C_DEV float2 ex2_poly(float2 x) {
    const float2 big = make_float2(12582912.f, 12582912.f), less = make_float2(-12582912.f, -12582912.f);
    x.x = fmaxf(x.x, -125.f);
    x.y = fmaxf(x.y, -125.f);
    const float2 r = add2(x, big), n = add2(r, less);
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 y = fma2(make_float2(9.5701e-3f, 9.5701e-3f), f, make_float2(5.591786e-2f, 5.591786e-2f));
    y = fma2(y, f, make_float2(2.4024745e-1f, 2.4024745e-1f));
    y = fma2(y, f, make_float2(6.9312181e-1f, 6.9312181e-1f));
    y = fma2(y, f, make_float2(9.9999926e-1f, 9.9999926e-1f));
    y.x = __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(r.x) << 23));
    y.y = __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(r.y) << 23));
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

// ---- pages of 8 bits (CODES). Codes become 16-bit numbers on their way from the stages that the loads fill to those that the
// products read, exactly (they are whole and at most 127): K's in q's type, V's in fp16. Scales stay out of the products; the
// softmax applies them, column by column. With kc = K's scale * c and vs V's:
//   logit_j = (q . code_j) kc_j,   m the largest logit_j + log2 vs_j of the keys that a row sees (less 2^8 at most)
//   out = sum_j P_j code_j / l,    P_j = 2^(logit_j - m) vs_j in fp16,   l = sum_j 2^(logit_j - m)
// so that P has the size that it has without scales, whatever theirs is, and a key adds what it adds whatever its neighbours
// and the keys out of sight are. (One power of two for a tile instead, near its largest scale, saves the logarithms' reads and
// loses every key whose scale is 2^14 below that one: a large token's neighbours, in sight of it or not.) Exponentials are held
// times 2^kSpare, and log2 vs is at least kLeastLog2: they reach 2^(8 + 96 + 16), a tile's sum 2^127, and at vs = 2^121,
// fp32's largest divided by 127, l still has the keys of weights down to 2^-21. A scale that is not finite makes its key, or the rows
// that meet its value, NaN. A head of zeros is held with the scale 1, but adds nothing: as a scale of 0 it leaves m to the others.
constexpr float kSpare = 16.0f, kLeastLog2 = -96.0f;
// log2 of a scale of V, and the scale as P's factor
E2C_DEV float scale_log2(float x) { return fabsf(x) < INFINITY ? fmaxf(lg2_approx(fabsf(x)), kLeastLog2) : 0.f; }
E2C_DEV float scale_factor(float x) { return fabsf(x) < INFINITY ? x * 0x1p-16f : NAN; }
// l 2^x by halves: m moves with the scales, by more than one factor can have, and l holds as much more or less
E2C_DEV float times_exp2(float l, float x) {
    const float half = ex2_approx(0.5f * x);
    return l * half * half;
}

// four codes as 16-bit floats
template <typename T>
E2C_DEV uint2 from_codes(uint32_t w);
// 128 + the low seven bits, less 128 or, with the sign's bit set, 256: bf16 holds both
template <>
E2C_DEV uint2 from_codes<__nv_bfloat16>(uint32_t w) {
    const uint32_t low = w & 0x7f7f7f7fu, sign = w & 0x80808080u;
    const uint32_t a = __byte_perm(low, 0x43434343u, 0x4140), b = __byte_perm(low, 0x43434343u, 0x4342);
    const uint32_t c = __byte_perm(sign, 0x43434343u, 0x4140), d = __byte_perm(sign, 0x43434343u, 0x4342);
    const __nv_bfloat162 x = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(a), reinterpret_cast<const __nv_bfloat162 &>(c));
    const __nv_bfloat162 y = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(b), reinterpret_cast<const __nv_bfloat162 &>(d));
    return make_uint2(reinterpret_cast<const uint32_t &>(x), reinterpret_cast<const uint32_t &>(y));
}
// 1024 + (code + 128), less 1152
template <>
E2C_DEV uint2 from_codes<__half>(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u, less = 0x64806480u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(reinterpret_cast<const __half2 &>(a), reinterpret_cast<const __half2 &>(less));
    const __half2 y = __hsub2(reinterpret_cast<const __half2 &>(b), reinterpret_cast<const __half2 &>(less));
    return make_uint2(reinterpret_cast<const uint32_t &>(x), reinterpret_cast<const uint32_t &>(y));
}
// sixteen columns' numbers, in registers
struct Columns {
    float4 x[4];
    E2C_DEV Columns(const float *p) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = reinterpret_cast<const float4 *>(p)[i];
    }
    E2C_DEV float2 operator[](int i) const { return i & 1 ? make_float2(x[i / 2].z, x[i / 2].w) : make_float2(x[i / 2].x, x[i / 2].y); }
};
// the products of sixteen columns times their kc
E2C_DEV void scale_logits(uint32_t (&s)[16], const Columns &k) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2 y = mul2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), k[i]);
        s[2 * i] = __float_as_uint(y.x), s[2 * i + 1] = __float_as_uint(y.y);
    }
}
// the same with the log2 of V's scales added, f
E2C_DEV void scale_logits(uint32_t (&s)[16], const Columns &k, const Columns &f) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2 y = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), k[i], f[i]);
        s[2 * i] = __float_as_uint(y.x), s[2 * i + 1] = __float_as_uint(y.y);
    }
}

// One stage: codes x of keys before `here` to y, zeros from there to `upto`. Eight neighbouring lanes
// take four pieces of 16 codes of row r and of row r ^ 5: with the loads' and the products' 128-byte swizzles these reads and both
// writes of each are in all banks. A thread's rows are 32 apart, which no swizzle tells apart, so that their addresses are constants
// away from one another: worked out for each piece they took half of this code.
// One piece a step: four at once took 189 us where this took 173 (6 prompts of 2000 tokens of texts of 2500, 12 heads of 64; 176 with
// the scales by column).
template <typename X, int D, int KIND, int ROWS>
E2C_DEV void convert_stage(const uint8_t *x, uint8_t *y, int here, int upto, int tid) {
    using C = Cfg<D, KIND>;
    // a panel of codes has ROWS rows of ROW bytes; the four warps take 32 rows by 64 bytes at a time
    constexpr int HALVES = C::ROW / 64, EACH = ROWS / 32, PARTS = C::CSTAGE / (ROWS * 64);
    const int pair = tid >> 3 & 3, r0 = (tid >> 5) * 8 + (tid & 4 ? pair ^ 5 : pair), piece = tid & 3;
    const uint32_t from = r0 * C::ROW + ((HALVES == 2 ? piece ^ (r0 & 7) : piece ^ (r0 >> 1 & 3)) << 4);
    y += r0 * 128;
    const int first = ((2 * piece) ^ (r0 & 7)) << 4;
#pragma unroll 1
    for (int part = 0; part < PARTS; part++) {  // of a panel's halves
        const uint8_t *p = x + (HALVES == 2 ? (part >> 1) * (ROWS * C::ROW) + (from ^ (part & 1) << 6) : from);
        uint4 next = *reinterpret_cast<const uint4 *>(p);
#pragma unroll 1
        for (int i = 0; i < EACH; i++, y += 32 * 128) {
            const uint4 c = next;
            if (i + 1 < EACH) next = *reinterpret_cast<const uint4 *>(p += 32 * C::ROW);
            uint2 s[4];
#pragma unroll
            for (int k = 0; k < 4; k++) s[k] = from_codes<X>((&c.x)[k]);
            if (here < ROWS) {  // the last keys' tile
                if (r0 + 32 * i >= here) s[0] = s[1] = s[2] = s[3] = make_uint2(0, 0);
                if (r0 + 32 * i >= upto) continue;
            }
            *reinterpret_cast<uint4 *>(y + first) = make_uint4(s[0].x, s[0].y, s[1].x, s[1].y);
            *reinterpret_cast<uint4 *>(y + (first ^ 16)) = make_uint4(s[2].x, s[2].y, s[3].x, s[3].y);
        }
    }
}

// Whether the codes of a key's head of v, whose scale is 1, are zeros. From the pages, since scales are prepared before V's codes
// have arrived; other heads' scales are hardly ever 1.
template <int D>
E2C_DEV bool zero_codes(const Args &p, const Item &it, int key) {
    if (it.seq < 0) return false;
    const int shift = 31 - __clz(p.pc.page), page = p.pc.table[(int64_t)it.seq * p.pc.max_blocks + (key >> shift)];
    if ((unsigned)page >= (unsigned)p.pc.n_pages) return false;  // reported where its codes are loaded
    const int64_t row = ((int64_t)page << shift) + (key & (p.pc.page - 1));
    const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const int8_t *>(p.pc.v) + (row * p.pc.KV + it.kvh) * D);
    uint32_t any = 0;
#pragma unroll 1
    for (int i = 0; i < D / 16 && any == 0; i += 4)
#pragma unroll
        for (int k = 0; k < 4; k++) any |= x[i + k].x | x[i + k].y | x[i + k].z | x[i + k].w;
    return any == 0;
}

// Four warps for K (w < 4) and four for V: every stage's codes, of as many keys as the product takes, into the 128-byte swizzle that
// it reads; rows past the last key become zeros. K's warps also prepare the tile's scales.
template <typename T, int D, int KIND, typename Bar, typename Take>
E2C_DEV void convert_codes(const Args &p, uint8_t *smem, int w, int lane, Bar bar, Take take) {
    using C = Cfg<D, KIND>;
    const bool is_v = w >= 4;
    const int tid = (w & 3) * 32 + lane;
    const int FULL = is_v ? B_VCF : B_KCF, FREE = is_v ? B_VCE : B_KCE, NST = is_v ? C::NVC : C::NKC;
    const int OUT = is_v ? B_VF : B_KF, TAKEN = is_v ? B_VE : B_KE, NOUT = is_v ? C::NVS : C::NKS;
    const int pitch = is_v ? C::CSTAGE : C::KCSTAGE;
    const uint8_t *ring = smem + (is_v ? C::VC_OFF : C::KC_OFF);
    uint8_t *to = smem + (is_v ? C::V_OFF : C::K_OFF);
    int st = 0, out = 0, g = 0;
    uint32_t sp = 0, op = 1;
    Item it;
    for (int n = 0; take(n, it); n++) {
#pragma unroll 1
        for (int j = 0; j < it.nt; j++, g++) {
            const int nk = min(TK, tile_end<KIND>(p, it, j) - tile_key<KIND>(it, j)), sb = g % C::NC;
            float *sc = reinterpret_cast<float *>(smem + C::SC_OFF) + sb * C::SC;
#pragma unroll 1
            for (int h = 0; h < C::KPARTS; h++) {
                if (!wait_warp(bar(FULL + st), sp, p.status, E2C_ERR_WAIT_PRODUCER)) return;
                const uint8_t *x = ring + st * pitch;
                if (h == 0 && !is_v) {
                    const float *from = reinterpret_cast<const float *>(x + C::CSTAGE);
                    if (!wait_warp(bar(B_SCE + sb), (uint32_t)(((g / C::NC) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER)) return;
                    sc[tid] = tid < nk ? from[tid] * p.c : 0.f;
                    float vs = tid < nk ? from[TK + tid] : 0.f;
                    if (vs == 1.f && zero_codes<D>(p, it, tile_key<KIND>(it, j) + tid)) vs = 0.f;
                    sc[TK + tid] = scale_log2(vs);
                    sc[2 * TK + tid] = scale_factor(vs);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_SCF + sb));
                }
                if (!wait_warp(bar(TAKEN + out), op, p.status, E2C_ERR_WAIT_PRODUCER)) return;
                const int here = is_v ? min(nk - h * C::VROWS, C::VROWS) : nk, upto = (here + 15) & ~15;
                uint8_t *y = to + out * C::STAGE;
                if (is_v || (__is_same(T, __half) && C::VROWS == TK))
                    convert_stage<__half, D, KIND, C::VROWS>(x, y, here, upto, tid);
                else
                    convert_stage<T, D, KIND, TK>(x, y, here, upto, tid);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(OUT + out));
                    mbar_arrive(bar(FREE + st));
                }
                if (++st == NST) {
                    st = 0;
                    sp ^= 1;
                }
                if (++out == NOUT) {
                    out = 0;
                    op ^= 1;
                }
            }
        }
    }
}

template <typename T, int D, int KIND>
__global__ void __launch_bounds__(Cfg<D, KIND>::NTHREADS, 1)
    k_attention_pages(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQp,
                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ Args p, const int q_box, const int qp_box) {
    using C = Cfg<D, KIND>;
    using X = std::conditional_t<C::CODE, __half, T>;  // of the second product's operands
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    if (smem_u32(smem) & 1023) {
        griddep_wait();
        if (threadIdx.x == 0) record_status(p.status, E2C_ERR_SMEM_ALIGN);
        if (blockIdx.x == 0 && threadIdx.x < 2) p.before[p.n + threadIdx.x] = 0;  // the join has nothing to do
        return;
    }
    const uint32_t sbase = smem_u32(smem);
    auto bar = [&](int i) { return sbase + C::BARS + 8u * i; };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + C::BARS + B_NUM * 8);
    Item *items = reinterpret_cast<Item *>(smem + C::ITEMS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == C::W_ITEMS && lane == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(B_QF + i), 1);
            mbar_init(bar(B_QE + i), 1);
            mbar_init(bar(B_PV + i), 1);
            mbar_init(bar(B_OF + i), 1);
            mbar_init(bar(B_OE + i), 4);
            mbar_init(bar(B_MLF + i), 4 * C::NG);
            mbar_init(bar(B_MLE + i), 4);
        }
        for (int i = 0; i < 3; i++) {
            mbar_init(bar(B_SF + i), 1);
            mbar_init(bar(B_PF + i), 4);
        }
        for (int i = 0; i < 4 * C::NG; i++) mbar_init(bar(B_MX + i), 1);
        for (int i = 0; i < NI; i++) {
            mbar_init(bar(B_ITF + i), 1);
            mbar_init(bar(B_ITE + i), 8 + 4 * C::NG + (C::CODE ? 8 : 0));  // K, V, QK, PV, the epilogue, softmax and converting warps
        }
        for (int i = 0; i < 5; i++) {
            mbar_init(bar(B_KF + i), C::CODE ? 4 : 1);
            mbar_init(bar(B_KE + i), 1);
            mbar_init(bar(B_VF + i), C::CODE ? 4 : 1);
            mbar_init(bar(B_VE + i), 1);
        }
        for (int i = 0; C::CODE && i < 4; i++) {
            mbar_init(bar(B_KCF + i), 1);
            mbar_init(bar(B_KCE + i), 4);
            mbar_init(bar(B_VCF + i), 1);
            mbar_init(bar(B_VCE + i), 4);
            mbar_init(bar(B_SCF + i), 4);
            mbar_init(bar(B_SCE + i), 4);
        }
        mbar_init(bar(B_DRAIN), 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == C::W_MMA) {
        tmem_alloc(sbase + C::BARS + B_NUM * 8, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = *tmem_slot;

    Plan pl;
    make_plan<C::WARPS, KIND>(p, pl, *reinterpret_cast<PlanScratch<C::WARPS> *>(smem + C::SCAN));

    // A consumer's copy of item n; false after the last one (or a failure). The slot is released at once.
    auto take = [&](int n, Item &it) -> bool {
        const int s = n & (NI - 1);
        if (!wait_warp(bar(B_ITF + s), (uint32_t)((n / NI) & 1), p.status, E2C_ERR_WAIT_ATTN)) return false;
        const int4 *d = reinterpret_cast<const int4 *>(items + s);
        int4 *o = reinterpret_cast<int4 *>(&it);
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = d[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_ITE + s));
        return it.ntok >= 0;
    };

    // CODES: 768 threads begin with 80 registers each; the softmax's take of the others': (2 * 104 + 72 + 72 + 2 * 64) / 6 = 80
    if constexpr (C::CODE) {
        static_assert(C::REGISTERS == 768 * 80 && C::NTHREADS == 768, "shares of registers");
        if (warp < C::W_EPI)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_SOFTMAX));
        else if (warp < C::W_CONVERT)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_OTHERS));
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_CONVERT));
    }
    if (C::CODE && warp >= C::W_CONVERT) {
        convert_codes<T, D, KIND>(p, smem, warp - C::W_CONVERT, lane, bar, take);
    } else if (warp >= C::W_ITEMS) {
        if (warp == C::W_ITEMS) {
            // ------------------------------------------------------------ items and Q loads
            const int L0 = pl.share.begin(blockIdx.x), L1 = pl.share.begin(blockIdx.x + 1);
            if (p.shared == 0 && lane == 0 && L0 < L1) p.split[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
            __syncwarp();
            int n = 0;
            bool ok = true;
            Item it = {};
            // Q of an item is loaded once the next one is published: the K and V loads then know of an item more
            // than Q's buffers hold
            int q_t0 = 0, q_kvh = 0, q_prefix = 0, loaded = 0;
            auto load_q = [&]() {
                const int qb = loaded % C::NQ;
                if (!(ok = wait_warp(bar(B_QE + qb), (uint32_t)(((loaded / C::NQ) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER))) return;
                if (elect_one()) {
                    const CUtensorMap *tm = q_prefix ? &tmQp : &tmQ;
                    mbar_arrive_expect_tx(bar(B_QF + qb), (uint32_t)(C::PANELS * (q_prefix ? qp_box : q_box) * p.G * 128));
#pragma unroll
                    for (int i = 0; i < C::PANELS; i++)
                        tma_load_3d(sbase + qb * C::Q_BYTES + i * (TR * 128), tm, 64 * i, q_kvh * p.G, q_t0, bar(B_QF + qb));
                }
                __syncwarp();
                loaded++;
            };
            auto publish = [&]() {
                const int sl = n & (NI - 1);
                if (!(ok = wait_warp(bar(B_ITE + sl), (uint32_t)(((n / NI) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER))) return;
                if (lane == 0) {
                    const int4 *d = reinterpret_cast<const int4 *>(&it);
                    int4 *o = reinterpret_cast<int4 *>(items + sl);
#pragma unroll
                    for (int k = 0; k < 4; k++) o[k] = d[k];
                    mbar_arrive(bar(B_ITF + sl));
                }
                __syncwarp();
                if (n++ > 0) load_q();
                q_t0 = it.t0;
                q_kvh = it.kvh;
                q_prefix = it.prefix;
            };
            // Neighbours share a run of the prefix; every other group of them begins with its sequence items, so
            // that products (the prefix) and loads (the sequences) go on side by side.
            const bool late = pl.share.items > 0 && (blockIdx.x / pl.npt & 1);
#pragma unroll 1
            for (int half = 0; half < 2; half++) {
                if ((half == 1) == late) {
                    it.prefix = 1;
                    it.masked = pl.masked;
                    it.seq = pl.pseq;
                    it.dst = TO_SLOT;
#pragma unroll 1
                    for (int q = blockIdx.x; ok && q < pl.share.items; q += gridDim.x) {
                        const int u = q / pl.npt, rt = q - u * pl.npt, kvh = u / pl.share.splits, s = u - kvh * pl.share.splits;
                        it.kvh = kvh;
                        it.t0 = rt * p.tpt;
                        it.ntok = min(p.tpt, p.T - it.t0);
                        pl.pspan.cut(p, s * pl.share.chunk, min(pl.share.chunk, pl.ptiles - s * pl.share.chunk), it);
                        it.klim = min(it.klim, tile_key<KIND>(it, it.nt - 1) + TK);
                        it.slot = 2 * gridDim.x + q;
                        publish();
                    }
                    continue;
                }
                it.prefix = 0;
                it.base = p.shared;
                it.masked = 1;
                Walk<KIND> walk;
                walk.begin(pl, L0, L1);
#pragma unroll 1
                while (ok && walk.next(p, pl, it, lane)) publish();
            }
            // the last one, after which Q of the last item follows
            if (ok) {
                const bool any = n > 0;
                if (wait_warp(bar(B_ITE + (n & (NI - 1))), (uint32_t)(((n / NI) & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER)) {
                    if (lane == 0) {
                        items[n & (NI - 1)].ntok = -1;
                        mbar_arrive(bar(B_ITF + (n & (NI - 1))));
                    }
                    __syncwarp();
                    if (any) load_q();
                }
            }
            // every load that was issued has landed before the block may end
            for (int i = loaded - C::NQ < 0 ? 0 : loaded - C::NQ; i < loaded; i++)
                wait_warp(bar(B_QF + i % C::NQ), (uint32_t)((i / C::NQ) & 1), nullptr, E2C_ERR_WAIT_DRAIN);
        } else if (warp == C::W_MMA) {
            // ------------------------------------------------------------ MMA issue (one thread)
            // QK runs LOOK tiles ahead of PV; each has a cursor over the items
            if (elect_one()) {
                constexpr int LOOK = C::NS - 1;
                constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(128 >> 4) << 24);
                constexpr uint32_t id_pv = idesc | type_bits<X>() | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // B: N contiguous
                const uint32_t id_qk = idesc | type_bits<T>() | (p.neg << 13);
                auto wait1 = [&](int b, uint32_t parity) -> bool {
#pragma unroll 1
                    for (uint32_t i = 0; i < kTries; i++)
                        if (mbar_try_wait_sleep(bar(b), parity, kTryNs)) return true;
                    record_status(p.status, E2C_ERR_WAIT_MMA);
                    return false;
                };
                // the keys and tiles of item n; no tiles: the last one
                // (SIGHT: keys are those of its first ns tiles, if any, and more those of the tiles after them)
                auto item = [&](int n, int &left, int &keys, int &ns, int &more) -> bool {
                    const int s = n & (NI - 1);
                    if (!wait1(B_ITF + s, (uint32_t)((n / NI) & 1))) return false;
                    left = items[s].ntok < 0 ? 0 : items[s].nt;
                    keys = items[s].klim - items[s].k0;
                    if (KIND & SIGHT) {
                        ns = items[s].ns;
                        more = keys - ns * TK - items[s].gap;
                        if (ns > 0) keys = p.sinks - items[s].k0;
                    }
                    mbar_arrive(bar(B_ITE + s));
                    return true;
                };
                int nq = 0, nv = 0;          // items taken
                int lq = 0, lv = 0;          // tiles of the item left
                int kq = 0, kv = 0;          // keys left
                int sq_n = 0, sv_n = 0, kq2 = 0, kv2 = 0;  // tiles of sinks left, and the keys after them
                int ks = 0, vs = 0;          // stages, and the parity of their round
                uint32_t kp = 0, vp = 0;
                int sq = 0, sv = 0;          // S buffers
                uint32_t pp = 0;             // parity of P in S buffer sv
                int ahead = 0, odd = 0;      // QK products not yet used; parity of PV's tile
                bool more = true, ok = true; // more: QK has tiles left
                int qb = 0, ob = 0;          // Q and O buffers, and their parities
                uint32_t qp = 0, op = 1;
                bool first = false;
#pragma unroll 1
                while (ok && (more || ahead > 0)) {
                    // with one Q buffer an item's first QK waits for the last PV before it
                    const bool qk_now = more && (C::CROSS || lq > 0 || ahead == 0);
                    if (qk_now) {
                        if (lq == 0) {
                            if (!(ok = item(nq, lq, kq, sq_n, kq2))) break;
                            if (lq == 0) {
                                more = false;
                                continue;
                            }
                            qb = nq % C::NQ;
                            qp = (uint32_t)((nq / C::NQ) & 1);
                            nq++;
                            if (!(ok = wait1(B_QF + qb, qp))) break;
                        }
                        const uint32_t id = id_qk | (uint32_t)(((min(TK, kq) + 15) >> 4) << 1) << 17;
                        const uint32_t d = tmem + (uint32_t)(sq * 128);
                        lq--;
                        kq -= TK;
                        if (KIND & SIGHT && --sq_n == 0) kq = kq2;
                        uint64_t qd = smem_desc_sw128(sbase + qb * C::Q_BYTES);
#pragma unroll
                        for (int h = 0; h < C::KPARTS; h++) {
                            if (!(ok = wait1(B_KF + ks, kp))) break;
                            const uint64_t kd = smem_desc_sw128(sbase + C::K_OFF + ks * C::STAGE);
#pragma unroll
                            for (int k = 0; k < C::PANELS / C::KPARTS * 4; k++) {
                                const int off = ((k >> 2) * (TR * 128) + (k & 3) * 32) >> 4;
                                mma_bf16(d, qd + off, kd + off, id, h != 0 || k != 0);
                            }
                            mma_commit(bar(B_KE + ks));
                            qd += (C::PANELS / C::KPARTS * TR * 128) >> 4;
                            if (++ks == C::NKS) {
                                ks = 0;
                                kp ^= 1;
                            }
                        }
                        if (!ok) break;
                        mma_commit(bar(B_SF + sq));
                        if (lq == 0) mma_commit(bar(B_QE + qb));
                        if (++sq == C::NS) sq = 0;
                        ahead++;
                    }
                    if (ahead > LOOK || (ahead > 0 && !qk_now) || (ahead > 0 && !more)) {
                        if (lv == 0) {
                            if (!(ok = item(nv, lv, kv, sv_n, kv2))) break;  // QK has taken it: it is there
                            ob = nv % C::NO;
                            op = (uint32_t)(((nv / C::NO) & 1) ^ 1);
                            nv++;
                            first = true;
                        }
                        const int nk16 = (min(TK, kv) + 15) & ~15;
                        const uint32_t d = tmem + (uint32_t)(C::O_COL + ob * D);
                        uint32_t a = tmem + (uint32_t)(sv * 128);
                        lv--;
                        kv -= TK;
                        if (KIND & SIGHT && --sv_n == 0) kv = kv2;
                        if (!(ok = wait1(B_PF + sv, pp))) break;
                        if (first && !(ok = wait1(B_OE + ob, op))) break;
                        tc_fence_after();
#pragma unroll
                        for (int h = 0; h < C::KPARTS; h++) {  // half tiles of V
                            if (!(ok = wait1(B_VF + vs, vp))) break;
                            const uint64_t vd = smem_desc_sw128_mn(sbase + C::V_OFF + vs * C::STAGE, C::VROWS * 128);
                            const int here = min(C::VROWS, nk16 - h * C::VROWS);
#pragma unroll 2
                            for (int k = 0; k < here / 16; k++)
                                mma_bf16_ts(d, a + 8 * k, vd + 128 * k, id_pv, !first || h != 0 || k != 0);
                            mma_commit(bar(B_VE + vs));
                            a += C::VROWS / 2;
                            if (++vs == C::NVS) {
                                vs = 0;
                                vp ^= 1;
                            }
                        }
                        if (!ok) break;
                        mma_commit(bar(B_PV + odd));
                        odd ^= 1;
                        if (lv == 0) mma_commit(bar(B_OF + ob));
                        first = false;
                        if (++sv == C::NS) {
                            sv = 0;
                            pp ^= 1;
                        }
                        ahead--;
                    }
                }
                // all products are done before the block frees tensor memory or ends
                mma_commit(bar(B_DRAIN));
                wait1(B_DRAIN, 0);
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------------ K loads, V loads
            const bool is_v = warp == C::W_V;
            const CUtensorMap *tm = is_v ? &tmV : &tmK;
            const int F = C::CODE ? (is_v ? B_VCF : B_KCF) : is_v ? B_VF : B_KF, E = C::CODE ? (is_v ? B_VCE : B_KCE) : is_v ? B_VE : B_KE;
            const int NST = C::CODE ? (is_v ? C::NVC : C::NKC) : is_v ? C::NVS : C::NKS;
            const uint32_t ring = sbase + (C::CODE ? (is_v ? C::VC_OFF : C::KC_OFF) : is_v ? C::V_OFF : C::K_OFF);
            const int PB = min(p.pc.page, C::VROWS), shift = 31 - __clz(p.pc.page);
            Item it = {};
            int n = 0, j = 0, st = 0, total = 0;
            uint32_t par = 1;
            // the tile whose boxes are issued next, its rows asked for one tile before
            int row = 0, kvh = 0, nk = 0;
            bool ok = true, have = false, more = true;
#pragma unroll 1
            while (ok) {
                int row2 = 0, kvh2 = 0, nk2 = 0;
                bool have2 = false;
                if (more && j == it.nt) {
                    more = take(n, it);
                    ok = more || it.ntok < 0;
                    n++;
                    j = 0;
                }
                if (more) {
                    const int kk = tile_key<KIND>(it, j), end = tile_end<KIND>(p, it, j), key = kk + lane * PB;
                    int page = 0;
                    if (it.seq >= 0 && key < min(end, kk + TK))
                        page = p.pc.table[(int64_t)it.seq * p.pc.max_blocks + (key >> shift)];
                    if ((unsigned)page >= (unsigned)p.pc.n_pages) {  // page 0 instead, reported
                        record_status(p.status, E2C_ERR_BAD_SEQ);
                        page = 0;
                    }
                    row2 = (page << shift) + (key & (p.pc.page - 1));
                    nk2 = min(TK, end - kk);
                    kvh2 = it.kvh;
                    have2 = true;
                    j++;
                }
                if (have) {
                    const int nb = (nk + PB - 1) / PB;
                    // a K stage holds PANELS / KPARTS panels of every key, a V stage every panel of VROWS keys
                    const int np = is_v ? C::PANELS : C::PANELS / C::KPARTS;
                    const int pitch = (is_v ? C::VROWS : TK) * 128;
#pragma unroll 1
                    for (int h = 0; h < C::KPARTS; h++) {
                        const int b0 = is_v ? min(nb, h * C::VROWS / PB) : 0, b1 = is_v ? min(nb, (h + 1) * C::VROWS / PB) : nb;
                        const int x = kvh * D + (is_v ? 0 : h * np * 64);
                        // the first rows are in every lane before the wait: from a free stage to its loads is the
                        // shortest way
                        int y = __shfl_sync(0xffffffffu, row, b0), y2 = __shfl_sync(0xffffffffu, row, min(b0 + 1, 31));
                        if (!(ok = wait_warp(bar(E + st), par, p.status, E2C_ERR_WAIT_PRODUCER))) break;
                        const uint32_t full = bar(F + st);
                        if constexpr (C::CODE) {
                            // panels of ROW bytes a key, and with a tile's first codes of K the scales of both
                            constexpr int WIDE = D == 256 ? 2 : 1;
                            const int panels = is_v ? WIDE : 1;
                            const bool scales = !is_v && h == 0;
                            uint32_t dst = ring + st * (is_v ? C::CSTAGE : C::KCSTAGE), sd = ring + st * C::KCSTAGE + C::CSTAGE;
                            const int x8 = kvh * D + (is_v ? 0 : h * C::ROW);
                            if (elect_one()) mbar_arrive_expect_tx(full, (uint32_t)((b1 - b0) * PB * (panels * C::ROW + (scales ? 8 : 0))));
                            __syncwarp();
#pragma unroll 1
                            for (int b = b0; b < b1; b++, dst += PB * C::ROW, sd += PB * 4) {
                                if (elect_one()) {
                                    tma_load_2d(dst, tm, x8, y, full);
                                    if (WIDE == 2 && is_v) tma_load_2d(dst + C::VROWS * C::ROW, tm, x8 + C::ROW, y, full);
                                    if (scales) {
                                        const int64_t at = ((int64_t)(y >> shift) * p.pc.KV + kvh) * p.pc.page + (y & (p.pc.page - 1));
                                        bulk_load(sd, p.pc.ks + at, (uint32_t)PB * 4, full);
                                        bulk_load(sd + TK * 4, p.pc.vs + at, (uint32_t)PB * 4, full);
                                    }
                                }
                                y = y2;
                                y2 = __shfl_sync(0xffffffffu, row, min(b + 2, 31));
                            }
                            if (++st == NST) {
                                st = 0;
                                par ^= 1;
                            }
                            total++;
                            continue;
                        }
                        uint32_t dst = ring + st * C::STAGE;
                        if (elect_one()) mbar_arrive_expect_tx(full, (uint32_t)((b1 - b0) * PB * 128 * np));
                        __syncwarp();
#pragma unroll 1
                        for (int b = b0; b < b1; b++, dst += PB * 128) {
                            if (elect_one()) {
#pragma unroll
                                for (int i = 0; i < C::PANELS; i++)
                                    if (i < np) tma_load_2d(dst + i * pitch, tm, x + 64 * i, y, full);
                            }
                            y = y2;
                            y2 = __shfl_sync(0xffffffffu, row, min(b + 2, 31));
                        }
                        if (++st == NST) {
                            st = 0;
                            par ^= 1;
                        }
                        total++;
                    }
                } else if (!more) {
                    break;
                }
                row = row2;
                kvh = kvh2;
                nk = nk2;
                have = have2;
            }
            for (int i = total - NST < 0 ? 0 : total - NST; i < total; i++)
                wait_warp(bar(F + i % NST), (uint32_t)((i / NST) & 1), nullptr, E2C_ERR_WAIT_DRAIN);
        }
    } else if (warp < C::W_EPI) {
        // ---------------------------------------------------------------- softmax
        constexpr int NG = C::NG;
        const int quad = warp & 3, group = warp >> 2, prev = (group + NG - 1) % NG, row = quad * 32 + lane;
        const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16);
        float *xm = reinterpret_cast<float *>(smem + C::XM);
        float2 *ml = reinterpret_cast<float2 *>(smem + C::ML);
        const int tok = row / p.G;
        bool ok = true;
        int g = 0;
        Item it;
        for (int item = 0; take(item, it); item++) {
            const bool live = tok < it.ntok;
            const bool busy = quad * 32 < it.ntok * p.G;  // some row of this warp is live
            int lo = 0, hi = it.klim;
            Seen sight = {};
            if (KIND & SIGHT && live && it.masked) {
                const int t = it.t0 + tok;
                int pos = it.pos0 + tok, len = it.len, first = it.base;
                if (it.prefix) {
                    int last;
                    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last);
                    const int seq = i < 0 ? -1 : p.seqs[i];
                    len = (unsigned)seq < (unsigned)p.pc.max_seqs ? min(max(p.pc.len[seq], 0), p.pc.max_blocks * p.pc.page) : 0;
                    pos = len - (last - t);
                    first = i < 0 ? 0 : len - (last - p.q_start[i]);
                }
                sight.set(p, t, pos, len, first);
                lo = sight.lo = max(sight.lo, it.prefix ? 0 : p.shared);
                hi = sight.hi = min(hi, sight.hi);
            } else if (live && it.masked) {
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
                if (g % NG != group) continue;
                const int sb = g % C::NS, kk = tile_key<KIND>(it, j), nk = min(TK, tile_end<KIND>(p, it, j) - kk);
                // the running maximum, from the tile before (its wait runs while this tile's products do)
                if (g > 0 && !wait_warp(bar(B_MX + prev * 4 + quad), (uint32_t)(((g - 1) / NG) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                    ok = false;
                    break;
                }
                const float before = j > 0 ? xm[prev * TR + row] : -INFINITY;
                if (!wait_warp(bar(B_SF + sb), (uint32_t)((g / C::NS) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t ts = ta + (uint32_t)(sb * 128);
                const int ra = lo - kk, rb = max(hi - kk, ra);  // columns [ra, rb) are seen
                const bool masked = __any_sync(0xffffffffu, live && (ra > 0 || rb < TK));
                // The columns are read twice, for the maximum and for the exponentials, in loops short enough
                // for the instruction cache: a row of 128 logits held in registers is straight code that does
                // not stay in it (the 4 prompts above, 16 heads of 128: 443 us, 370 with loops of 64 columns; of 32, 368)
                // columns from the next 16 bits of `row` (SIGHT), or from [ra, rb), on
                uint32_t row4[4] = {};
                if (KIND & SIGHT && masked && live) {
                    const int from = it.prefix ? 0 : p.shared;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        row4[i] = it.masked ? sight.keys(p, kk + 32 * i) & Seen::between(from - kk - 32 * i, it.klim - kk - 32 * i)
                                            : Seen::below(it.klim - kk - 32 * i);
                }
                auto hide = [&](int c0, uint32_t (&s)[16], uint32_t (&row)[4]) {
                    // bit i: column c0 + i is seen
                    uint32_t seen;
                    if (KIND & SIGHT) {
                        seen = row[0] & 0xffffu;
#pragma unroll
                        for (int i = 0; i < 4; i++) row[i] = __funnelshift_r(row[i], i < 3 ? row[i + 1] : 0u, 16);
                    } else {
                        const int a = min(max(ra - c0, 0), 16), b = min(max(rb - c0, 0), 16);
                        seen = (1u << b) - (1u << a);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) s[i] = seen & (1u << i) ? s[i] : 0xff800000u;
                };
                const float *sc = reinterpret_cast<const float *>(smem + C::SC_OFF) + (g % C::NC) * C::SC;
                if (C::CODE && !wait_warp(bar(B_SCF + g % C::NC), (uint32_t)((g / C::NC) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                    ok = false;
                    break;
                }
                float mx = -INFINITY;
                if (busy) {
                    float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (C::CODE && !masked) {
#pragma unroll 1
                        for (int c0 = 0; c0 < TK; c0 += 16) {  // (and below: with 32 columns a step a call of 173 us took 200)
                            uint32_t s[16];
                            tmem_ld16(ts + c0, s);
                            const Columns k(sc + c0), f(sc + TK + c0);  // they arrive while the products do
                            tmem_wait_ld();
                            scale_logits(s, k, f);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) mm[i / 2 & 3] = max3(mm[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        }
                    } else if (!masked) {
#pragma unroll 1
                        for (int c0 = 0; c0 < TK; c0 += 32) {
                            uint32_t s[32];
                            tmem_ld32(ts + c0, s);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 2) mm[i / 2 & 3] = max3(mm[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        }
                    } else {
                        uint32_t row4c[4] = {row4[0], row4[1], row4[2], row4[3]};
#pragma unroll 1
                        for (int c0 = 0; c0 < nk; c0 += 16) {
                            uint32_t s[16];
                            tmem_ld16(ts + c0, s);
                            if constexpr (C::CODE) {
                                const Columns k(sc + c0), f(sc + TK + c0);
                                tmem_wait_ld();
                                scale_logits(s, k, f);
                            } else {
                                tmem_wait_ld();
                            }
                            hide(c0, s, row4c);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) mm[i / 2 & 3] = max3(mm[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        }
                    }
                    mx = max2(max2(mm[0], mm[1]), max2(mm[2], mm[3]));
                    if (!C::CODE) mx *= p.c;
                }
                float now = before, alpha = 1.f;
                if (live && !(mx <= before + kRescaleLog2)) {  // so also from -infinity, and for a NaN
                    now = max2(before, mx);
                    alpha = ex2_approx(before - now);
                }
                xm[group * TR + row] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_MX + group * 4 + quad));
                if (busy) {
                    if (now != m) {
                        l = C::CODE ? times_exp2(l, m - now) : l * ex2_approx(m - now);
                        m = now;
                    }
                    if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // O holds the tiles before this one once their products are done
                        if (!wait_warp(bar(B_PV + ((g - 1) & 1)), (uint32_t)(((g - 1) >> 1) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t to = ta + (uint32_t)(C::O_COL + item % C::NO * D);
#pragma unroll 1
                        for (int c = 0; c < D / 16; c++) {
                            uint32_t o[16];
                            tmem_ld16(to + 16 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st16(to + 16 * c, o);
                        }
                        tmem_wait_st();
                    }
                    // a row that has seen nothing yet has only -inf: any finite maximum gives it zeros
                    const float2 cc = make_float2(p.c, p.c);
                    const float mneg = m == -INFINITY ? 0.f : C::CODE ? kSpare - m : -m;
                    const float2 mm = make_float2(mneg, mneg);
                    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
                    if (C::CODE && !masked) {
#pragma unroll 1
                        for (int c0 = 0; c0 < TK; c0 += 16) {
                            uint32_t s[16], pk[8];
                            tmem_ld16(ts + c0, s);
                            const Columns k(sc + c0), v(sc + 2 * TK + c0);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                float2 x = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), k[i], mm);
                                x = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                                sum[i & 1] = add2(sum[i & 1], x);
                                x = mul2(x, v[i]);
                                pk[i] = pack2<X>(x.x, x.y);
                            }
                            tmem_st8(ts + c0 / 2, pk);
                        }
                    } else if (!masked) {
#pragma unroll 1
                        for (int c0 = 0; c0 < TK; c0 += 32) {
                            uint32_t s[32], pk[16];
                            tmem_ld32(ts + c0, s);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float2 x = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), cc, mm);
                                x = i % kPoly == kPoly - 1 ? ex2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
                                sum[i & 1] = add2(sum[i & 1], x);
                                pk[i] = pack2<X>(x.x, x.y);
                            }
                            tmem_st16(ts + c0 / 2, pk);
                        }
                    } else {
#pragma unroll 1
                        for (int c0 = 0; c0 < nk; c0 += 16) {
                            uint32_t s[16], pk[8];
                            tmem_ld16(ts + c0, s);
                            if constexpr (C::CODE) {  // before what is hidden becomes -infinity: a scale may be zero
                                const Columns k(sc + c0);
                                tmem_wait_ld();
                                scale_logits(s, k);
                            } else {
                                tmem_wait_ld();
                            }
                            hide(c0, s, row4);
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float2 y = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
                                float2 x = C::CODE ? add2(y, mm) : fma2(y, cc, mm);
                                x = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                                sum[i & 1] = add2(sum[i & 1], x);
                                if constexpr (C::CODE) x = mul2(x, *reinterpret_cast<const float2 *>(sc + 2 * TK + c0 + 2 * i));
                                pk[i] = pack2<X>(x.x, x.y);
                            }
                            tmem_st8(ts + c0 / 2, pk);
                        }
                    }
                    const float2 all = add2(sum[0], sum[1]);
                    l += C::CODE ? (all.x + all.y) * 0x1p-16f : all.x + all.y;
                    tmem_wait_st();
                }
                if (C::CODE) {  // the tile's scales have been read
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_SCE + g % C::NC));
                } else if (nk & 15) {
                    // V's rows past the last key, up to the product's 16: each of the group's warps zeroes panels
                    const int part = nk / C::VROWS, vt = g * C::KPARTS + part, vs = vt % C::NVS;
                    // Parities tell only neighbouring phases apart: the stage's load before this one, of tile
                    // g - BACK, must be known to have landed. S(g) says so of tile g - NS; for a shorter ring its
                    // product is waited for.
                    constexpr int BACK = C::NVS / C::KPARTS;
                    if (BACK < C::NS && g >= BACK &&
                        !wait_warp(bar(B_PV + ((g - BACK) & 1)), (uint32_t)(((g - BACK) >> 1) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                        ok = false;
                        break;
                    }
                    if (!wait_warp(bar(B_VF + vs), (uint32_t)((vt / C::NVS) & 1), p.status, E2C_ERR_WAIT_ATTN)) {
                        ok = false;
                        break;
                    }
                    const int pieces = (16 - (nk & 15)) * 8;  // of 16 bytes, in one panel
#pragma unroll 1
                    for (int panel = quad; panel < C::PANELS; panel += 4) {
                        uint8_t *v = smem + C::V_OFF + vs * C::STAGE + panel * (C::VROWS * 128) + (nk - part * C::VROWS) * 128;
#pragma unroll 1
                        for (int x = lane; x < pieces; x += 32) *reinterpret_cast<uint4 *>(v + x * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PF + sb));
            }
            if (!ok) break;
            // the slot's last reader was the epilogue two items ago
            if (!wait_warp(bar(B_MLE + (item & 1)), (uint32_t)(((item >> 1) & 1) ^ 1), p.status, E2C_ERR_WAIT_ATTN))
                break;
            ml[((item & 1) * NG + group) * TR + row] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_MLF + (item & 1)));
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3, row = quad * 32 + lane;
        const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16);
        const float2 *ml = reinterpret_cast<const float2 *>(smem + C::ML);
        const int tok = row / p.G, hd = row - tok * p.G;
        Item it;
        for (int item = 0; take(item, it); item++) {
            const int ob = item % C::NO;
            if (!wait_warp(bar(B_MLF + (item & 1)), (uint32_t)((item >> 1) & 1), p.status, E2C_ERR_WAIT_EPI))
                break;
            float2 a[C::NG];
#pragma unroll
            for (int i = 0; i < C::NG; i++) a[i] = ml[((item & 1) * C::NG + i) * TR + row];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_MLE + (item & 1)));
            // the groups' sums, to the largest maximum; l = 0: every logit was -infinity, or no key was seen
            float m = a[0].x, l = 0.f;
#pragma unroll
            for (int i = 1; i < C::NG; i++) m = max2(m, a[i].x);
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < C::NG; i++) l += C::CODE ? times_exp2(a[i].y, a[i].x - ref) : a[i].y * ex2_approx(a[i].x - ref);
            const bool live = tok < it.ntok, bad = no_softmax(m), some = bad || l > 0.f;
            const float inv = bad ? NAN : some ? __fdividef(1.0f, l) : 0.f;
            float none = 0.f;  // the result of a row with l = 0; a part leaves that to the join
            const int64_t t = it.t0 + tok;
            const int h = it.kvh * p.G + hd;
            const bool busy = quad * 32 < it.ntok * p.G;
            T *out = nullptr;
            float *part = nullptr;
            if (busy) {
                const float sums = bad ? m : some ? m + __log2f(l) : -INFINITY;
                if (it.dst == TO_OUT) {
                    if (!some && sees_keys<KIND>(p, t, it.pos0 + tok, it.len, it.base)) none = NAN;
                    out = static_cast<T *>(p.out) + t * p.ldo + h * D;
                    if (live && p.lse) p.lse[t * p.H + h] = sums * LN2;
                } else {
                    const int64_t at = it.dst == TO_SLOT ? (int64_t)it.slot * SLOT<KIND> + row : t * p.H + h;
                    part = (it.dst == TO_SLOT ? p.po : p.dpo) + at * D;
                    if (live) (it.dst == TO_SLOT ? p.pl : p.dpl)[at] = sums;
                }
            }
            if (!wait_warp(bar(B_OF + ob), (uint32_t)((item / C::NO) & 1), p.status, E2C_ERR_WAIT_EPI)) break;
            tc_fence_after();
            // 16 columns a step, the next ones on their way: short code, which an item runs through only once
            const uint32_t to = ta + (uint32_t)(C::O_COL + ob * D);
            uint32_t nx[16];
            if (busy) tmem_ld16(to, nx);
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                float o[16];
                if (busy) {
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = __uint_as_float(nx[i]) * inv;
                    if (c + 16 < D) tmem_ld16(to + c + 16, nx);
                }
                if (c + 16 == D) {  // O has been read: the next item may use it while this one is stored
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_OE + ob));
                }
                if (live && !some) {  // such a row may have met a page's NaN: its zeros are not a product
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = none;
                }
                if (live && out) {
                    uint4 *y = reinterpret_cast<uint4 *>(out + c);
                    y[0] = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
                    y[1] = make_uint4(pack2<T>(o[8], o[9]), pack2<T>(o[10], o[11]), pack2<T>(o[12], o[13]), pack2<T>(o[14], o[15]));
                } else if (live) {
                    float4 *y = reinterpret_cast<float4 *>(part + c);
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == C::W_MMA) {
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
    // a part's sums and its log-sum-exp; -infinity: it adds nothing
    E2C_DEV void add(const float *o, const float *sums, int x) {
        const float4 v = *reinterpret_cast<const float4 *>(o + 4 * x);
        const float s = *sums, mn = max2(m, s), ref = mn == -INFINITY ? 0.f : mn;
        const float a = exp2f(m - ref), w = exp2f(s - ref);
        acc.x = acc.x * a + w * v.x;
        acc.y = acc.y * a + w * v.y;
        acc.z = acc.z * a + w * v.z;
        acc.w = acc.w * a + w * v.w;
        l = l * a + w;
        m = mn;
    }
    // sees(): whether the row sees any key, asked only if its parts add up to nothing
    template <typename Sees>
    E2C_DEV void put(const Args &p, int64_t t, int h, int x, Sees sees) {
        const bool bad = no_softmax(m);
        const float inv = bad ? NAN : l > 0.f ? __fdiv_rn(1.0f, l) : sees() ? NAN : 0.f;
        T *y = static_cast<T *>(p.out) + t * p.ldo + (int64_t)h * D + 4 * x;
        uint2 v;
        v.x = pack2<T>(acc.x * inv, acc.y * inv);
        v.y = pack2<T>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2 *>(y) = v;
        if (p.lse && x == 0) p.lse[t * p.H + h] = bad ? m : l > 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
    }
};

// without a prefix: the items that blocks share, one grid row per reporting block
template <typename T, int D, int KIND>
__global__ void __launch_bounds__(JOIN) k_join_split(const Args p, int grid) {
    using J = Join<T, D>;
    griddep_launch_dependents();
    griddep_wait();
    // asked for at once; what a block without a share holds there means nothing
    const int tiles = p.before[p.n], c1 = p.split[2 * blockIdx.x + 1].x;
    const int4 a = p.split[2 * blockIdx.x];
    const int hs = hs_of<KIND>(p), c0 = blockIdx.x / hs, head = blockIdx.x - c0 * hs;
    Share share;
    share.set(1, 0, tiles, grid / hs);
    if (share.begin(c0) == share.begin(c0 + 1) || a.y == 0) return;
    const int x = threadIdx.x % J::LANES, rows = a.y * p.G;
    for (int row = blockIdx.y * J::ROWS + threadIdx.x / J::LANES; row < rows; row += gridDim.y * J::ROWS) {
        J j;
        constexpr int64_t R = SLOT<KIND>;
        j.add(p.po + (a.w * R + row) * D, p.pl + a.w * R + row, x);
#pragma unroll 4
        for (int c = c0; c <= c1; c++) {
            const int64_t at = 2 * (c * hs + head) * R + row;
            j.add(p.po + at * D, p.pl + at, x);
        }
        const int tok = row / p.G;
        j.put(p, a.x + tok, a.z * p.G + (row - tok * p.G), x, [&]() {
            int last;
            const int i = e2c_token_seq(p.q_start, p.n, p.T, a.x + tok, last);
            if (i < 0) return false;
            const Entry e = entry_of(p, i, false);
            return sees_keys<KIND>(p, a.x + tok, e.len - (last - a.x - tok), e.len, e.len - e.nq);
        });
    }
}

// with a prefix: every row's prefix parts and its own
template <typename T, int D, int KIND>
__global__ void __launch_bounds__(JOIN) k_join_prefix(const Args p, int grid) {
    using J = Join<T, D>;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t u = (int64_t)blockIdx.x * J::ROWS + threadIdx.x / J::LANES;
    const int64_t t = u / p.H;
    if (t >= p.T || p.before[p.n] == 0) return;  // no such row; or a batch that is too large, and was left
    const int h = (int)(u - t * p.H), kvh = h / p.G, hd = h - kvh * p.G, x = threadIdx.x % J::LANES;
    const int npt = (p.T + p.tpt - 1) / p.tpt;
    Share share;
    share.set(p.pc.KV * npt, p.before[p.n + 1], p.before[p.n], grid);
    J j;
    auto slot = [&](int k, int row) { j.add(p.po + ((int64_t)k * TR + row) * D, p.pl + (int64_t)k * TR + row, x); };
    if (share.items) {
        const int rt = (int)(t / p.tpt), row = (int)(t - (int64_t)rt * p.tpt) * p.G + hd;
#pragma unroll 4
        for (int s = 0; s < share.splits; s++) slot(2 * grid + (kvh * share.splits + s) * npt + rt, row);
    }
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, (int)t, last);
    if (i < 0) return;
    const Entry e = entry_of(p, i, false);
    if (e.nq == 0) return;
    // an entry has one row tile here
    const int nt = span_of<KIND>(p, e.len, e.nq, 0, p.shared).nt;
    const int s = p.before[i] + kvh * (nt + ITEM_COST), c0 = share.block(s), c1 = share.block(s + nt - 1);
    if (c0 == c1) {
        j.add(p.dpo + (t * p.H + h) * D, p.dpl + t * p.H + h, x);
    } else {
        const int row = (int)(t - e.q0) * p.G + hd;
        for (int c = c0; c <= c1; c++) slot(2 * c + (c == c0 && s > share.begin(c0) ? 1 : 0), row);
    }
    j.put(p, t, h, x, [&]() { return sees_keys<KIND>(p, t, e.len - e.nq + (int)t - e.q0, e.len, e.len - e.nq); });
}

int launch_error(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 0;
    e2c_set_msg("%s launch: %s", what, cudaGetErrorString(e));
    return -2;
}

template <typename T, int D, int KIND>
int run(const Args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    using C = Cfg<D, KIND>;
    static E2cPerDev attr;
    const int dev = e2c_device();
    if (!attr.get(dev)) {
        if (cudaFuncSetAttribute(k_attention_pages<T, D, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D, KIND>()) !=
            cudaSuccess) {
            cudaGetLastError();
            e2c_set_msg("pages_attention: cannot reserve %d bytes of shared memory", smem_bytes<D, KIND>());
            return -2;
        }
        if constexpr (C::CODE) {  // fewer than the roles' shares add up to: the softmax would wait for registers for good
            cudaFuncAttributes has = {};
            if (cudaFuncGetAttributes(&has, k_attention_pages<T, D, KIND>) != cudaSuccess || has.numRegs * C::NTHREADS < C::REGISTERS) {
                cudaGetLastError();
                e2c_set_msg("pages_attention: the kernel for pages of 8 bits was built with %d registers a thread, and needs %d", has.numRegs,
                            C::REGISTERS / C::NTHREADS);
                return -2;
            }
        }
        attr.set(dev, 1);
    }
    const CUtensorMapDataType dt = __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int q_box = a.tpt < a.max_q ? a.tpt : a.max_q, qp_box = a.tpt < a.T ? a.tpt : a.T;
    const uint64_t rows = (uint64_t)a.pc.n_pages * a.pc.page, width = (uint64_t)a.pc.KV * D;
    const uint32_t box = a.pc.page < C::VROWS ? a.pc.page : C::VROWS;
    CUtensorMap tq, tqp, tk, tv;
    if (e2c_tmap_3d(&tq, q, dt, 2, D, a.H, a.T, D * 2, (uint64_t)ldq * 2, 64, a.G, q_box) ||
        (prefix && e2c_tmap_3d(&tqp, q, dt, 2, D, a.H, a.T, D * 2, (uint64_t)ldq * 2, 64, a.G, qp_box)) ||
        (C::CODE ? e2c_tmap_bytes(&tk, a.pc.k, width, rows, C::ROW, box, 1)
                 : e2c_tmap_2d(&tk, a.pc.k, dt, 2, width, rows, width * 2, 64, box)) ||
        (C::CODE ? e2c_tmap_bytes(&tv, a.pc.v, width, rows, C::ROW, box, 1)
                 : e2c_tmap_2d(&tv, a.pc.v, dt, 2, width, rows, width * 2, 64, box)))
        return -3;
    if (!prefix) tqp = tq;
    e2c_launch_as(true, k_attention_pages<T, D, KIND>, dim3(sms), dim3(C::NTHREADS), smem_bytes<D, KIND>(), st, tq, tqp, tk, tv, a, q_box, qp_box);
    if (launch_error("pages_attention")) return -2;
    using J = Join<T, D>;
    if (prefix)
        e2c_launch_as(true, k_join_prefix<T, D, KIND>, dim3((unsigned)(((int64_t)a.T * a.H + J::ROWS - 1) / J::ROWS)), dim3(JOIN), 0, st, a, sms);
    else
        e2c_launch_as(true, k_join_split<T, D, KIND>, dim3(sms, (unsigned)((a.G * (a.max_q < a.tpt ? a.max_q : a.tpt) + J::ROWS - 1) / J::ROWS)), dim3(JOIN), 0, st, a, sms);
    return launch_error("pages_attention join");
}

template <int KIND>
int run_kind(const Args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    const bool bf = a.q_type == E2C_BF16;
    if (a.pc.D == 64)
        return bf ? run<__nv_bfloat16, 64, KIND>(a, q, ldq, prefix, sms, st) : run<__half, 64, KIND>(a, q, ldq, prefix, sms, st);
    if (a.pc.D == 128)
        return bf ? run<__nv_bfloat16, 128, KIND>(a, q, ldq, prefix, sms, st) : run<__half, 128, KIND>(a, q, ldq, prefix, sms, st);
    return bf ? run<__nv_bfloat16, 256, KIND>(a, q, ldq, prefix, sms, st) : run<__half, 256, KIND>(a, q, ldq, prefix, sms, st);
}

}  // namespace
