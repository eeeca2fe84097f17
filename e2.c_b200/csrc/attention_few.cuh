// attention_few.cuh — attention over pages for entries of few rows (at most 16: a token or a few, by the query heads of a key
// head), the form of single tokens.
//
// Such a call is bound by reading the cache, and a product of 128 rows would be nearly empty: the tiles' way through
// shared memory, tensor memory and back takes longer than their reading does (pages of 8 bits, 64 sequences of 5470 to 8192 tokens,
// 32 heads of 128 over 8: 488 us). Here keys are the products' M side and the rows their N side (mma.sync m16n8k16), so that 8
// rows waste nothing; a warp takes 16 keys at a time, with a running maximum and sums of its own:
//   S' = K Q'      16 keys x 8 rows, fp32
//   P' = 2^(S' - m) in 16 bits, transposed in registers (movmatrix) into the second product's operand
//   O' += V' P'    head dim x 8 rows, fp32
// P is rounded to the operands' type, as in the tiles' kernel (the error that it adds is given there), so that a row comes out as
// exact in either. One more warp walks the block's share of items (those of attention_pages.cuh, as are the joins) and loads their keys by TMA, 16 for
// each warp at once, a lane for each page; at an item's end the warps' sums are added up pair by pair, in a fixed order. Head
// dimensions are contracted in the order in which 16-byte loads from shared memory hold them.
//
// Where blocks suffice, the key heads of a share go to neighbouring blocks, which read the heads of a token at the same time: a
// head's 64 to 128 bytes of a token alone make short bursts (64 x 8192 tokens of 8 bits above: 184 us with a block's share going
// through one head after the other). Calls of few and short items (a window, or a short table) take a block an item: no
// plan, and no join.
//
// Codes (8 bits) become fp16, exactly, in registers; scales are factors of a lane's own keys, and m is the largest
// logit_j + log2 vs_j (less 2^8 at most), vs V's scale, so that P_j = 2^(logit_j - m) vs_j has the size that it has without scales;
// a head of zeros, held with the scale 1, counts as one of scale 0. Exponentials are held as those of the tiles are (kSpare).
// Q in bf16 is scaled by a power of two, one for a row, so that fp16 holds it: exact but for values below 2^-28 of the row's
// largest, which lose 2^-39 of that at most.
#pragma once
#include "attention_pages.cuh"

namespace {

// the keys of an item's part: [k0, end1) before the gap, if it has one, and [k2, end2); in tiles of `each`
struct Runs {
    int first, count, k0, k2, end1, end2;  // tiles of the first run, and of both
    E2C_DEV void set(const Args &p, const Item &it, int each) {
        k0 = it.k0;
        end1 = p.sinks;
        k2 = it.k0 + (it.ns > 0 ? it.ns * TK + it.gap : 0);
        end2 = min(it.klim, k2 + (it.nt - it.ns) * TK);
        first = it.ns > 0 ? (end1 - k0 + each - 1) / each : 0;
        count = first + (end2 - k2 + each - 1) / each;
    }
    E2C_DEV int key(int j, int each) const { return j < first ? k0 + each * j : k2 + each * (j - first); }
    E2C_DEV int end(int j) const { return j < first ? end1 : end2; }
};

// an item for the warps that use it
struct __align__(16) FewItem {
    Item it;
    Runs runs;
    int pad[2];
};

template <bool CODE, int D, int NT>
struct Few {
    static constexpr int ROWS = 8 * NT, ROW = CODE ? D : 2 * D;      // bytes of a key
    // 4 to 16 warps an SM that compute, with 100 to 200 KB of stages: what is on its way from memory is what its latency takes
    static constexpr int WARPS = D == 256 && (!CODE || NT == 2) ? 4 : 8, KEYS = 16 * WARPS;
    static constexpr int WIDE = ROW < 128 ? ROW : 128, PANELS = ROW / WIDE, PANEL = KEYS * WIDE;
    static constexpr int UNIT = KEYS * ROW, STAGE = 2 * UNIT;       // K and V of a tile
    static constexpr int CTAS = NT == 1 && STAGE <= 32768 ? 2 : 1;
    static constexpr int MOST = (CTAS == 2 ? 98 : NT == 1 ? 192 : 184) * 1024 / STAGE, NS = MOST > 5 ? 5 : MOST;
    static constexpr int NQ = 2;             // items
    // Adding up: with `a` warps left the last b = min(SLOTS, a / 2) of them give their sums to the b before them. Warp w writes
    // in slot GIVES[w] (four bits each): the one that it read itself in the step before, at first in order.
    static constexpr int SLOTS = WARPS == 8 && CODE && NT == 1 && D >= 128 ? 3 : WARPS / 2, SLOT_BYTES = D * ROWS * 4;
    static constexpr uint32_t GIVES = WARPS == 4 ? 0x1010u : SLOTS == 3 ? 0x21021220u : 0x32103230u;
    static constexpr int SCALES = NS * STAGE;                       // [NS][2][KEYS]
    static constexpr int MERGE = SCALES + (CODE ? NS * 2 * KEYS * 4 : 0);
    static constexpr int ML = MERGE + SLOTS * SLOT_BYTES;           // [SLOTS][ROWS] (m, l)
    static constexpr int SEEN = ML + SLOTS * ROWS * 8;              // [WARPS][ROWS]: lo, hi and se of Seen
    static constexpr int QUEUE = SEEN + WARPS * ROWS * 16;
    static constexpr int BARS = QUEUE + NQ * (int)sizeof(FewItem);
    static constexpr int NBARS = 2 * NS + 2 * NQ + WARPS;
    static constexpr int SCAN = BARS + NBARS * 8;
    static constexpr int BYTES = SCAN + 256;
    static_assert(NS >= 2 && BYTES <= (CTAS == 2 ? 115712 : 232448) && sizeof(PlanScratch<WARPS + 1>) <= 256, "shared memory");
    static_assert(STAGE % 1024 == 0 && ML % 16 == 0 && QUEUE % 16 == 0 && BARS % 8 == 0, "alignment");
    // where 16-byte piece c of key r lies in K or V of a stage: the loads' swizzle
    static E2C_DEV int piece(int r, int c) {
        if constexpr (WIDE == 64) return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
        return (c >> 3) * PANEL + r * 128 + (((c ^ r) & 7) << 4);
    }
};

template <typename T>
E2C_DEV void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
E2C_DEV void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
E2C_DEV void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the transpose of an 8 x 8 matrix of 16-bit values, a row's pair in each lane
E2C_DEV uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
E2C_DEV void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The plan of at most 32 entries by one warp, a lane each, with its walk begun
template <int KIND>
E2C_DEV void plan_of_few(const Args &p, Plan &pl, Walk<KIND> &walk, int lane) {
    Entry e = {};
    if (lane < p.n) e = entry_of(p, lane, blockIdx.x == 0);
    const int etiles = (int)min((int64_t)1 << 30, tiles_of<KIND>(p, e.len, e.nq, 0));
    const int64_t mine = (int64_t)etiles * (p.pc.KV / p.hs);
    int64_t x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    const int64_t all = __shfl_sync(0xffffffffu, x, 31);
    const bool fits = all < 1ll << 30;
    if (!fits && lane == 0) record_status(p.status, E2C_ERR_TOO_LARGE);
    pl.tiles = fits ? (int)all : 0;
    pl.ptiles = 0;
    pl.share.set(1, 0, pl.tiles, gridDim.x / p.hs);
    const int at = pl.share.begin(blockIdx.x / p.hs);
    const uint32_t here = __ballot_sync(0xffffffffu, at >= x - mine && at < x);
    pl.first = here ? __ffs(here) - 1 : p.n;
    pl.first_before = (int)__shfl_sync(0xffffffffu, x - mine, pl.first & 31);
    walk.begin(pl, at, pl.share.begin(blockIdx.x / p.hs + 1));
    walk.base = 0;
    walk.e = e;
    walk.etiles = etiles;
    if (blockIdx.x == 0 && lane == 0) {
        p.before[p.n] = pl.tiles;
        p.before[p.n + 1] = 0;
    }
}

// T: of q and out; X: of the products' operands
template <typename T, bool CODE, int D, int NT>
__global__ void __launch_bounds__(32 * (Few<CODE, D, NT>::WARPS + 1), Few<CODE, D, NT>::CTAS)
    k_attention_few(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Args p,
                    const void *q_rows, const int64_t ldq) {
    using C = Few<CODE, D, NT>;
    using X = std::conditional_t<CODE, __half, T>;
    constexpr int KIND = SIGHT | FEW | (CODE ? CODES : 0), W = C::WARPS;
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    if (smem_u32(smem) & 1023) {
        griddep_wait();
        if (threadIdx.x == 0) record_status(p.status, E2C_ERR_SMEM_ALIGN);
        if (blockIdx.x == 0 && threadIdx.x < 2) p.before[p.n + threadIdx.x] = 0;  // a join has nothing to do
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = smem_u32(smem) + C::BARS;
    auto full = [&](int st) { return bars + 8u * st; };
    auto empty = [&](int st) { return bars + 8u * (C::NS + st); };
    auto item_full = [&](int i) { return bars + 8u * (2 * C::NS + i); };
    auto item_empty = [&](int i) { return bars + 8u * (2 * C::NS + C::NQ + i); };
    // sums that warp w has handed on, w > 0; those of the item before have all been taken
    auto given = [&](int w) { return bars + 8u * (2 * C::NS + 2 * C::NQ + w); };
    const uint32_t taken = bars + 8u * (2 * C::NS + 2 * C::NQ);
    FewItem *queue = reinterpret_cast<FewItem *>(smem + C::QUEUE);
    if (threadIdx.x < C::NBARS) {
        const int b = threadIdx.x;
        mbar_init(bars + 8u * b, (b >= C::NS && b < 2 * C::NS) || (b >= 2 * C::NS + C::NQ && b < 2 * C::NS + 2 * C::NQ) ? W : 1);
        fence_mbar_init();
    }
    if (warp == W && lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    __syncthreads();
    griddep_wait();
    Plan pl;
    const bool whole = p.whole, wide = !whole && p.n > 32;
    if (wide) make_plan<W + 1, KIND>(p, pl, *reinterpret_cast<PlanScratch<W + 1> *>(smem + C::SCAN));

    if (warp == W) {
        // ------------------------------------------------------------ items, and loads of their slices
        Walk<KIND> walk;
        Entry e = {};
        if (wide)
            walk.begin(pl, pl.share.begin(blockIdx.x / p.hs), pl.share.begin(blockIdx.x / p.hs + 1));
        else if (!whole)
            plan_of_few<KIND>(p, pl, walk, lane);
        else
            e = entry_of(p, blockIdx.x / p.pc.KV, blockIdx.x % p.pc.KV == 0 && lane == 0);
        if (!whole && lane == 0 && walk.pos < walk.end) p.split[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        __syncwarp();
        const int PB = min(p.pc.page, C::KEYS), shift = 31 - __clz(p.pc.page);
        Item it = {};
        it.masked = 1;
        int n = 0, g = 0;
        bool ok = true;
#pragma unroll 1
        for (;; n++) {
            bool more;
            if (whole) {
                more = n == 0 && e.nq > 0;
                it.seq = e.len > 0 ? e.seq : -1;
                it.len = e.len;
                it.base = it.pos0 = e.len - e.nq;
                it.kvh = blockIdx.x % p.pc.KV;
                it.t0 = e.q0;
                it.ntok = e.nq;
                const Span sp = span_of<KIND>(p, e.len, e.nq, 0, 0);
                sp.cut(p, 0, sp.nt, it);
                it.dst = TO_OUT;
            } else {
                more = walk.next(p, pl, it, lane);
            }
            FewItem &to = queue[n % C::NQ];
            if (!(ok = wait_warp(item_empty(n % C::NQ), (uint32_t)((n / C::NQ & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER))) break;
            if (!more) {
                if (lane == 0) {
                    to.it.ntok = -1;
                    mbar_arrive(item_full(n % C::NQ));
                }
                break;
            }
            Runs runs;
            runs.set(p, it, C::KEYS);
            // a lane's page of tile j, looked at when it is used
            auto page_of = [&](int j) -> int {
                const int key = runs.key(j, C::KEYS) + lane * PB;
                return j < runs.count && lane * PB < C::KEYS && it.seq >= 0 && key < runs.end(j)
                           ? p.pc.table[(int64_t)it.seq * p.pc.max_blocks + (key >> shift)] : 0;
            };
            int page = page_of(0);
            if (lane == 0) {
                to.it = it;
                to.runs = runs;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(item_full(n % C::NQ));
#pragma unroll 1
            for (int j = 0; j < runs.count; j++, g++) {
                const int st = g % C::NS, key = runs.key(j, C::KEYS), nb = min(C::KEYS, runs.end(j) - key + PB - 1) / PB;
                const int next = page_of(j + 1);
                if ((unsigned)page >= (unsigned)p.pc.n_pages) {  // page 0 instead, reported
                    record_status(p.status, E2C_ERR_BAD_SEQ);
                    page = 0;
                }
                if (!(ok = wait_warp(empty(st), (uint32_t)((g / C::NS & 1) ^ 1), p.status, E2C_ERR_WAIT_PRODUCER))) break;
                if (lane == 0) mbar_arrive_expect_tx(full(st), (uint32_t)(nb * PB * (2 * C::ROW + (CODE ? 8 : 0))));
                __syncwarp();
                if (lane < nb) {
                    const int slot = (key + lane * PB) & (p.pc.page - 1), y = (page << shift) + slot;
                    const uint32_t k = smem_u32(smem) + st * C::STAGE + lane * PB * C::WIDE;
#pragma unroll
                    for (int i = 0; i < C::PANELS; i++) {
                        const int x = it.kvh * D + i * (CODE ? 128 : 64);
                        tma_load_2d(k + i * C::PANEL, &tmK, x, y, full(st));
                        tma_load_2d(k + C::UNIT + i * C::PANEL, &tmV, x, y, full(st));
                    }
                    if constexpr (CODE) {
                        const int64_t at = ((int64_t)page * p.pc.KV + it.kvh) * p.pc.page + slot;
                        const uint32_t sc = smem_u32(smem) + C::SCALES + st * (2 * C::KEYS * 4) + lane * PB * 4;
                        bulk_load(sc, p.pc.ks + at, (uint32_t)PB * 4, full(st));
                        bulk_load(sc + C::KEYS * 4, p.pc.vs + at, (uint32_t)PB * 4, full(st));
                    }
                }
                __syncwarp();
                page = next;
            }
            if (!ok) break;
        }
        // every load that was issued has landed before the block may end
        for (int i = max(0, g - C::NS); i < g; i++)
            wait_warp(full(i % C::NS), (uint32_t)(i / C::NS & 1), nullptr, E2C_ERR_WAIT_DRAIN);
        return;
    }

    // ---------------------------------------------------------------- products
    const int quad = lane & 3, oct = lane >> 2;
    float2 *ml = reinterpret_cast<float2 *>(smem + C::ML);
    uint32_t qf[D / 16][NT][2];
    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2], less[NT][2];  // less: -m (CODE: + kSpare), or 0 for a row that has only seen -infinity
    int4 *seen = reinterpret_cast<int4 *>(smem + C::SEEN) + warp * C::ROWS;
    int all_lo = 0, all_hi = 0;             // keys that every row sees
    constexpr bool TURNED = CODE && !std::is_same<T, __half>::value;  // Q becomes fp16 too, times a power of two for each row
    const float c = p.neg ? -p.c : p.c;
    float up[NT][2];                        // TURNED: back from that
    auto begin = [&](const Item &it) {
        const int rows = it.ntok * p.G;
        // Q: a lane's 16 (8 bits) or 8 neighbouring dimensions of each 64 or 32, of row `oct`
        constexpr int PER = CODE ? 16 : 8;
        uint4 w[NT][D / 32];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = nt * 8 + oct, tok = row / p.G, hd = row - tok * p.G;
            const T *q = static_cast<const T *>(q_rows) + (int64_t)(it.t0 + tok) * ldq + (it.kvh * p.G + hd) * D;
#pragma unroll
            for (int j = 0; j < D / (4 * PER); j++)
#pragma unroll
                for (int k = 0; k < PER / 8; k++)
                    w[nt][j * (PER / 8) + k] = row < rows ? *reinterpret_cast<const uint4 *>(q + j * 4 * PER + quad * PER + k * 8) : make_uint4(0, 0, 0, 0);
        }
        if constexpr (TURNED) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint32_t top = 0;  // the row's largest finite magnitude
#pragma unroll
                for (int k = 0; k < D / 8; k++) {
                    const uint32_t b = reinterpret_cast<const uint32_t *>(w[nt])[k], b0 = b << 16 & 0x7fffffffu, b1 = b & 0x7fff0000u;
                    top = max(top, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t ex = max(top >> 23, 15u);  // its exponent becomes 14
                const float scale = __uint_as_float((268u - ex) << 23);
#pragma unroll
                for (int i = 0; i < 2; i++) up[nt][i] = __uint_as_float((__shfl_sync(0xffffffffu, ex, 4 * (2 * quad + i)) - 14u) << 23);
#pragma unroll
                for (int k = 0; k < D / 8; k++) {
                    const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 *>(w[nt])[k]);
                    reinterpret_cast<uint32_t *>(w[nt])[k] = pack2<__half>(f.x * scale, f.y * scale);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                qf[k][nt][0] = reinterpret_cast<const uint32_t *>(w[nt])[2 * k];
                qf[k][nt][1] = reinterpret_cast<const uint32_t *>(w[nt])[2 * k + 1];
            }
        int lo = 0, hi = it.klim;
        if (lane < rows) {
            const int tok = lane / p.G;
            Seen x;
            x.set(p, it.t0 + tok, it.pos0 + tok, it.len, it.base);
            seen[lane] = make_int4(x.lo, x.hi, x.se, 0);
            lo = x.lo;
            hi = x.hi;
        }
        all_lo = __reduce_max_sync(0xffffffffu, lo);
        all_hi = __reduce_min_sync(0xffffffffu, hi);
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[nt][i] = -INFINITY;
                less[nt][i] = 0.f;
                l[nt][i] = 0.f;
            }
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[i][nt][k] = 0.f;
    };

    // keys [kk, kk + 16) before `end`, of which stage st holds K and V from its row r0 on
    auto use = [&](const Item &it, int st, int r0, int kk, int end) {
        const uint8_t *k = smem + st * C::STAGE + r0 * C::WIDE, *v = k + C::UNIT;
        float s[NT][4] = {}, s2[NT][4] = {};  // two sums, so that products need not wait for one another
        if constexpr (CODE) {
#pragma unroll
            for (int j = 0; j < D / 64; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(k + C::piece(oct, 4 * j + quad));
                const uint4 y = *reinterpret_cast<const uint4 *>(k + C::piece(oct + 8, 4 * j + quad));
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint2 a = from_codes<__half>((&x.x)[t]), b = from_codes<__half>((&y.x)[t]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma_16816<X>(t & 1 ? s2[nt] : s[nt], a.x, b.x, a.y, b.y, qf[4 * j + t][nt][0], qf[4 * j + t][nt][1]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(k + C::piece(oct, 4 * j + quad));
                const uint4 y = *reinterpret_cast<const uint4 *>(k + C::piece(oct + 8, 4 * j + quad));
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        mma_16816<X>(t & 1 ? s2[nt] : s[nt], (&x.x)[2 * t], (&y.x)[2 * t], (&x.x)[2 * t + 1], (&y.x)[2 * t + 1], qf[2 * j + t][nt][0], qf[2 * j + t][nt][1]);
            }
        }
        // s[nt][2 h + i]: key oct + 8 h, row 8 nt + 2 quad + i
        float lv[2] = {0.f, 0.f}, vs[2] = {1.f, 1.f}, kc[2] = {c, c};
        if constexpr (CODE) {
            const float *sc = reinterpret_cast<const float *>(smem + C::SCALES) + st * (2 * C::KEYS) + r0 + oct;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                kc[h] = sc[8 * h] * c;
                lv[h] = scale_log2(sc[C::KEYS + 8 * h]);
                vs[h] = scale_factor(sc[C::KEYS + 8 * h]);
            }
            constexpr float ONE = 0x1p-16f;  // scale_factor(1)
            if (__any_sync(0xffffffffu, vs[0] == ONE || vs[1] == ONE)) {  // heads of zeros, if their codes are that
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < D / 64; i++) {  // the quad has a key's 16-byte pieces in turn
                        const uint4 w = *reinterpret_cast<const uint4 *>(v + C::piece(oct + 8 * h, 4 * i + quad));
                        any |= w.x | w.y | w.z | w.w;
                    }
                    any |= __shfl_xor_sync(0xffffffffu, any, 1);
                    any |= __shfl_xor_sync(0xffffffffu, any, 2);
                    if (vs[h] == ONE && any == 0) {
                        lv[h] = kLeastLog2;
                        vs[h] = 0.f;
                    }
                }
            }
        }
        // the logits, and, as y, with the log2 of their weights' scale
        float y[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[nt][e] = (s[nt][e] + s2[nt][e]) * (TURNED ? kc[e >> 1] * up[nt][e & 1] : kc[e >> 1]);
                y[nt][e] = CODE ? s[nt][e] + lv[e >> 1] : s[nt][e];
            }
        if (kk < all_lo || kk + 16 > min(end, all_hi)) {  // some row does not see some of them
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int row = 8 * nt + 2 * quad + i;
                    uint32_t bits = Seen::below(end - kk);
                    if (row < it.ntok * p.G) {
                        const int4 x = seen[row];
                        const Seen sight = {x.x, x.y, x.z, it.base, it.len, p.tree ? p.tree + (int64_t)(it.t0 + row / p.G) * p.words : nullptr};
                        bits &= sight.keys(p, kk);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (!(bits >> (oct + 8 * h) & 1)) s[nt][2 * h + i] = y[nt][2 * h + i] = -INFINITY;
                }
            if (end - kk < 16) {  // past the last key a stage holds anything
                if constexpr (CODE) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (oct + 8 * h >= end - kk) vs[h] = 0.f;
                } else {
                    uint8_t *y = const_cast<uint8_t *>(v);
                    for (int e = lane; e < (16 - (end - kk)) * (C::ROW / 16); e += 32) {
                        const int r = end - kk + e / (C::ROW / 16);
                        *reinterpret_cast<uint4 *>(y + C::piece(r, e % (C::ROW / 16))) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
            }
        }
        // m is the rows' own in all lanes, and moves when some lane's logit is more than 2^8 above it (so also from
        // -infinity, and for a NaN)
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) over |= !(max2(y[nt][i], y[nt][2 + i]) <= m[nt][i] + kRescaleLog2);
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float x = max2(y[nt][i], y[nt][2 + i]);
                    x = max2(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = max2(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = max2(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    if (x <= m[nt][i] + kRescaleLog2) continue;
                    const float now = max2(m[nt][i], x), alpha = ex2_approx(m[nt][i] - now);
                    l[nt][i] = CODE ? times_exp2(l[nt][i], m[nt][i] - now) : l[nt][i] * alpha;
                    m[nt][i] = now;
                    less[nt][i] = now == -INFINITY ? 0.f : CODE ? kSpare - now : -now;
#pragma unroll
                    for (int d = 0; d < D / 16; d++) o[d][nt][i] *= alpha, o[d][nt][2 + i] *= alpha;
                }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float x = ex2_approx(s[nt][2 * h + i] + less[nt][i]);
                    l[nt][i] = CODE ? fmaf(x, 0x1p-16f, l[nt][i]) : l[nt][i] + x;
                    s[nt][2 * h + i] = CODE ? x * vs[h] : x;
                }
            }
            pb[nt][0] = transpose8(pack2<X>(s[nt][0], s[nt][1]));
            pb[nt][1] = transpose8(pack2<X>(s[nt][2], s[nt][3]));
        }
        if constexpr (CODE) {
            // a lane's D / 8 dimensions of keys 2 quad, 2 quad + 1 and the same + 8
            constexpr int WORDS = D == 64 ? 2 : 4;
#pragma unroll
            for (int part = 0; part < D / (32 * WORDS); part++) {
                uint32_t w[4][WORDS];
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const int r = 2 * quad + (a & 1) + 8 * (a >> 1);
                    if constexpr (D == 64) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(v + C::piece(r, oct >> 1) + (oct & 1) * 8);
                        w[a][0] = x.x, w[a][1] = x.y;
                    } else {
                        const uint4 x = *reinterpret_cast<const uint4 *>(v + C::piece(r, oct * (D / 128) + part));
                        w[a][0] = x.x, w[a][1] = x.y, w[a][2] = x.z, w[a][3] = x.w;
                    }
                }
#pragma unroll
                for (int d = 0; d < WORDS; d++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {  // two dimensions of a word: rows oct and oct + 8 of a tile
                        const int pick = t ? 0x7362 : 0x5140, tile = 2 * (part * WORDS + d) + t;
                        const uint2 a = from_codes<__half>(__byte_perm(w[0][d], w[1][d], pick)), b = from_codes<__half>(__byte_perm(w[2][d], w[3][d], pick));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_16816<X>(o[tile][nt], a.x, a.y, b.x, b.y, pb[nt][0], pb[nt][1]);
                    }
            }
        } else {
            const int r = (lane >> 4) * 8 + (lane & 7), c = lane >> 3 & 1;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                uint32_t a[4];
                ldmatrix_trans(a, smem_u32(v) + C::piece(r, 2 * i + c));
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma_16816<X>(o[i][nt], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
            }
        }
    };

    // the n-th item's sums from all warps; false if a wait ran out
    auto finish = [&](const Item &it, int n) -> bool {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                l[nt][i] = x;
            }
        // (a loop, not its steps one after the other: this code runs once an item, and the small calls wait for
        // instructions a seventh of their time as it is)
        auto slot = [&](int w) { return reinterpret_cast<float4 *>(smem + C::MERGE + (C::GIVES >> 4 * w & 15) * C::SLOT_BYTES) + lane; };
        auto slot_rows = [&](int w) { return ml + (C::GIVES >> 4 * w & 15) * C::ROWS + 2 * quad; };
#pragma unroll 1
        for (int a = W, b; a > 1; a -= b) {
            b = min(C::SLOTS, a >> 1);
            if (warp >= a - b) break;
            if (warp < a - 2 * b) continue;
            const int w = warp + b;
            if (!wait_warp(given(w), (uint32_t)(n & 1), p.status, E2C_ERR_WAIT_ATTN)) return false;
            const float4 *sums = slot(w);
            const float2 *rows = slot_rows(w);
            float f[NT][2], g[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float2 x = rows[8 * nt + i];
                    const float top = max2(m[nt][i], x.x), ref = top == -INFINITY ? 0.f : top;
                    f[nt][i] = ex2_approx(m[nt][i] - ref);
                    g[nt][i] = ex2_approx(x.x - ref);
                    l[nt][i] = CODE ? times_exp2(l[nt][i], m[nt][i] - ref) + times_exp2(x.y, x.x - ref) : l[nt][i] * f[nt][i] + x.y * g[nt][i];
                    m[nt][i] = top;
                }
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float4 x = sums[(i * NT + nt) * 32];
                    o[i][nt][0] = o[i][nt][0] * f[nt][0] + x.x * g[nt][0];
                    o[i][nt][1] = o[i][nt][1] * f[nt][1] + x.y * g[nt][1];
                    o[i][nt][2] = o[i][nt][2] * f[nt][0] + x.z * g[nt][0];
                    o[i][nt][3] = o[i][nt][3] * f[nt][1] + x.w * g[nt][1];
                }
            __syncwarp();
        }
        if (warp > 0) {
            // slots are free once the first warp has the sums of the item before
            if (warp >= W - C::SLOTS && !wait_warp(taken, (uint32_t)(n & 1) ^ 1, p.status, E2C_ERR_WAIT_ATTN)) return false;
            float4 *sums = slot(warp);
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) sums[(i * NT + nt) * 32] = make_float4(o[i][nt][0], o[i][nt][1], o[i][nt][2], o[i][nt][3]);
            if (oct == 0)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 2; i++) slot_rows(warp)[8 * nt + i] = make_float2(m[nt][i], l[nt][i]);
            __syncwarp();
            if (lane == 0) mbar_arrive(given(warp));
            return true;
        }
        if (lane == 0) mbar_arrive(taken);
        const int rows = it.ntok * p.G;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = 8 * nt + 2 * quad + i, tok = row / p.G, hd = row - tok * p.G;
                const int64_t t = it.t0 + tok, h = it.kvh * p.G + hd;
                if (row >= rows) continue;
                // l = 0: every logit was -infinity, or no key was seen; a part leaves that to the join
                const bool bad = no_softmax(m[nt][i]), some = bad || l[nt][i] > 0.f, part = it.dst != TO_OUT;
                const float sums = bad ? m[nt][i] : some ? m[nt][i] + __log2f(l[nt][i]) : -INFINITY;
                const float inv = bad ? NAN : __fdividef(1.f, l[nt][i]);
                if (oct == 0) {
                    if (part)
                        p.pl[(int64_t)it.slot * SLOT<KIND> + row] = sums;
                    else if (p.lse)
                        p.lse[t * p.H + h] = sums * LN2;
                }
                float none = 0.f;
                if (!some && !part && sees_keys<KIND>(p, t, it.pos0 + tok, it.len, it.base)) none = NAN;
                float y[D / 8];
#pragma unroll
                for (int k = 0; k < D / 16; k++) {  // (a row without sums may have met a page's NaN)
                    y[2 * k] = some ? o[k][nt][i] * inv : none;
                    y[2 * k + 1] = some ? o[k][nt][2 + i] * inv : none;
                }
                // codes: a lane's neighbouring dimensions; otherwise every eighth
                const int64_t at = CODE ? oct * (D / 8) : oct;
                if (part) {
                    float *to = p.po + ((int64_t)it.slot * SLOT<KIND> + row) * D + at;
#pragma unroll
                    for (int k = 0; k < D / 8; k += CODE ? 4 : 1) {
                        if constexpr (CODE)
                            *reinterpret_cast<float4 *>(to + k) = make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
                        else
                            to[8 * k] = y[k];
                    }
                } else {
                    T *to = static_cast<T *>(p.out) + t * p.ldo + h * D + at;
#pragma unroll
                    for (int k = 0; k < D / 8; k += CODE ? 8 : 1) {
                        if constexpr (CODE)
                            *reinterpret_cast<uint4 *>(to + k) = make_uint4(pack2<T>(y[k], y[k + 1]), pack2<T>(y[k + 2], y[k + 3]), pack2<T>(y[k + 4], y[k + 5]), pack2<T>(y[k + 6], y[k + 7]));
                        else
                            reinterpret_cast<uint16_t *>(to)[8 * k] = (uint16_t)pack2<T>(y[k], 0.f);
                    }
                }
            }
        return true;
    };

    int st = 0, slice = warp;  // stage, and the warp's keys in it: tiles that are not full fall to other warps each time
    uint32_t parity = 0;
#pragma unroll 1
    for (int n = 0;; n++) {
        if (!wait_warp(item_full(n % C::NQ), (uint32_t)(n / C::NQ & 1), p.status, E2C_ERR_WAIT_ATTN)) return;
        const FewItem &fi = queue[n % C::NQ];
        if (fi.it.ntok < 0) return;
        begin(fi.it);
        const Runs runs = fi.runs;
        int key = runs.key(0, C::KEYS), end = runs.end(0);
#pragma unroll 1
        for (int j = 1; j <= runs.count; j++) {
            // (also without keys of its own: a warp that ran ahead would count twice in the stage's barrier)
            if (!wait_warp(full(st), parity, p.status, E2C_ERR_WAIT_ATTN)) return;
            const int kk = key + 16 * slice;
            if (kk < end) use(fi.it, st, 16 * slice, kk, end);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(st));
            if (++st == C::NS) {
                st = 0;
                parity ^= 1;
            }
            slice = (slice + 1) % W;
            key += C::KEYS;
            if (j == runs.first) {
                key = runs.k2;
                end = runs.end2;
            }
        }
        if (!finish(fi.it, n)) return;
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty(n % C::NQ));
    }
}

// Calls with an item a block at most, and so few keys an item that reading them takes one block no longer than the plan and the join of
// divided items take. One token an entry, us whole and divided: 4 sequences of 300, 500, 700 and 1000 tokens (256 bytes of a key
// and value; 77, 128, 179 and 256 KB), 8-bit heads of 128 over 4, in a graph 9.8, 12.0, 14.5 and 18.2, divided 12.0, 12.9, 12.9 and 13.9, and
// through Python, which saves a launch, 14.7, -, 14.9 and 18.7, divided 16.7; 30 sequences of 500 and 1000 in a graph 13.5 and 20.7, divided 15.1 and
// 19.3; 3 sequences, 16-bit heads of 256 over 2, windows of 100, 200 and 400 (1 KB a key) 7.9, 10.2 and 14.2, divided 10.9, 11.4 and 11.7. So it turns at 140 KB
// (few items, in a graph) to 250 KB (many, or without one).
constexpr int WHOLE_BYTES = 192 << 10;
template <typename T, bool CODE, int D, int NT>
int run_few(Args a, const void *q, int64_t ldq, int sms, cudaStream_t st) {
    using C = Few<CODE, D, NT>;
    constexpr int KIND = SIGHT | FEW | (CODE ? CODES : 0);
    static E2cPerDev attr;
    const int dev = e2c_device(), KV = a.pc.KV;
    if (!attr.get(dev)) {
        if (cudaFuncSetAttribute(k_attention_few<T, CODE, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES) != cudaSuccess) {
            cudaGetLastError();
            e2c_set_msg("pages_attention: cannot reserve %d bytes of shared memory", C::BYTES);
            return -2;
        }
        attr.set(dev, 1);
    }
    // a bound on an item's keys, whose lengths are on the device: the table's (a short text in a wide table counts as a long one), or
    // those of a window before its rows, and behind them where they see that side, and the sinks
    int64_t keys = (int64_t)a.pc.max_blocks * a.pc.page;
    if (a.window >= 0) {
        const int64_t seen = (a.causal || a.tree ? 1 : 2) * (int64_t)a.window + 1 + a.max_q + a.sinks + 2 * a.align;
        keys = keys < seen ? keys : seen;
    }
    int grid = sms * C::CTAS;
    a.whole = (int64_t)a.n * KV <= grid && keys * 2 * C::ROW <= WHOLE_BYTES;
    // a head for each of KV neighbouring blocks, if that leaves no more than one in twenty without work
    a.hs = !a.whole && grid / KV * KV * 20 >= grid * 19 ? KV : 1;
    grid = a.whole ? a.n * KV : grid / a.hs * a.hs;
    const CUtensorMapDataType dt = __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint64_t rows = (uint64_t)a.pc.n_pages * a.pc.page, width = (uint64_t)KV * D;
    const uint32_t box = a.pc.page < C::KEYS ? a.pc.page : C::KEYS;
    CUtensorMap tk, tv;
    if (CODE ? e2c_tmap_bytes(&tk, a.pc.k, width, rows, C::WIDE, box, 1) || e2c_tmap_bytes(&tv, a.pc.v, width, rows, C::WIDE, box, 1)
             : e2c_tmap_2d(&tk, a.pc.k, dt, 2, width, rows, width * 2, 64, box) || e2c_tmap_2d(&tv, a.pc.v, dt, 2, width, rows, width * 2, 64, box))
        return -3;
    e2c_launch_as(true, k_attention_few<T, CODE, D, NT>, dim3(grid), dim3(32 * (C::WARPS + 1)), C::BYTES, st, tk, tv, a, q, ldq);
    if (launch_error("pages_attention")) return -2;
    if (a.whole) return 0;
    using J = Join<T, D>;
    e2c_launch_as(true, k_join_split<T, D, KIND>, dim3(grid, (unsigned)((a.G * a.max_q + J::ROWS - 1) / J::ROWS)), dim3(JOIN), 0, st, a, grid);
    return launch_error("pages_attention join");
}
template <typename T, bool CODE>
int few_of(const Args &a, const void *q, int64_t ldq, int sms, cudaStream_t st) {
    const bool one = a.G * a.max_q <= 8;
    if (a.pc.D == 64) return one ? run_few<T, CODE, 64, 1>(a, q, ldq, sms, st) : run_few<T, CODE, 64, 2>(a, q, ldq, sms, st);
    if (a.pc.D == 128) return one ? run_few<T, CODE, 128, 1>(a, q, ldq, sms, st) : run_few<T, CODE, 128, 2>(a, q, ldq, sms, st);
    return one ? run_few<T, CODE, 256, 1>(a, q, ldq, sms, st) : run_few<T, CODE, 256, 2>(a, q, ldq, sms, st);
}

}  // namespace
