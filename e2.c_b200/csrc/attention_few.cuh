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
// One more warp walks the block's share of items (those of attention_pages.cuh, as are the joins) and loads their keys by TMA, 16 for
// each warp at once, a lane for each page; at an item's end the warps' sums are added up in a fixed order. Head dimensions are
// contracted, and put out, in the order in which 16-byte loads from shared memory hold them.
//
// Codes (8 bits) become fp16, exactly, in registers; scales are factors of a lane's own keys, applied as in attention_pages.cuh.
// Q in bf16 is scaled by a power of two for each row, so that fp16 holds it: exact but for values below 2^-28 of the row's
// largest.
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
template <int ROWS>
struct __align__(16) FewItem {
    Item it;
    Runs runs;
    int all_lo, all_hi;  // keys that every row sees
    int pad[2];
    Seen seen[ROWS];
};

template <bool CODE, int D, int NT>
struct Few {
    static constexpr int ROWS = 8 * NT, ROW = CODE ? D : 2 * D;      // bytes of a key
    // 4 to 16 warps an SM that compute, with 100 to 200 KB of stages: what is on its way from memory is what its latency takes
    static constexpr int WARPS = D == 256 && (!CODE || NT == 2) ? 4 : 8, KEYS = 16 * WARPS;
    static constexpr int WIDE = ROW < 128 ? ROW : 128, PANELS = ROW / WIDE, PANEL = KEYS * WIDE;
    static constexpr int UNIT = KEYS * ROW, STAGE = 2 * UNIT;       // K and V of a tile
    static constexpr int CTAS = NT == 1 && STAGE <= 32768 ? 2 : 1;
    static constexpr int MOST = (CTAS == 2 ? 100 : 192) * 1024 / STAGE, NS = MOST > 5 ? 5 : MOST;
    static constexpr int NQ = 4;             // items
    static constexpr int MT = CTAS == 2 || NT == 2 ? 2 : 4;  // tiles of 16 head dimensions added up at once
    static constexpr int SCALES = NS * STAGE;                       // [NS][2][KEYS]
    static constexpr int MERGE = SCALES + (CODE ? NS * 2 * KEYS * 4 : 0);
    static constexpr int ML = MERGE + WARPS * MT * 16 * ROWS * 4;   // [WARPS][ROWS] (m, l)
    static constexpr int INV = ML + WARPS * ROWS * 8;               // [ROWS] (1 / l, what a row without sums gets)
    static constexpr int QUEUE = INV + ROWS * 8;
    static constexpr int BARS = QUEUE + NQ * (int)sizeof(FewItem<ROWS>);
    static constexpr int NBARS = 2 * NS + 2 * NQ + 1;
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
    const int64_t mine = (int64_t)etiles * p.pc.KV;
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
    pl.share.set(1, 0, pl.tiles, gridDim.x);
    const int at = pl.share.begin(blockIdx.x);
    const uint32_t here = __ballot_sync(0xffffffffu, at >= x - mine && at < x);
    pl.first = here ? __ffs(here) - 1 : p.n;
    pl.first_before = (int)__shfl_sync(0xffffffffu, x - mine, pl.first & 31);
    walk.begin(pl, at, pl.share.begin(blockIdx.x + 1));
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
        if (blockIdx.x == 0 && threadIdx.x < 2) p.before[p.n + threadIdx.x] = 0;  // the join has nothing to do
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = smem_u32(smem) + C::BARS;
    auto full = [&](int st) { return bars + 8u * st; };
    auto empty = [&](int st) { return bars + 8u * (C::NS + st); };
    auto item_full = [&](int i) { return bars + 8u * (2 * C::NS + i); };
    auto item_empty = [&](int i) { return bars + 8u * (2 * C::NS + C::NQ + i); };
    const uint32_t merged = bars + 8u * (2 * C::NS + 2 * C::NQ);
    FewItem<C::ROWS> *queue = reinterpret_cast<FewItem<C::ROWS> *>(smem + C::QUEUE);
    if (threadIdx.x < C::NBARS) {
        const int b = threadIdx.x;
        mbar_init(bars + 8u * b, b < C::NS || (b >= 2 * C::NS && b < 2 * C::NS + C::NQ) ? 1 : W);
        fence_mbar_init();
    }
    if (warp == W && lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    __syncthreads();
    griddep_wait();
    Plan pl;
    if (p.n > 32) make_plan<W + 1, KIND>(p, pl, *reinterpret_cast<PlanScratch<W + 1> *>(smem + C::SCAN));

    if (warp == W) {
        // ------------------------------------------------------------ items, and loads of their slices
        Walk<KIND> walk;
        if (p.n > 32)
            walk.begin(pl, pl.share.begin(blockIdx.x), pl.share.begin(blockIdx.x + 1));
        else
            plan_of_few<KIND>(p, pl, walk, lane);
        if (lane == 0 && walk.pos < walk.end) p.split[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        __syncwarp();
        const int PB = min(p.pc.page, C::KEYS), shift = 31 - __clz(p.pc.page);
        Item it = {};
        it.masked = 1;
        int n = 0, g = 0;
        bool ok = true;
#pragma unroll 1
        for (;; n++) {
            const bool more = walk.next(p, pl, it, lane);
            FewItem<C::ROWS> &to = queue[n % C::NQ];
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
            int lo = 0, hi = it.klim;
            if (lane < it.ntok * p.G) {
                const int tok = lane / p.G;
                Seen x;
                x.set(p, it.t0 + tok, it.pos0 + tok, it.len, it.base);
                to.seen[lane] = x;
                lo = x.lo;
                hi = x.hi;
            }
            lo = __reduce_max_sync(0xffffffffu, lo);
            hi = __reduce_min_sync(0xffffffffu, hi);
            if (lane == 0) {
                to.it = it;
                to.runs = runs;
                to.all_lo = lo;
                to.all_hi = hi;
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
    float2 *ml = reinterpret_cast<float2 *>(smem + C::ML), *fin = reinterpret_cast<float2 *>(smem + C::INV);
    float *merge = reinterpret_cast<float *>(smem + C::MERGE);
    uint32_t qf[D / 16][NT][2];
    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2], cr[NT][2];
    uint32_t turn = 0;
    auto together = [&]() -> bool {  // the block's other warps have come here too
        __syncwarp();
        if (lane == 0) mbar_arrive(merged);
        const bool ok = wait_warp(merged, turn, p.status, E2C_ERR_WAIT_ATTN);
        turn ^= 1;
        return ok;
    };

    auto begin = [&](const Item &it) {
        const int rows = it.ntok * p.G;
        // Q: a lane's 16 (8 bits) or 8 neighbouring dimensions of each 64 or 32, of row `oct`
        float up[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = nt * 8 + oct, tok = row / p.G, hd = row - tok * p.G;
            const T *q = static_cast<const T *>(q_rows) + (int64_t)(it.t0 + tok) * ldq + (it.kvh * p.G + hd) * D;
            constexpr int PER = CODE ? 16 : 8;
            uint4 w[D / 32];
#pragma unroll
            for (int j = 0; j < D / (4 * PER); j++)
#pragma unroll
                for (int k = 0; k < PER / 8; k++)
                    w[j * (PER / 8) + k] = row < rows ? *reinterpret_cast<const uint4 *>(q + j * 4 * PER + quad * PER + k * 8) : make_uint4(0, 0, 0, 0);
            up[nt] = 1.f;
            if constexpr (CODE && !std::is_same<T, __half>::value) {
                const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162 *>(w);
                uint32_t top = 0;  // the largest finite magnitude
#pragma unroll
                for (int k = 0; k < D / 8; k++) {
                    const uint32_t b = reinterpret_cast<const uint32_t *>(w)[k], b0 = b << 16 & 0x7fffffffu, b1 = b & 0x7fff0000u;
                    top = max(top, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t ex = max(top >> 23, 15u);  // its exponent becomes 14
                const float scale = __uint_as_float((268u - ex) << 23);
                up[nt] = __uint_as_float((ex - 14u) << 23);
#pragma unroll
                for (int k = 0; k < D / 8; k++) {
                    const float2 f = __bfloat1622float2(x[k]);
                    reinterpret_cast<uint32_t *>(w)[k] = pack2<__half>(f.x * scale, f.y * scale);
                }
            }
            const uint32_t *b = reinterpret_cast<const uint32_t *>(w);
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                qf[k][nt][0] = b[2 * k];
                qf[k][nt][1] = b[2 * k + 1];
            }
        }
        const float c = p.neg ? -p.c : p.c;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                cr[nt][i] = c * __shfl_sync(0xffffffffu, up[nt], (2 * quad + i) * 4);
                m[nt][i] = -INFINITY;
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
    auto use = [&](const FewItem<C::ROWS> &fi, int st, int r0, int kk, int end) {
        const uint8_t *k = smem + st * C::STAGE + r0 * C::WIDE, *v = k + C::UNIT;
        float s[NT][4] = {}, s2[NT][4] = {};  // two sums, so that products need not wait for one another
        if constexpr (CODE) {
#pragma unroll
            for (int j = 0; j < D / 64; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(k + C::piece(oct, 4 * j + quad));
                const uint4 y = *reinterpret_cast<const uint4 *>(k + C::piece(oct + 8, 4 * j + quad));
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint2 a = from_codes<X>((&x.x)[t]), b = from_codes<X>((&y.x)[t]);
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
        float lv[2] = {0.f, 0.f}, vs[2] = {1.f, 1.f}, ks[2] = {1.f, 1.f};
        if constexpr (CODE) {
            const float *sc = reinterpret_cast<const float *>(smem + C::SCALES) + st * (2 * C::KEYS) + r0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                ks[h] = sc[oct + 8 * h];
                const float x = sc[C::KEYS + oct + 8 * h];
                const bool fine = fabsf(x) < INFINITY;
                lv[h] = fine ? fminf(fmaxf(__log2f(fabsf(x)), -100.f), 100.f) : 0.f;
                vs[h] = fine ? x : NAN;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[nt][e] = (s[nt][e] + s2[nt][e]) * (CODE ? ks[e >> 1] * cr[nt][e & 1] : cr[nt][e & 1]);
        if (kk < fi.all_lo || kk + 16 > min(end, fi.all_hi)) {  // some row does not see some of them
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int row = 8 * nt + 2 * quad + i;
                    uint32_t bits = Seen::below(end - kk);
                    if (row < fi.it.ntok * p.G) bits &= fi.seen[row].keys(p, kk);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (!(bits >> (oct + 8 * h) & 1)) s[nt][2 * h + i] = -INFINITY;
                }
            if (end - kk < 16) {  // past the last key a stage holds anything
                if constexpr (CODE) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (oct + 8 * h >= end - kk) lv[h] = vs[h] = 0.f;
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
        bool moved = false;
        float alpha[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float x = max2(s[nt][i] + lv[0], s[nt][2 + i] + lv[1]);
                x = max2(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = max2(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = max2(x, __shfl_xor_sync(0xffffffffu, x, 16));
                alpha[nt][i] = 1.f;
                if (!(x <= m[nt][i] + kRescaleLog2)) {  // so also from -infinity, and for a NaN
                    const float now = max2(m[nt][i], x);
                    alpha[nt][i] = ex2_approx(m[nt][i] - now);
                    m[nt][i] = now;
                    l[nt][i] *= alpha[nt][i];
                    moved = true;
                }
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][nt][e] *= alpha[nt][e & 1];
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float ref = m[nt][i] == -INFINITY ? 0.f : m[nt][i];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float x = ex2_approx(s[nt][2 * h + i] - ref);
                    l[nt][i] += x;
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
                        const uint2 a = from_codes<X>(__byte_perm(w[0][d], w[1][d], pick)), b = from_codes<X>(__byte_perm(w[2][d], w[3][d], pick));
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

    auto finish = [&](const Item &it) -> bool {  // the item's sums from all warps, in their order
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (oct == 0) ml[warp * C::ROWS + 8 * nt + 2 * quad + i] = make_float2(m[nt][i], x);
            }
        if (!together()) return false;
        float f[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < W; k++) top = max2(top, ml[k * C::ROWS + 8 * nt + 2 * quad + i].x);
                f[nt][i] = ex2_approx(m[nt][i] - (top == -INFINITY ? 0.f : top));
            }
        const int rows = it.ntok * p.G;
        if (threadIdx.x < rows) {
            const int row = threadIdx.x, tok = row / p.G, hd = row - tok * p.G;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < W; k++) top = max2(top, ml[k * C::ROWS + row].x);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int k = 0; k < W; k++) {
                const float2 x = ml[k * C::ROWS + row];
                sum += x.y * ex2_approx(x.x - ref);
            }
            // sum = 0: every logit was -infinity, or no key was seen; a part leaves that to the join
            const bool bad = no_softmax(top), some = bad || sum > 0.f;
            const float sums = bad ? top : some ? top + __log2f(sum) : -INFINITY;
            const int64_t t = it.t0 + tok, h = it.kvh * p.G + hd;
            float none = 0.f;
            if (it.dst == TO_OUT) {
                if (!some && sees_keys<KIND>(p, t, it.pos0 + tok, it.len, it.base)) none = NAN;
                if (p.lse) p.lse[t * p.H + h] = sums * LN2;
            } else {
                p.pl[(int64_t)it.slot * SLOT<KIND> + row] = sums;
            }
            fin[row] = make_float2(bad ? NAN : some ? __fdividef(1.f, sum) : 0.f, some ? 0.f : none);
        }
#pragma unroll
        for (int i0 = 0; i0 < D / 16; i0 += C::MT) {
#pragma unroll
            for (int i = 0; i < C::MT; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float *y = merge + ((warp * C::MT + i) * C::ROWS + 8 * nt + 2 * quad + k) * 16;
                        const float a = o[i0 + i][nt][k] * f[nt][k], b = o[i0 + i][nt][2 + k] * f[nt][k];
                        if constexpr (CODE)
                            *reinterpret_cast<float2 *>(y + 2 * oct) = make_float2(a, b);
                        else
                            y[oct] = a, y[oct + 8] = b;
                    }
            if (!together()) return false;
            for (int e = threadIdx.x; e < C::MT * 8 * C::ROWS; e += 32 * W) {
                const int pair = e & 7, row = (e >> 3) % C::ROWS, i = (e >> 3) / C::ROWS;
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < W; k++) sum = add2(sum, *reinterpret_cast<const float2 *>(merge + ((k * C::MT + i) * C::ROWS + row) * 16 + 2 * pair));
                if (row >= rows) continue;
                const int dim = CODE ? pair * (D / 8) + 2 * (i0 + i) : 16 * (i0 + i) + 2 * pair;
                const float2 u = fin[row];
                // a row without sums may have met a page's NaN: its zeros are not a product
                const float2 y = u.x == 0.f ? make_float2(u.y, u.y) : make_float2(sum.x * u.x, sum.y * u.x);
                if (it.dst == TO_OUT) {
                    const int tok = row / p.G, hd = row - tok * p.G;
                    *reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + (it.t0 + tok) * p.ldo + (it.kvh * p.G + hd) * D + dim) = pack2<T>(y.x, y.y);
                } else {
                    *reinterpret_cast<float2 *>(p.po + ((int64_t)it.slot * SLOT<KIND> + row) * D + dim) = y;
                }
            }
            if (!together()) return false;
        }
        return true;
    };

#pragma unroll 1
    for (int n = 0, g = 0;; n++) {
        if (!wait_warp(item_full(n % C::NQ), (uint32_t)(n / C::NQ & 1), p.status, E2C_ERR_WAIT_ATTN)) return;
        const FewItem<C::ROWS> &fi = queue[n % C::NQ];
        if (fi.it.ntok < 0) return;
        begin(fi.it);
        const int count = fi.runs.count;
#pragma unroll 1
        for (int j = 0; j < count; j++, g++) {
            const int st = g % C::NS, key = fi.runs.key(j, C::KEYS), end = fi.runs.end(j);
            const int r0 = ((warp + g) % W) * 16;  // tiles that are not full fall to other warps each time
            // (also without keys of its own: a warp that ran ahead would count twice in the stage's barrier)
            if (!wait_warp(full(st), (uint32_t)(g / C::NS & 1), p.status, E2C_ERR_WAIT_ATTN)) return;
            if (key + r0 < end) use(fi, st, r0, key + r0, end);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(st));
        }
        if (!finish(fi.it)) return;
        if (lane == 0) mbar_arrive(item_empty(n % C::NQ));
    }
}

template <typename T, bool CODE, int D, int NT>
int run_few(const Args &a, const void *q, int64_t ldq, int sms, cudaStream_t st) {
    using C = Few<CODE, D, NT>;
    constexpr int KIND = SIGHT | FEW | (CODE ? CODES : 0);
    static E2cPerDev attr;
    const int dev = e2c_device(), grid = sms * C::CTAS;
    if (!attr.get(dev)) {
        if (cudaFuncSetAttribute(k_attention_few<T, CODE, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES) != cudaSuccess) {
            cudaGetLastError();
            e2c_set_msg("pages_attention: cannot reserve %d bytes of shared memory", C::BYTES);
            return -2;
        }
        attr.set(dev, 1);
    }
    const CUtensorMapDataType dt = CODE ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int es = CODE ? 1 : 2;
    const uint64_t rows = (uint64_t)a.pc.n_pages * a.pc.page, width = (uint64_t)a.pc.KV * D;
    const uint32_t box = a.pc.page < C::KEYS ? a.pc.page : C::KEYS;
    const auto map = C::WIDE == 64 ? e2c_tmap_2d_sw64 : e2c_tmap_2d;
    CUtensorMap tk, tv;
    if (map(&tk, a.pc.k, dt, es, width, rows, width * es, C::WIDE / es, box) ||
        map(&tv, a.pc.v, dt, es, width, rows, width * es, C::WIDE / es, box))
        return -3;
    e2c_launch_as(true, k_attention_few<T, CODE, D, NT>, dim3(grid), dim3(32 * (C::WARPS + 1)), C::BYTES, st, tk, tv, a, q, ldq);
    if (launch_error("pages_attention")) return -2;
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
