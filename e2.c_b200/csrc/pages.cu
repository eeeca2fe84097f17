// pages.cu — the page operations of the key/value cache: fork, append, free, compact, copy.
//
// The whole state of a cache lives on the device: a sequence's page table and length, and a count
// for each page of the sequences that map it (0: free). So every operation is stream-ordered, needs
// no host round trip and can be captured in a graph with the rest of a decode step.
//
// Which page goes where is fixed by a rule, not by the order in which threads run: an append
// takes the lowest free pages, given out in the batch's order and block by block, and a compaction
// moves the k-th page in use past the used count to the k-th hole below it. Both are prefix sums over
// the page counts, by one block of 1024 threads that reads 16 KB a step; counts are otherwise
// changed by integer atomics, whose order does not matter.
//
// Moving pages is bound by memory: every page is one contiguous run of page * KV * D elements in each
// layer of K and of V (1021 pages of 16 layers, 32 KB a run: 326 us, 6.5 TB/s; compaction of 718 MB of
// pages with its plan 236 us, 6.1 TB/s). The bookkeeping kernels take 2 to 8 us, which their launches
// bound.
#include <cuda_runtime.h>
#include <stdint.h>

#include "devstate.cuh"
#include "launch.h"
#include "pdl.h"
#include "ptx.cuh"

namespace {

constexpr int PLAN = 1024;  // threads of the planning block

// the workspace: counters, an append's offsets and copies (one per entry), page lists
enum { W_MOVES = 0, W_HEAD = 16 };
struct Ws {
    int32_t *off, *src, *dst, *list, *high, *remap;
};
E2C_DEV Ws ws_of(const e2c_pages &p) {
    int32_t *b = p.ws + W_HEAD;
    return {b, b + p.max_seqs, b + 2 * (int64_t)p.max_seqs, b + 3 * (int64_t)p.max_seqs,
            b + 3 * (int64_t)p.max_seqs + p.n_pages, b + 3 * (int64_t)p.max_seqs + 2 * (int64_t)p.n_pages};
}

E2C_DEV int ceil_div(int a, int b) { return (int)(((int64_t)a + b - 1) / b); }

// exclusive prefix sum over the block's threads; `total` gets the sum. Every thread calls it.
E2C_DEV int block_scan(int v, int &total, int32_t *warp_sums) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();  // the sums of the call before have been read
    if (lane == 31) warp_sums[w] = x;
    __syncthreads();
    int s = warp_sums[lane];  // 32 warps
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += y;
    }
    total = __shfl_sync(0xffffffffu, s, 31);
    const int before = __shfl_sync(0xffffffffu, s, w > 0 ? w - 1 : 0);
    return x - v + (w > 0 ? before : 0);
}

// Appends the pages of [from, to) for which `want(refs)` holds to list[count...], in order, until
// `most` have been found; returns how many there are by then (possibly more than `most`; entries past
// `most` are not stored). Four pages a thread a step.
template <typename Want>
E2C_DEV int list_pages(const int32_t *refs, int from, int to, int most, int32_t *list, int32_t *sums, Want want) {
    int count = 0;
    for (int base = from & ~3; base < to && count < most; base += 4 * PLAN) {
        const int p0 = base + 4 * (int)threadIdx.x;
        int hit = 0;
        if (p0 + 4 <= to && p0 >= from) {
            const int4 r = *reinterpret_cast<const int4 *>(refs + p0);
            hit = (want(r.x) ? 1 : 0) | (want(r.y) ? 2 : 0) | (want(r.z) ? 4 : 0) | (want(r.w) ? 8 : 0);
        } else {
            for (int i = 0; i < 4; i++)
                if (p0 + i >= from && p0 + i < to && want(refs[p0 + i])) hit |= 1 << i;
        }
        int total;
        int at = count + block_scan(__popc(hit), total, sums);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (hit >> i & 1) {
                if (at < most) list[at] = p0 + i;
                at++;
            }
        count += total;
    }
    return count;
}

// what an append asks for: sequence s grows from `held` tokens to `grown`, with a copy of its last
// page first when that page is partly filled and mapped by others too
struct Grow {
    int s, held, grown, b0, b1, cow, last;
};
E2C_DEV Grow grow_of(const e2c_pages &p, const int32_t *seqs, const int32_t *counts, int i, bool &bad) {
    Grow g = {};
    g.s = seqs[i];
    const int c = counts[i];
    bad = (unsigned)g.s >= (unsigned)p.max_seqs || c < 0;
    if (bad) return g;
    g.held = p.len[g.s];
    const int64_t grown = (int64_t)g.held + c;
    if (g.held < 0 || grown > (int64_t)p.max_blocks * p.page) {
        bad = true;
        return g;
    }
    g.grown = (int)grown;
    g.b0 = ceil_div(g.held, p.page);
    g.b1 = ceil_div(g.grown, p.page);
    if (c > 0 && g.held % p.page) {
        g.last = p.table[(int64_t)g.s * p.max_blocks + g.b0 - 1];
        if ((unsigned)g.last >= (unsigned)p.n_pages)
            bad = true;
        else
            g.cow = p.refs[g.last] > 1;
    }
    return g;
}

// One block: how many pages each entry needs and where its share of the free list begins; the free
// list; then the tables, lengths and counts. Copies of shared pages are left in ws (src < 0: none).
__global__ void __launch_bounds__(PLAN) k_append(const e2c_pages p, const int32_t *seqs, const int32_t *counts, int n, int *status) {
    __shared__ int32_t sums[32];
    griddep_launch_dependents();
    griddep_wait();
    const Ws w = ws_of(p);
    const int tid = threadIdx.x;
    int need = 0;
    for (int base = 0; base < n; base += PLAN) {
        const int i = base + tid;
        int want = 0;
        if (i < n) {
            bool bad;
            const Grow g = grow_of(p, seqs, counts, i, bad);
            if (bad)
                record_status(status, E2C_ERR_BAD_SEQ);
            else
                want = g.b1 - g.b0 + g.cow;
            w.src[i] = !bad && g.cow ? g.last : -1;
        }
        int total;
        const int at = block_scan(want, total, sums);
        if (i < n) w.off[i] = need + at;
        // totals saturate: more pages than the cache has are refused below whatever the number
        need = (int)min((int64_t)need + total, (int64_t)1 << 30);
    }
    const int found = need > p.n_pages ? 0 : list_pages(p.refs, 0, p.n_pages, need, w.list, sums, [](int r) { return r == 0; });
    if (found < need) {
        if (tid == 0) record_status(status, E2C_ERR_NO_PAGES);
        for (int i = tid; i < n; i += PLAN) w.src[i] = -1;
        return;
    }
    __syncthreads();
    // a warp per entry: a long prompt's blocks are mapped 32 at a time
    const int lane = tid & 31;
    for (int i = tid >> 5; i < n; i += PLAN / 32) {
        bool bad;
        Grow g = grow_of(p, seqs, counts, i, bad);
        // whether the last page is copied was settled above, before any count changed
        const int copied = w.src[i];
        __syncwarp();
        if (bad) continue;
        int32_t *row = p.table + (int64_t)g.s * p.max_blocks;
        const int at = w.off[i];
        const int cow = copied >= 0, first = g.b0 - cow, pages = g.b1 - first;
        for (int b = lane; b < pages; b += 32) {
            const int pg = w.list[at + b];
            if ((unsigned)pg >= (unsigned)p.n_pages) continue;  // only with a sequence named twice
            row[first + b] = pg;
            p.refs[pg] = 1;
        }
        if (lane == 0) {
            if (cow) {
                w.dst[i] = w.list[at];
                atomicSub(p.refs + copied, 1);
            }
            p.len[g.s] = g.grown;
        }
    }
}

// page tables: a block per (parent, child) or per freed sequence
__global__ void __launch_bounds__(256) k_fork(const e2c_pages p, const int32_t *parents, const int32_t *children, int *status) {
    griddep_launch_dependents();
    griddep_wait();
    const int a = parents[blockIdx.x], c = children[blockIdx.x];
    const bool in = (unsigned)a < (unsigned)p.max_seqs && (unsigned)c < (unsigned)p.max_seqs && a != c;
    const int held = in ? p.len[a] : 0;
    if (!in || held < 0 || (int64_t)held > (int64_t)p.max_blocks * p.page || p.len[c] != 0) {
        if (threadIdx.x == 0) record_status(status, E2C_ERR_BAD_SEQ);
        return;
    }
    const int32_t *from = p.table + (int64_t)a * p.max_blocks;
    int32_t *to = p.table + (int64_t)c * p.max_blocks;
    const int blocks = ceil_div(held, p.page);
    for (int b = threadIdx.x; b < blocks; b += 256) {
        const int pg = from[b];
        to[b] = pg;
        if ((unsigned)pg < (unsigned)p.n_pages) atomicAdd(p.refs + pg, 1);
    }
    __syncthreads();  // every thread has read the child's length
    if (threadIdx.x == 0) p.len[c] = held;
}

__global__ void __launch_bounds__(256) k_free(const e2c_pages p, const int32_t *seqs, int *status) {
    griddep_launch_dependents();
    griddep_wait();
    const int s = seqs[blockIdx.x];
    if ((unsigned)s >= (unsigned)p.max_seqs) {
        if (threadIdx.x == 0) record_status(status, E2C_ERR_BAD_SEQ);
        return;
    }
    const int blocks = min(ceil_div(max(p.len[s], 0), p.page), p.max_blocks);
    const int32_t *row = p.table + (int64_t)s * p.max_blocks;
    for (int b = threadIdx.x; b < blocks; b += 256)
        if ((unsigned)row[b] < (unsigned)p.n_pages) atomicSub(p.refs + row[b], 1);
    __syncthreads();
    if (threadIdx.x == 0) p.len[s] = 0;
}

// One block: the used count, the holes below it and the pages in use past it, matched in order; the
// counts follow their pages, and `remap` says where every page went.
__global__ void __launch_bounds__(PLAN) k_compact(const e2c_pages p, int32_t *used_out) {
    __shared__ int32_t sums[32];
    griddep_launch_dependents();
    griddep_wait();
    const Ws w = ws_of(p);
    const int tid = threadIdx.x;
    int mine = 0;
    for (int q = tid; q < p.n_pages; q += PLAN) {
        mine += p.refs[q] > 0;
        w.remap[q] = q;
    }
    int used;
    block_scan(mine, used, sums);
    const int moves = list_pages(p.refs, 0, used, p.n_pages, w.list, sums, [](int r) { return r <= 0; });
    list_pages(p.refs, used, p.n_pages, p.n_pages, w.high, sums, [](int r) { return r > 0; });  // as many
    __syncthreads();
    for (int m = tid; m < moves; m += PLAN) {
        const int from = w.high[m], to = w.list[m];
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
        w.remap[from] = to;
    }
    if (tid == 0) {
        p.ws[W_MOVES] = moves;
        if (used_out) *used_out = used;
    }
}

__global__ void __launch_bounds__(256) k_remap(const e2c_pages p) {
    griddep_launch_dependents();
    griddep_wait();
    const Ws w = ws_of(p);
    const int s = blockIdx.x;
    const int blocks = min(ceil_div(max(p.len[s], 0), p.page), p.max_blocks);
    int32_t *row = p.table + (int64_t)s * p.max_blocks;
    for (int b = threadIdx.x; b < blocks; b += 256)
        if ((unsigned)row[b] < (unsigned)p.n_pages) row[b] = w.remap[row[b]];
}

// src[i] -> dst[i] in every layer of K and V, i < n (or *count where that is given); src < 0: none.
// A step moves one piece of a page's run in one layer: 2^shift threads x UNROLL 16-byte vectors. A run
// shorter than 16 KB takes fewer threads, and the block moves several pieces at once.
constexpr int UNROLL = 4;
__global__ void __launch_bounds__(256) k_move(const e2c_pages p, const int32_t *src, const int32_t *dst, int n, const int32_t *count,
                                              int vecs, int pieces, int shift, int *status) {
    griddep_launch_dependents();
    griddep_wait();
    if (count) n = min(n, *count);
    const int per_page = 2 * p.layers * pieces;
    const int64_t total = (int64_t)n * per_page, layer = (int64_t)p.n_pages * vecs;
    const int width = 1 << shift, lane = threadIdx.x & (width - 1);
    for (int64_t u = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> shift; u < total; u += (int64_t)gridDim.x * (256 >> shift)) {
        const int i = (int)(u / per_page);
        const int from = src[i];
        if (from < 0) continue;
        const int to = dst[i], rem = (int)(u - (int64_t)i * per_page);
        if (from >= p.n_pages || (unsigned)to >= (unsigned)p.n_pages) {
            if (lane == 0) record_status(status, E2C_ERR_BAD_SEQ);
            continue;
        }
        const int l2 = rem / pieces, piece = rem - l2 * pieces;  // layer 2 l of K, 2 l + 1 of V
        uint4 *base = static_cast<uint4 *>(l2 & 1 ? p.v : p.k) + (l2 >> 1) * layer;
        const uint4 *a = base + (int64_t)from * vecs;
        uint4 *b = base + (int64_t)to * vecs;
        const int v0 = piece * (width * UNROLL) + lane;
        uint4 r[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; j++)
            if (v0 + width * j < vecs) r[j] = a[v0 + width * j];
#pragma unroll
        for (int j = 0; j < UNROLL; j++)
            if (v0 + width * j < vecs) b[v0 + width * j] = r[j];
    }
}

int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 0;
    e2c_set_msg("%s launch: %s", what, cudaGetErrorString(e));
    return -2;
}

int move_pages(const e2c_pages *pc, const int32_t *src, const int32_t *dst, int n, const int32_t *count, int *status, void *stream,
               const char *what) {
    if (n <= 0) return 0;
    const int sms = e2c_sm_count(e2c_device());
    if (!sms) {
        e2c_set_msg("%s: no CUDA device", what);
        return -2;
    }
    const int64_t bytes = (int64_t)pc->page * pc->KV * pc->D * 2;
    const int vecs = (int)(bytes / 16);
    int shift = 3;
    while (shift < 8 && (UNROLL << shift) < vecs) shift++;
    const int pieces = (vecs + (UNROLL << shift) - 1) / (UNROLL << shift);
    const int64_t blocks = ((int64_t)n * 2 * pc->layers * pieces * (1 << shift) + 255) / 256;
    // A block a piece where the host knows how many there are (1021 pages of 16 layers, 32 KB a run: 326 us,
    // the rate of a plain copy; 373 us with 8 blocks an SM that go round); where only the device does,
    // enough of them that go round.
    const int64_t most = (int64_t)sms * (count ? 64 : 1 << 20);
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    e2c_launch_as(true, k_move, dim3(grid), dim3(256), 0, (cudaStream_t)stream, *pc, src, dst, n, count, vecs, pieces, shift,
               status);
    return launched(what);
}

int32_t *ws_at(const e2c_pages *pc, int64_t ints) { return pc->ws + W_HEAD + ints; }

}  // namespace

extern "C" size_t e2c_pages_ws_ints(int n_pages, int max_seqs) {
    return W_HEAD + 3 * ((size_t)max_seqs + (size_t)n_pages);
}

extern "C" int e2c_pages_copy(const e2c_pages *pc, const int32_t *src, const int32_t *dst, int n, int *status, void *stream) {
    return move_pages(pc, src, dst, n, nullptr, status, stream, "pages_copy");
}

extern "C" int e2c_pages_fork(const e2c_pages *pc, const int32_t *parents, const int32_t *children, int n, int *status, void *stream) {
    if (n <= 0) return 0;
    e2c_launch_as(true, k_fork, dim3(n), dim3(256), 0, (cudaStream_t)stream, *pc, parents, children, status);
    return launched("pages_fork");
}

extern "C" int e2c_pages_append(const e2c_pages *pc, const int32_t *seqs, const int32_t *counts, int n, int *status, void *stream) {
    if (n <= 0) return 0;
    e2c_launch_as(true, k_append, dim3(1), dim3(PLAN), 0, (cudaStream_t)stream, *pc, seqs, counts, n, status);
    if (launched("pages_append")) return -2;
    return move_pages(pc, ws_at(pc, pc->max_seqs), ws_at(pc, 2 * (int64_t)pc->max_seqs), n, nullptr, status, stream, "pages_append");
}

extern "C" int e2c_pages_free(const e2c_pages *pc, const int32_t *seqs, int n, int *status, void *stream) {
    if (n <= 0) return 0;
    e2c_launch_as(true, k_free, dim3(n), dim3(256), 0, (cudaStream_t)stream, *pc, seqs, status);
    return launched("pages_free");
}

extern "C" int e2c_pages_compact(const e2c_pages *pc, int32_t *used, int *status, void *stream) {
    e2c_launch_as(true, k_compact, dim3(1), dim3(PLAN), 0, (cudaStream_t)stream, *pc, used);
    if (launched("pages_compact")) return -2;
    e2c_launch_as(true, k_remap, dim3(pc->max_seqs), dim3(256), 0, (cudaStream_t)stream, *pc);
    if (launched("pages_compact")) return -2;
    const int64_t list = 3 * (int64_t)pc->max_seqs;
    return move_pages(pc, ws_at(pc, list + pc->n_pages), ws_at(pc, list), pc->n_pages / 2 + 1, pc->ws + W_MOVES, status, stream,
                      "pages_compact");
}
