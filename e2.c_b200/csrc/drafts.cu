// drafts.cu — trees of drafted tokens at the end of cached sequences: what each sees and where it stands, and
// what stays of them.
//
// A tree is given by its rows' parents, each before its row. A row's bits are found by walking up: indices fall, so that
// its words are filled from the highest down and written once each. One thread a row; the walk's length is the
// row's depth, a load that the L1 cache answers each (64 trees of 31 rows: bound by the launch).
//
// Kept tokens move up behind the text, in every layer of k and v. Their order stays, so a token moves towards the front or not
// at all: where a block has loaded some tokens, it may overwrite anything before the last of them. What moves is
// little; the chain of lookups and the two launches bound it (64 sequences that keep some of 31 tokens in 12 layers of 4 heads
// of 128: 3.5 us in a graph).
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.h"
#include "pages.cuh"
#include "pdl.h"
#include "ptx.cuh"

namespace {

constexpr int ROWS = 128;  // threads of a k_tree block
constexpr int MOVE = 256, UNROLL = 4;

struct TreeArgs {
    e2c_pages pc;
    const int32_t *parents, *seqs, *q_start;
    int n, T, words;
    uint32_t *tree;
    int32_t *pos;
    int *status;
};

__global__ void __launch_bounds__(ROWS) k_tree(const TreeArgs p) {
    griddep_launch_dependents();
    griddep_wait();
    const int t = blockIdx.x * ROWS + threadIdx.x;
    if (t >= p.T) return;
    uint32_t *out = p.tree + (int64_t)t * p.words;
    int last;
    const int i = e2c_token_seq(p.q_start, p.n, p.T, t, last), q0 = i < 0 ? 0 : p.q_start[i];
    const int seq = i < 0 ? -1 : p.seqs[i];
    // a row outside the call's entries, or past what its words hold: no bits
    const bool ok = (unsigned)seq < (unsigned)p.pc.max_seqs && q0 >= 0 && last <= p.T && (t - q0) >> 5 < p.words;
    if (!ok) {
        for (int w = 0; w < p.words; w++) out[w] = 0;
        if (p.pos) p.pos[t] = 0;
        record_status(p.status, E2C_ERR_BAD_SEQ);
        return;
    }
    int r = t - q0, depth = 0;
    bool bad = false;
    for (int w = p.words - 1; w >= 0; w--) {
        uint32_t bits = 0;
        while (r >= 32 * w && r >= 0) {
            bits |= 1u << (r & 31);
            depth++;
            int up = p.parents[q0 + r];
            if (up >= r || up < -1) {
                bad = true;
                up = -1;
            }
            r = up;
        }
        out[w] = bits;
    }
    if (bad) record_status(p.status, E2C_ERR_BAD_SEQ);
    if (p.pos) p.pos[t] = p.pc.len[seq] - (last - q0) + depth - 1;
}

struct KeepArgs {
    e2c_pages pc;  // at layer 0
    const int32_t *seqs, *q_start, *kept, *counts;
    int n, T;
    int *status;
};
// entry i: its sequence, the tokens before its rows, its rows and those kept
struct Kept {
    int seq, text, rows, count, q0;
};
E2C_DEV bool kept_of(const KeepArgs &p, int i, Kept &k) {
    k.seq = p.seqs[i];
    k.q0 = p.q_start[i];
    const int64_t rows = (int64_t)p.q_start[i + 1] - k.q0;
    k.count = p.counts[i];
    if ((unsigned)k.seq >= (unsigned)p.pc.max_seqs || k.q0 < 0 || rows < 0 || k.q0 + rows > p.T || k.count < 0 || k.count > rows) return false;
    k.rows = (int)rows;
    const int len = p.pc.len[k.seq];
    if (len < k.rows || len > p.pc.max_blocks * p.pc.page) return false;
    k.text = len - k.rows;
    return true;
}
E2C_DEV int page_of(const e2c_pages &c, int seq, int at) { return c.table[(int64_t)seq * c.max_blocks + at / c.page]; }

// The kept tokens' `width` pieces each, in one layer: side by side (values, codes), or a page's tokens apart (scales)
template <typename V>
E2C_DEV void move_rows(const KeepArgs &p, const Kept &k, V *base, int width, bool apart) {
    const e2c_pages &c = p.pc;
    auto at = [&](int row, int x) -> V * {
        const int tok = k.text + row, page = page_of(c, k.seq, tok), slot = tok & (c.page - 1);
        const int64_t u = apart ? ((int64_t)page * width + x) * c.page + slot : ((int64_t)page * c.page + slot) * width + x;
        return base + u;
    };
    const int32_t *kept = p.kept + k.q0;
    const int cols = min(width, MOVE * UNROLL), most = MOVE * UNROLL / cols;
    for (int x0 = 0; x0 < width; x0 += cols) {
        for (int j0 = 0; j0 < k.count; j0 += most) {
            V v[UNROLL];
            const int rows = min(most, k.count - j0);
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int e = threadIdx.x + u * MOVE, j = e / cols, x = x0 + e - j * cols;
                if (j < rows && x < width && kept[j0 + j] != j0 + j) v[u] = *at(kept[j0 + j], x);
            }
            __syncthreads();  // all of these tokens are read before one of them is written
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int e = threadIdx.x + u * MOVE, j = e / cols, x = x0 + e - j * cols;
                if (j < rows && x < width && kept[j0 + j] != j0 + j) *at(j0 + j, x) = v[u];
            }
        }
    }
}

// A block per entry and (grid y) layer of k or v. Every block checks its entry, and those of the first layer's k leave the
// verdict for k_keep_end in the workspace.
__global__ void __launch_bounds__(MOVE) k_keep_move(const KeepArgs p) {
    griddep_launch_dependents();
    griddep_wait();
    const e2c_pages &c = p.pc;
    Kept k;
    const bool in = kept_of(p, blockIdx.x, k);
    bool bad = !in;
    if (in)
        for (int j = threadIdx.x; j < k.count; j += MOVE) {
            const int r = p.kept[k.q0 + j];
            if (r < j || r >= k.rows || (j > 0 && p.kept[k.q0 + j - 1] >= r)) {
                bad = true;
                continue;
            }
            if (r == j) continue;
            const int from = page_of(c, k.seq, k.text + r), to = page_of(c, k.seq, k.text + j);
            if ((unsigned)from >= (unsigned)c.n_pages || (unsigned)to >= (unsigned)c.n_pages || c.refs[to] > 1) bad = true;
        }
    bad = __syncthreads_or(bad);
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        c.ws[E2C_PAGES_WS_HEAD + blockIdx.x] = bad ? -1 : k.text + k.count;
        if (bad) record_status(p.status, E2C_ERR_BAD_SEQ);
    }
    if (bad) return;
    const int es = c.type == E2C_I8 ? 1 : 2;
    const int64_t row = (int64_t)c.KV * c.D * es, layer = (int64_t)c.n_pages * c.page * row;
    for (int l = blockIdx.y; l < 2 * c.layers; l += gridDim.y) {
        uint8_t *values = static_cast<uint8_t *>(l & 1 ? c.v : c.k) + (l >> 1) * layer;
        move_rows(p, k, reinterpret_cast<uint4 *>(values), (int)(row / 16), false);
        if (c.type == E2C_I8) move_rows(p, k, (l & 1 ? c.vs : c.ks) + (int64_t)(l >> 1) * c.n_pages * c.page * c.KV, c.KV, true);
    }
}

// Lengths, and the pages past them
__global__ void __launch_bounds__(MOVE) k_keep_end(const KeepArgs p) {
    griddep_launch_dependents();
    griddep_wait();
    const e2c_pages &c = p.pc;
    const int len = c.ws[E2C_PAGES_WS_HEAD + blockIdx.x];
    if (len < 0) return;
    const int seq = p.seqs[blockIdx.x], old = c.len[seq];
    const int b0 = (len + c.page - 1) / c.page, b1 = min((old + c.page - 1) / c.page, c.max_blocks);
    for (int b = b0 + threadIdx.x; b < b1; b += MOVE) {
        const int page = c.table[(int64_t)seq * c.max_blocks + b];
        if ((unsigned)page < (unsigned)c.n_pages) atomicSub(c.refs + page, 1);
    }
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) c.len[seq] = len;
}

int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 0;
    e2c_set_msg("%s launch: %s", what, cudaGetErrorString(e));
    return -2;
}

}  // namespace

extern "C" int e2c_pages_tree(const e2c_pages *pc, const int32_t *parents, const int32_t *seqs, const int32_t *q_start, int n, int T,
                              uint32_t *tree, int words, int32_t *pos, int *status, void *stream) {
    const TreeArgs a = {*pc, parents, seqs, q_start, n, T, words, tree, pos, status};
    e2c_launch_as(true, k_tree, dim3((T + ROWS - 1) / ROWS), dim3(ROWS), 0, (cudaStream_t)stream, a);
    return launched("pages_tree");
}

extern "C" int e2c_pages_keep(const e2c_pages *pc, const int32_t *seqs, const int32_t *q_start, const int32_t *kept, const int32_t *counts,
                              int n, int T, int *status, void *stream) {
    const KeepArgs a = {*pc, seqs, q_start, kept, counts, n, T, status};
    const int layers = 2 * pc->layers < 65535 ? 2 * pc->layers : 65535;
    e2c_launch_as(true, k_keep_move, dim3(n, layers), dim3(MOVE), 0, (cudaStream_t)stream, a);
    if (launched("pages_keep")) return -2;
    e2c_launch_as(true, k_keep_end, dim3(n), dim3(MOVE), 0, (cudaStream_t)stream, a);
    return launched("pages_keep");
}
