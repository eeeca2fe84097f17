// attention_pages.cu — attention over a paged cache: when a call reads a shared prefix by itself, its
// workspace, and the kernels (attention_pages.cuh) of rows that see what causal order and a window leave.
#include "attention_pages.cuh"

namespace {

// Sequences of few query tokens fill a small part of a 128-row tile each; packed, the batch reads the prefix
// once per 128 rows instead of once per sequence. It is done up to half a tile of the longest entry's rows (max_q
// stands for it: the rows themselves are on the device). Past that the gain fades and turns over (us a call,
// packed and not; 128 sequences behind 16384 tokens, 32 heads of 128 over 8, 68 rows each 632 and 1042, 96 rows 905 and
// 1045, 112 rows 1050 and 1082, 128 rows 1159 and 1105; 256 behind 6144, 4 heads of 256 over 2, 66 rows 240 and
// 300, 80 rows 329 and 302, 112 rows 443 and 316; 32 behind 4096, heads of 128, 68 rows 79 and 103, 96 rows 111
// and 97), and entries of more rows than a tile would need a join that knows their tiles. Where
// all sequences' own passes over the prefix are a dozen tiles a block, joining two parts of every row
// costs more than it saves (8 key heads of 128, 300 tokens past the prefix, us a call, packed and not: 16
// sequences behind 1024 tokens, 6.5 tiles a block, 28.4 and 23.8; 32 behind 1024, 13.4 tiles, 31.2 and 32.7;
// 64 behind 512, 13.6 tiles, 35.2 and 38.5).
bool use_prefix(int n, int max_q, int KV, int G, int shared, int sms) {
    return shared > 0 && 2 * max_q * G <= TR && (int64_t)(n - 1) * KV * ((shared + TK - 1) / TK) > PREFIX_TILES * sms;
}

bool few_rows(bool here, bool prefix, int max_q, int G) { return here && !prefix && (int64_t)max_q * G <= FEW_ROWS; }

struct Layout {
    size_t split, before, po, pl, dpo, dpl, bytes;
};
// Blocks an SM and rows of a part that a call for few rows has at most: its parts take no more than the others' (16 of 128 rows, twice)
constexpr int FEW_BLOCKS = 2;
static_assert(FEW_BLOCKS * FEW_ROWS <= 128, "workspace");
Layout layout(int blocks, int n, int T, int H, int KV, int D, bool prefix) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    // a prefix has at most one item a block, or one for each row tile of each key head if those are more
    const size_t tpt = TR / (H / KV), rows = KV * ((T + tpt - 1) / tpt);
    const size_t slots = 2 * (size_t)blocks + (prefix ? (rows > (size_t)blocks ? rows : (size_t)blocks) : 0);
    l.split = take(sizeof(int4) * 2 * FEW_BLOCKS * blocks);
    l.before = take(sizeof(int) * ((size_t)n + 2));
    l.pl = take(sizeof(float) * slots * TR);
    l.po = take(sizeof(float) * slots * TR * D);
    l.dpl = take(prefix ? sizeof(float) * (size_t)T * H : 0);
    l.dpo = take(prefix ? sizeof(float) * (size_t)T * H * D : 0);
    l.bytes = at;
    return l;
}

}  // namespace

extern "C" size_t e2c_pages_attention_ws_bytes(int n, int T, int max_q, int H, int KV, int D, int shared) {
    const int sms = e2c_sm_count(e2c_device());
    return sms ? layout(sms, n, T, H, KV, D, use_prefix(n, max_q, KV, H / KV, shared, sms)).bytes : 0;
}

extern "C" int e2c_pages_attention(const e2c_pages *pc, int q_type, const void *q, int64_t ldq, const int32_t *seqs,
                                   const int32_t *q_start, int n, int T, int max_q, int H, int shared, int causal, int window, int sinks,
                                   const uint32_t *tree, int words, float scale, void *out, int64_t ldo, float *lse, void *ws,
                                   size_t ws_bytes, int *status, void *stream) {
    const int sms = e2c_sm_count(e2c_device());
    if (!sms) {
        e2c_set_msg("pages_attention: no CUDA device");
        return -2;
    }
    const int G = H / pc->KV;
    const bool prefix = use_prefix(n, max_q, pc->KV, G, shared, sms);
    const Layout l = layout(sms, n, T, H, pc->KV, pc->D, prefix);
    if (ws_bytes < l.bytes) {
        e2c_set_msg("pages_attention: workspace");
        return -1;
    }
    e2c_attn_args a;
    a.pc = *pc;
    a.q_type = q_type;
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
    a.sinks = a.window >= 0 ? sinks : 0;
    a.tree = tree;
    a.words = words;
    a.align = pc->page < 16 ? 16 : pc->page < 128 ? pc->page : 128;
    // a scale of zero keeps masked logits (-inf) apart from the others (0)
    a.c = scale == 0.f ? 1e-30f : fabsf(scale) * LOG2E;
    a.neg = scale < 0.f;
    a.out = out;
    a.ldo = ldo;
    a.lse = lse;
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.split = reinterpret_cast<int4 *>(w + l.split);
    a.before = reinterpret_cast<int *>(w + l.before);
    a.po = reinterpret_cast<float *>(w + l.po);
    a.pl = reinterpret_cast<float *>(w + l.pl);
    a.dpo = reinterpret_cast<float *>(w + l.dpo);
    a.dpl = reinterpret_cast<float *>(w + l.dpl);
    a.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    const bool codes = pc->type == E2C_I8;
    if (few_rows(codes || a.sinks || a.tree, prefix, max_q, G)) return codes ? e2c_attn_few_codes(a, q, ldq, sms, st) : e2c_attn_few(a, q, ldq, sms, st);
    if (codes) return e2c_attn_codes(a, q, ldq, prefix, sms, st);
    return a.sinks || a.tree ? e2c_attn_sight(a, q, ldq, prefix, sms, st) : e2c_attn_plain(a, q, ldq, prefix, sms, st);
}

int e2c_attn_plain(const e2c_attn_args &a, const void *q, int64_t ldq, bool prefix, int sms, cudaStream_t st) {
    return run_kind<0>(a, q, ldq, prefix, sms, st);
}
