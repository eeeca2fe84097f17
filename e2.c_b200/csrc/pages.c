/* pages.c — the prompt cache's part of the C ABI (include/e2cuda.h): rotary tables and rotation, the
 * paged key/value cache and attention over it. Argument checks, then the launchers of launch.h. */
#include <math.h>
#include <stdio.h>

#include "internal.h"

#define E2CU_PI 3.14159265358979323846

static int bits16(int t) { return t == E2CUDA_BF16 || t == E2CUDA_F16; }

/* ------------------------------------------------------------------ rotary positions */
/* pair index at which a pair makes `turns` rotations over `original` positions */
static double pair_of(double turns, double original, double theta, int rot) {
    return rot * log(original / (turns * 2.0 * E2CU_PI)) / (2.0 * log(theta));
}

static int frequencies(double *f, int rot, float theta, const e2cuda_rope_scaling *s, double *gain) {
    const int half = rot / 2, kind = s ? s->kind : E2CUDA_ROPE_PLAIN;
    const double factor = s ? s->factor : 1.0;
    *gain = s && s->gain != 0.f ? s->gain : 1.0;
    if (kind < E2CUDA_ROPE_PLAIN || kind > E2CUDA_ROPE_BY_PAIRS) {
        e2cu_err("rope_table: scaling kind %d", kind);
        return -1;
    }
    if (kind != E2CUDA_ROPE_PLAIN && !(factor >= 1.0 && isfinite(factor))) {
        e2cu_err("rope_table: scaling factor %g (at least 1)", factor);
        return -1;
    }
    double base = theta;
    if (kind == E2CUDA_ROPE_NTK && rot > 2) base *= pow(factor, (double)rot / (rot - 2));
    for (int i = 0; i < half; i++) f[i] = pow(base, -2.0 * i / rot);
    if (kind == E2CUDA_ROPE_LINEAR)
        for (int i = 0; i < half; i++) f[i] /= factor;
    if (kind == E2CUDA_ROPE_BY_ROTATIONS || kind == E2CUDA_ROPE_BY_PAIRS) {
        const int by_pairs = kind == E2CUDA_ROPE_BY_PAIRS;
        const double fast = s->fast != 0.f ? s->fast : by_pairs ? 32.0 : 4.0, slow = s->slow != 0.f ? s->slow : 1.0;
        if (s->original < 1 || !(slow > 0.0 && fast > slow && isfinite(fast))) {
            e2cu_err("rope_table: original length %d, rotations %g to %g", s->original, slow, fast);
            return -1;
        }
        double first = 0, last = 0;
        if (by_pairs) {
            if (!(theta > 1.f)) {
                e2cu_err("rope_table: theta %g (above 1 for scaling by pairs)", theta);
                return -1;
            }
            first = fmax(floor(pair_of(fast, s->original, theta, rot)), 0.0);
            last = fmin(ceil(pair_of(slow, s->original, theta, rot)), rot - 1.0);
            if (last <= first) last = first + 1e-3;
            if (s->gain == 0.f) *gain = 0.1 * log(factor) + 1.0;
        }
        for (int i = 0; i < half; i++) {
            /* 1: the frequency is kept, 0: it is divided by the factor */
            double keep = by_pairs ? (last - i) / (last - first) : (s->original * f[i] / (2.0 * E2CU_PI) - slow) / (fast - slow);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f[i] *= keep + (1.0 - keep) / factor;
        }
    }
    return 0;
}

int e2cuda_rope_table(float *cos_t, float *sin_t, int positions, int rot, float theta, const e2cuda_rope_scaling *s, void *stream) {
    double f[256], gain;
    if (!cos_t || !sin_t || positions < 1 || rot < 2 || rot > 512 || rot % 2 || !(theta > 0.f) || !isfinite(theta)) {
        e2cu_err("rope_table: bad arguments (positions %d, rot %d, theta %g)", positions, rot, theta);
        return -1;
    }
    if (frequencies(f, rot, theta, s, &gain)) return -1;
    return e2cu_launch(e2c_rope_table(cos_t, sin_t, positions, rot / 2, f, gain, stream), "rope_table");
}

int e2cuda_rope(const void *x, int ldx, int x_type, void *y, int ldy, int y_type, const float *cos_t, const float *sin_t,
                int positions, int rot, const int32_t *pos, int T, int heads, int head_dim, int flags, void *stream) {
    const int known = E2CUDA_ROPE_INTERLEAVED | E2CUDA_ROPE_TRANSPOSE;
    if (T == 0) return 0;
    if (!x || !y || !cos_t || !sin_t || T < 0 || heads < 1 || head_dim < 2 || rot < 2 || rot % 2 || rot > head_dim ||
        positions < 1 || (flags & ~known) || ldx < (int64_t)heads * head_dim || ldy < (int64_t)heads * head_dim ||
        (!pos && T > positions)) {
        e2cu_err("rope: bad arguments (T %d, heads %d of %d, rot %d, ld %d %d, positions %d)", T, heads, head_dim, rot, ldx, ldy,
                 positions);
        return -1;
    }
    if (x_type < E2CUDA_F32 || x_type > E2CUDA_F16 || y_type < E2CUDA_F32 || y_type > E2CUDA_F16 ||
        (x_type != y_type && x_type != E2CUDA_F32) || (x == y && (x_type != y_type || ldx != ldy))) {
        e2cu_err("rope: types %d -> %d (equal, or from fp32; in place: equal with equal rows)", x_type, y_type);
        return -1;
    }
    return e2cu_launch(e2c_rope(x, ldx, x_type, y, ldy, y_type, cos_t, sin_t, positions, rot / 2, pos, T, heads, head_dim,
                                flags & E2CUDA_ROPE_INTERLEAVED, flags & E2CUDA_ROPE_TRANSPOSE, e2cu_status(), stream),
                       "rope");
}

/* ------------------------------------------------------------------ the paged cache */
size_t e2cuda_pages_ws_bytes(int n_pages, int max_seqs) {
    return n_pages < 0 || max_seqs < 0 ? 0 : e2c_pages_ws_ints(n_pages, max_seqs) * sizeof(int32_t);
}

/* checks a cache and gives the launchers' view of it, at `layer` */
static int view(const e2cuda_pages *p, int layer, e2c_pages *out, const char *what) {
    if (!p || !p->k || !p->v || !p->table || !p->len || !p->refs || !p->ws) {
        e2cu_err("%s: a cache's k, v, table, len, refs and ws must be given", what);
        return -1;
    }
    if ((!bits16(p->type) && p->type != E2CUDA_I8) || p->layers < 1 || p->n_pages < 1 || p->page < 8 || p->page > 1024 || (p->page & (p->page - 1)) ||
        p->kv_heads < 1 || p->kv_heads > 1024 || (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) ||
        p->max_seqs < 1 || p->max_blocks < 1 || p->max_blocks > 1 << 20 || (int64_t)p->max_blocks * p->page > 1 << 30 ||
        (int64_t)p->n_pages * p->page > INT32_MAX) {
        e2cu_err("%s: cache of type %d, %d layers, %d pages of %d, %d heads of %d, %d sequences of %d blocks", what, p->type,
                 p->layers, p->n_pages, p->page, p->kv_heads, p->head_dim, p->max_seqs, p->max_blocks);
        return -1;
    }
    if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->refs) & 15) {
        e2cu_err("%s: a cache's k, v and refs must be 16-byte aligned", what);
        return -1;
    }
    const int codes = p->type == E2CUDA_I8;
    if (codes && (!p->k_scale || !p->v_scale || (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 15))) {
        e2cu_err("%s: a cache of 8 bits needs k_scale and v_scale, 16-byte aligned", what);
        return -1;
    }
    if (layer < 0 || layer >= p->layers) {
        e2cu_err("%s: layer %d of %d", what, layer, p->layers);
        return -1;
    }
    const size_t heads = (size_t)layer * p->n_pages * p->page * p->kv_heads, at = heads * p->head_dim * (codes ? 1 : 2);
    *out = (e2c_pages){ .k = (char *)p->k + at, .v = (char *)p->v + at, .ks = codes ? p->k_scale + heads : NULL,
                        .vs = codes ? p->v_scale + heads : NULL, .table = p->table, .len = p->len, .refs = p->refs,
                        .ws = p->ws, .type = p->type, .layers = p->layers, .n_pages = p->n_pages, .page = p->page,
                        .KV = p->kv_heads, .D = p->head_dim, .max_seqs = p->max_seqs, .max_blocks = p->max_blocks };
    return 0;
}

/* a list of n device indices; more than `most` cannot be distinct */
static int list_ok(const void *a, const void *b, int n, int most, const char *what) {
    if (n >= 0 && n <= most && (n == 0 || (a && b))) return 1;
    e2cu_err("%s: bad list (n %d of at most %d)", what, n, most);
    return 0;
}

int e2cuda_pages_copy(const e2cuda_pages *pc, const int32_t *src, const int32_t *dst, int n, void *stream) {
    e2c_pages v;
    if (view(pc, 0, &v, "pages_copy") || !list_ok(src, dst, n, v.n_pages, "pages_copy")) return -1;
    return n ? e2cu_launch(e2c_pages_copy(&v, src, dst, n, e2cu_status(), stream), "pages_copy") : 0;
}

int e2cuda_pages_fork(const e2cuda_pages *pc, const int32_t *parents, const int32_t *children, int n, void *stream) {
    e2c_pages v;
    if (view(pc, 0, &v, "pages_fork") || !list_ok(parents, children, n, v.max_seqs, "pages_fork")) return -1;
    return n ? e2cu_launch(e2c_pages_fork(&v, parents, children, n, e2cu_status(), stream), "pages_fork") : 0;
}

int e2cuda_pages_append(const e2cuda_pages *pc, const int32_t *seqs, const int32_t *counts, int n, void *stream) {
    e2c_pages v;
    if (view(pc, 0, &v, "pages_append") || !list_ok(seqs, counts, n, v.max_seqs, "pages_append")) return -1;
    return n ? e2cu_launch(e2c_pages_append(&v, seqs, counts, n, e2cu_status(), stream), "pages_append") : 0;
}

int e2cuda_pages_free(const e2cuda_pages *pc, const int32_t *seqs, int n, void *stream) {
    e2c_pages v;
    if (view(pc, 0, &v, "pages_free") || !list_ok(seqs, seqs, n, v.max_seqs, "pages_free")) return -1;
    return n ? e2cu_launch(e2c_pages_free(&v, seqs, n, e2cu_status(), stream), "pages_free") : 0;
}

int e2cuda_pages_compact(const e2cuda_pages *pc, int32_t *used, void *stream) {
    e2c_pages v;
    if (view(pc, 0, &v, "pages_compact")) return -1;
    return e2cu_launch(e2c_pages_compact(&v, used, e2cu_status(), stream), "pages_compact");
}

/* the batch a store or an attention call describes */
static int batch_ok(const int32_t *seqs, const int32_t *q_start, int n, int T, int heads, int kv, const char *what) {
    if (seqs && q_start && n >= 1 && T >= 1 && heads >= kv && heads % kv == 0) return 1;
    e2cu_err("%s: bad batch (n %d, T %d, heads %d over %d)", what, n, T, heads, kv);
    return 0;
}

int e2cuda_pages_store(const e2cuda_pages *pc, int layer, int x_type, const void *q, int ldq, const void *k, int ldk,
                       const void *v, int ldv, void *q_out, int ldo, const float *cos_t, const float *sin_t, int positions,
                       int rot, int flags, const int32_t *seqs, const int32_t *q_start, int n, int T, int heads, void *stream) {
    const int q_type = pc && pc->type != E2CUDA_I8 ? pc->type : x_type;
    return e2cuda_pages_store_at(pc, layer, x_type, q, ldq, k, ldk, v, ldv, q_out, q_type, ldo, cos_t, sin_t, positions, rot, flags,
                                 NULL, seqs, q_start, n, T, heads, stream);
}

int e2cuda_pages_store_at(const e2cuda_pages *pc, int layer, int x_type, const void *q, int ldq, const void *k, int ldk,
                          const void *v, int ldv, void *q_out, int q_type, int ldo, const float *cos_t, const float *sin_t,
                          int positions, int rot, int flags, const int32_t *pos, const int32_t *seqs, const int32_t *q_start, int n,
                          int T, int heads, void *stream) {
    e2c_pages c;
    if (view(pc, layer, &c, "pages_store")) return -1;
    if (T == 0) return 0;
    if (!batch_ok(seqs, q_start, n, T, heads, c.KV, "pages_store")) return -1;
    const int64_t qrow = (int64_t)heads * c.D, krow = (int64_t)c.KV * c.D;
    if (!q || !k || !v || !q_out || !cos_t || !sin_t || ldq < qrow || ldo < qrow || ldk < krow || ldv < krow || positions < 1 ||
        rot < 2 || rot % 2 || rot > c.D || (flags & ~E2CUDA_ROPE_INTERLEAVED) || !bits16(q_type) ||
        (c.type == E2CUDA_I8 ? x_type != E2CUDA_F32 && !bits16(x_type) : q_type != c.type || (x_type != E2CUDA_F32 && x_type != c.type)) ||
        (q == q_out && (x_type != q_type || ldq != ldo))) {
        e2cu_err("pages_store: bad arguments (types %d -> %d, %d, ld %d %d %d -> %d, rot %d, positions %d, flags %d)", x_type, q_type,
                 c.type, ldq, ldk, ldv, ldo, rot, positions, flags);
        return -1;
    }
    return e2cu_launch(e2c_pages_store(&c, x_type, q, ldq, k, ldk, v, ldv, q_out, q_type, ldo, cos_t, sin_t, positions, rot / 2,
                                       flags & E2CUDA_ROPE_INTERLEAVED, pos, seqs, q_start, n, T, heads, e2cu_status(), stream),
                       "pages_store");
}

int e2cuda_pages_load(const e2cuda_pages *pc, int layer, const int32_t *seqs, const int32_t *first, const int32_t *q_start, int n, int T,
                      void *k_out, void *v_out, int y_type, void *stream) {
    e2c_pages c;
    if (view(pc, layer, &c, "pages_load")) return -1;
    if (T == 0) return 0;
    if (!seqs || !q_start || n < 1 || T < 1 || !k_out || !v_out || (((uintptr_t)k_out | (uintptr_t)v_out) & 15) ||
        (y_type != E2CUDA_F32 && !bits16(y_type))) {
        e2cu_err("pages_load: bad arguments (n %d, T %d, type %d; outputs 16-byte aligned)", n, T, y_type);
        return -1;
    }
    return e2cu_launch(e2c_pages_load(&c, seqs, first, q_start, n, T, k_out, v_out, y_type, e2cu_status(), stream), "pages_load");
}

/* ------------------------------------------------------------------ drafted tokens */
int e2cuda_pages_tree(const e2cuda_pages *pc, const int32_t *parents, const int32_t *seqs, const int32_t *q_start, int n, int T,
                      uint32_t *tree, int words, int32_t *pos, void *stream) {
    e2c_pages c;
    if (view(pc, 0, &c, "pages_tree")) return -1;
    if (T == 0) return 0;
    if (!parents || !seqs || !q_start || n < 1 || T < 1 || !tree || words < 1 || (int64_t)T * words > INT32_MAX) {
        e2cu_err("pages_tree: bad arguments (n %d, T %d, words %d)", n, T, words);
        return -1;
    }
    return e2cu_launch(e2c_pages_tree(&c, parents, seqs, q_start, n, T, tree, words, pos, e2cu_status(), stream), "pages_tree");
}

int e2cuda_pages_keep(const e2cuda_pages *pc, const int32_t *seqs, const int32_t *q_start, const int32_t *kept, const int32_t *counts,
                      int n, int T, void *stream) {
    e2c_pages c;
    if (view(pc, 0, &c, "pages_keep") || !list_ok(seqs, q_start, n, c.max_seqs, "pages_keep")) return -1;
    if (n == 0 || T == 0) return 0;
    if (T < 0 || !kept || !counts) {
        e2cu_err("pages_keep: bad arguments (T %d)", T);
        return -1;
    }
    return e2cu_launch(e2c_pages_keep(&c, seqs, q_start, kept, counts, n, T, e2cu_status(), stream), "pages_keep");
}

/* what an attention call and the size of its workspace take: a row tile holds 128 (token, head) rows, so one token's
 * heads over a key head must fit in it */
static int attention_ok(const e2c_pages *c, int n, int T, int max_q, int heads, int shared) {
    if (n >= 1 && T >= 1 && max_q >= 1 && heads >= c->KV && heads % c->KV == 0 && heads / c->KV <= 128 && shared >= 0) return 1;
    e2cu_err("pages_attention: bad batch (n %d, T %d, max_q %d, heads %d over %d, shared %d)", n, T, max_q, heads, c->KV, shared);
    return 0;
}

size_t e2cuda_pages_attention_ws_bytes(const e2cuda_pages *pc, int n, int T, int max_q, int heads, int shared) {
    e2c_pages c;
    if (view(pc, 0, &c, "pages_attention") || !attention_ok(&c, n, T, max_q, heads, shared)) return 0;
    return e2c_pages_attention_ws_bytes(n, T, max_q, heads, c.KV, c.D, shared);
}

int e2cuda_pages_attention(const e2cuda_pages *pc, int layer, const void *q, int ldq, const int32_t *seqs, const int32_t *q_start,
                           int n, int T, int max_q, int heads, int shared, int causal, int window, float scale, void *out, int ldo,
                           float *lse, void *ws, size_t ws_bytes, void *stream) {
    const e2cuda_sight s = { .causal = causal, .window = window };
    return e2cuda_pages_attention_sight(pc, layer, pc ? pc->type : 0, q, ldq, seqs, q_start, n, T, max_q, heads, shared, &s, scale, out,
                                        ldo, lse, ws, ws_bytes, stream);
}

int e2cuda_pages_attention_sight(const e2cuda_pages *pc, int layer, int q_type, const void *q, int ldq, const int32_t *seqs,
                                 const int32_t *q_start, int n, int T, int max_q, int heads, int shared, const e2cuda_sight *sight,
                                 float scale, void *out, int ldo, float *lse, void *ws, size_t ws_bytes, void *stream) {
    e2c_pages c;
    if (view(pc, layer, &c, "pages_attention")) return -1;
    if (T == 0) return 0;
    if (!batch_ok(seqs, q_start, n, T, heads, c.KV, "pages_attention") || !attention_ok(&c, n, T, max_q, heads, shared)) return -1;
    const int64_t row = (int64_t)heads * c.D;
    if (!q || !out || ldq < row || ldo < row || max_q > T || !isfinite(scale) || shared % c.page ||
        shared > (int64_t)c.max_blocks * c.page) {
        e2cu_err("pages_attention: bad arguments (ld %d -> %d, max_q %d, heads %d over %d, shared %d of pages of %d)", ldq, ldo,
                 max_q, heads, c.KV, shared, c.page);
        return -1;
    }
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ldq % 8 || ldo % 8) {
        e2cu_err("pages_attention: q and out must be 16-byte aligned with rows of a multiple of 8 elements");
        return -1;
    }
    if (!bits16(q_type) || (c.type != E2CUDA_I8 && q_type != c.type)) {
        e2cu_err("pages_attention: q of type %d for a cache of type %d", q_type, c.type);
        return -1;
    }
    if (!sight || sight->sinks < 0 || (sight->tree && (sight->words < 1 || (int64_t)sight->words * 32 < max_q || ((uintptr_t)sight->tree & 3)))) {
        e2cu_err("pages_attention: sinks %d, a tree of %d words a row for %d rows", sight ? sight->sinks : 0, sight ? sight->words : 0,
                 max_q);
        return -1;
    }
    const size_t need = e2c_pages_attention_ws_bytes(n, T, max_q, heads, c.KV, c.D, shared);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) {
        e2cu_err("pages_attention: needs %zu bytes of 16-byte aligned workspace, got %zu", need, ws ? ws_bytes : 0);
        return -1;
    }
    return e2cu_launch(e2c_pages_attention(&c, q_type, q, ldq, seqs, q_start, n, T, max_q, heads, shared, sight->causal, sight->window,
                                           sight->sinks, sight->tree, sight->words, scale, out, ldo, lse, ws, ws_bytes, e2cu_status(),
                                           stream),
                       "pages_attention");
}
