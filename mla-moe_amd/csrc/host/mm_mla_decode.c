/* mm_mla_decode.c -- forms of the absorbed decode attention for serving (host
 * side): sequences that share a prefix, and sliding windows with sinks.
 *
 * Both are the chain of mm_mla_absorbed_decode_dev (mm_mla.c) with other keys:
 * absorbed queries, chunk partials (maximum, sum, unnormalised context) per
 * (row, 16 heads, chunk), their merge, W_UV.  A prefix's partials and those of
 * a sequence's own keys stand in one list, so one merge joins them.
 */
#include "mm_internal.h"

static size_t al256(size_t b) { return (b + 255) & ~(size_t)255; }

#define MM_DECODE_ROWS (1 << 20)   /* rows of one call at most */

/* A call's rows, how their keys are cut, and where its workspace holds what. */
typedef struct {
    int R, HG;
    int shared;                    /* the prefix by mm_mla_attn_shared */
    int pchunk, np;                /* the shared prefix: keys per chunk, chunks */
    int ochunk, no;                /* each row's own keys */
    int direct;                    /* one chunk: its blocks write clat, no merge */
    int G;                         /* rows whose partials are held at once */
    size_t o_qhl, o_clat, o_ml, o_po, bytes;
} decode_plan;

/* Keys per chunk: as decode_rows (mm_mla.c), MM_MLA_CHUNK halved while the
 * grid has fewer than MM_MLA_MIN_BLOCKS blocks and a row at most 64 chunks;
 * doubled where a row would have more than maxch. */
static int chunk_keys(size_t blocks, int keys, int maxch) {
    int chunk = MM_MLA_CHUNK;
    while (chunk > 16 * MM_MLA_AW && blocks * ((keys + chunk - 1) / chunk) < MM_MLA_MIN_BLOCKS &&
           (keys + chunk / 2 - 1) / (chunk / 2) <= 64)
        chunk /= 2;
    if (chunk < MM_MLA_CHUNK && keys > chunk && keys <= chunk + chunk / 2) chunk *= 2;
    while ((keys + chunk - 1) / chunk > maxch) chunk *= 2;
    return chunk;
}

/* Keys per chunk of mm_mla_attn_shared: one block per CU, so rounds of the CUs
 * times a block's tiles (about 1.2 us of 32 keys) and its fixed part (about 7
 * us: queries, first loads, two tiles until all roles run, its output), and 4
 * KB per row and chunk of partials written and read back (4 TB/s). */
static int shared_chunk_keys(int M, int keys) {
    const int nrt = (M + 63) / 64, tiles = (keys + 31) / 32;
    double best = 0.0;
    int ct = tiles;
    for (int n = 1; n <= tiles && n <= MM_MLA_MAXCH / 2; n++) {
        const int t = (tiles + n - 1) / n, nch = (tiles + t - 1) / t;
        const double rounds = (double)(((size_t)nrt * nch + 255) / 256);
        const double us = rounds * (1.2 * t + 7.0) + (double)M * nch * 4096.0 / 4e6;
        if (n == 1 || us < best) {
            best = us;
            ct = t;
        }
    }
    return 32 * ct;
}

static void plan_decode(const mm_ctx *c, int R, int prefix, int keys, decode_plan *p) {
    const int NH = c->mla.n_heads;
    p->R = R;
    p->HG = (NH + 15) / 16;
    p->ochunk = keys > 0 ? chunk_keys((size_t)R * p->HG, keys, MM_MLA_MAXCH / 2) : 0;
    p->no = keys > 0 ? (keys + p->ochunk - 1) / p->ochunk : 0;
    p->shared = prefix > 0 && R * (size_t)NH >= (size_t)c->mla_shared_min;
    p->pchunk = p->shared ? shared_chunk_keys(R * NH, prefix)
                : prefix > 0 ? chunk_keys((size_t)R * p->HG, prefix, MM_MLA_MAXCH / 2) : 0;
    p->np = prefix > 0 ? (prefix + p->pchunk - 1) / p->pchunk : 0;
    p->direct = p->np == 0 && p->no == 1;
    const size_t row = p->direct ? 0 : (size_t)p->HG * (p->np + p->no) * (16 * MM_MLA_KVL + 32) * 4;
    p->G = R;
    if (row && (size_t)R * row > c->mla_part_max) p->G = c->mla_part_max / row > 0 ? (int)(c->mla_part_max / row) : 1;
    p->o_qhl = 0;
    p->o_clat = al256((size_t)R * NH * 2 * MM_MLA_KVL * 2);
    p->o_ml = p->o_clat + al256((size_t)R * NH * MM_MLA_KVL * 4);
    const size_t parts = p->direct ? 0 : (size_t)p->G * p->HG * (p->np + p->no);
    p->o_po = p->o_ml + al256(parts * 32 * 4);
    p->bytes = p->o_po + al256(parts * 16 * MM_MLA_KVL * 4);
}

/* The rows' keys: a prefix all of them read, and / or windows of their sequences'
 * caches, `rows` rows per sequence (one row and a window of kv_len: the cache). */
typedef struct {
    const uint16_t *prefix;
    int prefix_len;
    const uint16_t *cache;
    int seq_stride;
    const int32_t *kv_lens;
    int kv_len;                    /* the longest cache */
    int rows, sinks, window;
} decode_keys;

static int decode_run(mm_ctx *c, int layer, const decode_plan *p, const float *q, const decode_keys *k,
                      float *ctx_out, char *ws) {
    const mm_mla_config *g = &c->mla;
    const int NH = g->n_heads, QKN = g->qk_nope_head_dim, R = p->R;
    uint16_t *qhl = (uint16_t *)(ws + p->o_qhl);
    float *clat = (float *)(ws + p->o_clat), *ml = (float *)(ws + p->o_ml), *po = (float *)(ws + p->o_po);
    const uint16_t *kv_b = c->mla_kvb[layer];
    mm_mla_qprep_args qa = {q, kv_b + (size_t)NH * (QKN + g->v_head_dim) * MM_MLA_KVL, NULL, qhl, R, NH, QKN};
    const int wide = R >= MM_MLA_WIDE_B;
    const unsigned rt = (unsigned)((R + 31) / 32);
    int st = mm_launch(c, wide ? K_MLA_QPREP_W : K_MLA_QPREP, MM_MLA_KVL / (wide ? 64 * MM_MLA_WIDE_S : 64),
                       (unsigned)NH, rt, 256, 0, &qa);
    if (st) return st;
    const int nch = p->np + p->no;
    const size_t alds = (size_t)MM_MLA_AW * 2 * MM_MLA_TILE_B;
    mm_mla_combine_args ca = {ml, po, kv_b, NULL, 0, ctx_out, clat, NULL, 0, R, NH, QKN, g->v_head_dim,
                              p->HG, nch, NULL};
    for (int r0 = 0; r0 < R; r0 += p->G) {
        const int n = R - r0 < p->G ? R - r0 : p->G;
        const size_t h0 = (size_t)r0 * NH;
        mm_mla_attn_args a = {qhl + h0 * 2 * MM_MLA_KVL, q + h0 * (QKN + MM_MLA_QKR), NULL, NULL, 0, 0,
                              g->softmax_scale, ml, po, NULL, 0, NH, p->HG, 0, QKN, 0, NULL,
                              p->direct ? clat + h0 * MM_MLA_KVL : NULL, n, nch, 1, 0, 0, 0};
        if (p->shared) {
            const int M = n * NH;
            mm_mla_shared_args s = {a.qhl, a.q, k->prefix, g->softmax_scale, ml, po, M, NH, p->HG, QKN,
                                    k->prefix_len, p->pchunk, p->np, nch};
            const unsigned nt = (unsigned)((M + 63) / 64) * (unsigned)p->np;
            if ((st = mm_launch(c, K_MLA_ATTN_SHARED, 8 * ((nt + 7) / 8), 1, 1, 512, MM_MLA_SH_LDS, &s))) return st;
        } else if (p->np) {                           /* every row reads sequence 0 */
            a.cache = k->prefix;
            a.kv_len = k->prefix_len;
            a.nchunks = p->np;
            a.chunk = p->pchunk;
            const unsigned nt = (unsigned)n * (unsigned)p->HG * (unsigned)p->np;
            if ((st = mm_launch(c, K_MLA_ATTN, 8 * ((nt + 7) / 8), 1, 1, 64 * MM_MLA_AW, alds, &a))) return st;
        }
        if (p->no) {
            a.cache = k->cache;
            a.seq_stride = k->seq_stride;
            a.kv_lens = k->kv_lens;
            a.kv_len = k->kv_len;
            a.nchunks = p->no;
            a.chunk = p->ochunk;
            a.rows = k->rows;
            a.sinks = k->sinks;
            a.window = k->window;
            a.row0 = r0;
            a.part_ml = ml + (size_t)p->np * 32;
            a.part_o = po + (size_t)p->np * 16 * MM_MLA_KVL;
            const unsigned nt = (unsigned)n * (unsigned)p->HG * (unsigned)p->no;
            if ((st = mm_launch(c, K_MLA_ATTN_WINDOW, 8 * ((nt + 7) / 8), 1, 1, 64 * MM_MLA_AW, alds, &a))) return st;
        }
        if (!p->direct) {
            mm_mla_combine_args cg = ca;
            cg.clat = clat + h0 * MM_MLA_KVL;
            cg.B = n;
            const unsigned z = (size_t)NH * R < 128 ? MM_MLA_KVL / 128 : 1;
            if ((st = mm_launch(c, K_MLA_COMBINE_E, (unsigned)NH, (unsigned)n, z, 256, 0, &cg))) return st;
        }
    }
    const int vt = wide ? 16 * MM_MLA_WIDE_S : 16;
    return mm_launch(c, wide ? K_MLA_UV_W : K_MLA_UV, (unsigned)((g->v_head_dim + vt - 1) / vt), (unsigned)NH, rt,
                     256, 0, &ca);
}

/* ---- a prefix that every sequence shares ------------------------------------- */

static int prefix_check(const mm_ctx *c, const char *name, int B, int prefix_len, int kv_len) {
    if (!c) return mm_fail(MM_ERR_INVALID, "%s: NULL context", name);
    if (!c->mla_ready) return mm_fail(MM_ERR_STATE, "%s: call mm_mla_init first", name);
    if (B < 0 || prefix_len < 0 || kv_len < 0) return mm_fail(MM_ERR_INVALID, "%s: negative size", name);
    if (B > MM_DECODE_ROWS || prefix_len > MM_MAX_KV_LEN || kv_len > MM_MAX_KV_LEN)
        return mm_fail(MM_ERR_UNSUPPORTED, "%s: B <= %d, prefix_len and kv_len <= %d", name, MM_DECODE_ROWS, MM_MAX_KV_LEN);
    return MM_OK;
}

int mm_mla_prefix_decode_workspace(mm_ctx *c, int B, int prefix_len, int kv_len, size_t *bytes) {
    if (!bytes) return mm_fail(MM_ERR_INVALID, "mm_mla_prefix_decode_workspace: NULL argument");
    *bytes = 0;
    const int st = prefix_check(c, "mm_mla_prefix_decode_workspace", B, prefix_len, kv_len);
    if (st || B == 0) return st;
    decode_plan p;
    plan_decode(c, B, prefix_len, kv_len, &p);
    *bytes = p.bytes;
    return MM_OK;
}

int mm_mla_prefix_decode_dev(mm_ctx *c, int layer, int B, const float *q, const uint16_t *prefix,
                             int prefix_len, const uint16_t *cache, int seq_stride,
                             const int32_t *kv_lens, int kv_len, float *ctx_out, void *ws,
                             size_t ws_bytes) {
    static const char name[] = "mm_mla_prefix_decode_dev";
    int st = prefix_check(c, name, B, prefix_len, kv_len);
    if (st) return st;
    if (layer < 0 || layer >= c->mla_layers || !c->mla_kvb[layer])
        return mm_fail(MM_ERR_STATE, "%s: layer %d not loaded", name, layer);
    if (B == 0) return MM_OK;
    if (!q || !ctx_out || (prefix_len && !prefix) || (kv_len && !cache))
        return mm_fail(MM_ERR_INVALID, "%s: NULL argument", name);
    if (seq_stride < kv_len) return mm_fail(MM_ERR_INVALID, "%s: need kv_len <= seq_stride", name);
    if ((prefix_len && (uintptr_t)prefix % 16) || (kv_len && (uintptr_t)cache % 16) || (uintptr_t)q % 16)
        return mm_fail(MM_ERR_INVALID, "%s: q, prefix and cache must be 16-byte aligned", name);
    if ((st = mm_set_device(c))) return st;
    decode_plan p;
    plan_decode(c, B, prefix_len, kv_len, &p);
    char *w;
    if ((st = mm_call_workspace(c, name, ws, ws_bytes, p.bytes, (void **)&w))) return st;
    const decode_keys k = {prefix, prefix_len, cache, seq_stride, kv_lens, kv_len, 1, 0, kv_len};
    return decode_run(c, layer, &p, q, &k, ctx_out, w);
}

/* ---- sliding windows with sinks ------------------------------------------------ */

static int window_check(const mm_ctx *c, const char *name, int B, int rows, int kv_len, int sinks, int window) {
    if (!c) return mm_fail(MM_ERR_INVALID, "%s: NULL context", name);
    if (!c->mla_ready) return mm_fail(MM_ERR_STATE, "%s: call mm_mla_init first", name);
    if (B < 0 || rows < 1 || kv_len < 1 || sinks < 0 || window < 1)
        return mm_fail(MM_ERR_INVALID, "%s: need B, sinks >= 0 and rows, kv_len, window >= 1", name);
    if ((size_t)B * rows > MM_DECODE_ROWS || kv_len > MM_MAX_KV_LEN)
        return mm_fail(MM_ERR_UNSUPPORTED, "%s: B * rows <= %d, kv_len <= %d", name, MM_DECODE_ROWS, MM_MAX_KV_LEN);
    return MM_OK;
}

/* Keys that a row sees at most (both no longer than the cache: no overflow). */
static int window_keys(int kv_len, int *sinks, int *window) {
    if (*sinks > kv_len) *sinks = kv_len;
    if (*window > kv_len) *window = kv_len;
    return *sinks + *window < kv_len ? *sinks + *window : kv_len;
}

int mm_mla_window_decode_workspace(mm_ctx *c, int B, int rows, int kv_len, int sinks, int window, size_t *bytes) {
    if (!bytes) return mm_fail(MM_ERR_INVALID, "mm_mla_window_decode_workspace: NULL argument");
    *bytes = 0;
    const int st = window_check(c, "mm_mla_window_decode_workspace", B, rows, kv_len, sinks, window);
    if (st || B == 0) return st;
    decode_plan p;
    plan_decode(c, B * rows, 0, window_keys(kv_len, &sinks, &window), &p);
    *bytes = p.bytes;
    return MM_OK;
}

int mm_mla_window_decode_dev(mm_ctx *c, int layer, int B, int rows, const float *q, const uint16_t *cache,
                             int seq_stride, const int32_t *kv_lens, int kv_len, int sinks, int window,
                             float *ctx_out, void *ws, size_t ws_bytes) {
    static const char name[] = "mm_mla_window_decode_dev";
    int st = window_check(c, name, B, rows, kv_len, sinks, window);
    if (st) return st;
    if (layer < 0 || layer >= c->mla_layers || !c->mla_kvb[layer])
        return mm_fail(MM_ERR_STATE, "%s: layer %d not loaded", name, layer);
    if (B == 0) return MM_OK;
    if (!q || !cache || !ctx_out) return mm_fail(MM_ERR_INVALID, "%s: NULL argument", name);
    if (seq_stride < kv_len) return mm_fail(MM_ERR_INVALID, "%s: need kv_len <= seq_stride", name);
    if ((uintptr_t)cache % 16 || (uintptr_t)q % 16)
        return mm_fail(MM_ERR_INVALID, "%s: q and cache must be 16-byte aligned", name);
    if ((st = mm_set_device(c))) return st;
    const int keys = window_keys(kv_len, &sinks, &window);
    decode_plan p;
    plan_decode(c, B * rows, 0, keys, &p);
    char *w;
    if ((st = mm_call_workspace(c, name, ws, ws_bytes, p.bytes, (void **)&w))) return st;
    const decode_keys k = {NULL, 0, cache, seq_stride, kv_lens, kv_len, rows, sinks, window};
    return decode_run(c, layer, &p, q, &k, ctx_out, w);
}
