/* mm_mla_decode.c -- forms of the absorbed decode attention for serving (host
 * side): sequences that share a prefix, and sliding windows with sinks.
 *
 * Both are the chain of mm_mla_absorbed_decode_dev (mm_mla.c) with other keys:
 * absorbed queries, attention in 64-row tiles (mla_tiles.h) that leaves partials
 * (maximum, sum, unnormalised context) per (row, 16 heads, chunk), their merge,
 * W_UV.  A prefix's partials and those of a sequence's own keys stand in one
 * list, so one merge joins them.
 */
#include "mm_internal.h"

static size_t al256(size_t b) { return (b + 255) & ~(size_t)255; }

#define MM_DECODE_ROWS (1 << 20)   /* rows of one call at most */

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
    int own;                       /* keys of its own that a row (64 rows together) sees at most */
} decode_keys;

/* A call's rows, how their keys are cut, and where its workspace holds what. */
typedef struct {
    int R, HG;
    int pchunk, np;                /* the prefix: keys per chunk, chunks */
    int ochunk, no;                /* own keys */
    int G;                         /* rows whose queries and partials are held at once */
    size_t o_ml, o_po, bytes;      /* (the queries at 0) */
} decode_plan;

/* The chunks, one block per CU: us of a block with t tiles of 32
 * keys over 64 (or up to 32) rows -- queries, first loads, two tiles until all
 * roles run, its output --, and of the partials written and read back (4 KB per
 * row and chunk at 4 TB/s). */
static double tiles_us(int t, int nrows) { return (nrows > 32 ? 1.7 : 1.1) * t + 9.0; }

static void tiles_chunks(int R, int NH, int rows, int prefix, int own, decode_plan *p) {
    const size_t nrt = ((size_t)R * NH + 63) / 64, ort = (size_t)(R / rows) * ((rows * NH + 63) / 64);
    const int pt = (prefix + 31) / 32, ot = (own + 31) / 32, most = MM_MLA_MAXCH / 2;
    double best = -1.0;
    for (int n = 1; n <= (pt > 0 ? pt : ot) && n <= most; n++) {
        int t, u, np = 0, no = 0;
        if (pt > 0) {
            /* own chunks no longer than the prefix's, so that they fill in beside:
             * right where the prefix is the longer part; behind a shorter one they
             * are finer than is best (64 sequences of 16 heads, 64 + 2,048 keys 87
             * us; 2,112 of their own without a prefix 49) */
            t = (pt + n - 1) / n;
            u = t < ot ? t : ot;
        } else {
            t = 0;
            u = (ot + n - 1) / n;
        }
        if (u > 0 && (ot + u - 1) / u > most) u = (ot + most - 1) / most;
        if (t > 0) np = (pt + t - 1) / t;
        if (u > 0) no = (ot + u - 1) / u;
        const double lp = np ? tiles_us(t, 64) : 0.0, lo = no ? tiles_us(u, rows * NH) : 0.0;
        /* the prefix's blocks in rounds of the CUs, the own ones into what the
         * last round leaves, then in rounds */
        const size_t bp = nrt * np, bo = ort * no, q = bp / 256, r = bp % 256;
        size_t room = 0;
        if (r && bo) room = (256 - r) * (lp >= lo ? (size_t)(lp / lo) : 0);
        const size_t rest = bo > room ? bo - room : 0;
        double us = (double)(q + (r > 0)) * lp + (double)((rest + 255) / 256) * lo;
        us += (double)R * NH * (np + no) * 4096.0 / 4e6;
        if (best < 0.0 || us < best) {
            best = us;
            p->pchunk = 32 * t;
            p->np = np;
            p->ochunk = 32 * u;
            p->no = no;
        }
    }
}

static void plan_decode(const mm_ctx *c, int R, const decode_keys *k, decode_plan *p) {
    const int NH = c->mla.n_heads;
    p->R = R;
    p->HG = (NH + 15) / 16;
    p->pchunk = p->np = p->ochunk = p->no = 0;
    tiles_chunks(R, NH, k->rows, k->prefix_len, k->own, p);
    int unit = 1;                  /* rows that fill whole tiles */
    while ((unit * NH) % 64) unit++;
    const size_t row = (size_t)p->HG * (p->np + p->no) * (16 * MM_MLA_KVL + 32) * 4 +
                       (size_t)NH * (MM_MLA_QF_TILE / 32);
    p->G = R;
    if ((size_t)R * row > c->mla_part_max) {
        const size_t g = c->mla_part_max / row / unit * unit;
        p->G = g > 0 ? (int)g : unit;
        if (p->G > R) p->G = R;
    }
    p->o_ml = ((size_t)p->G * NH + 31) / 32 * MM_MLA_QF_TILE;
    const size_t parts = (size_t)p->G * p->HG * (p->np + p->no);
    p->o_po = p->o_ml + al256(parts * 32 * 4);
    p->bytes = p->o_po + al256(parts * 16 * MM_MLA_KVL * 4);
}

/* Rows r0 .. r0 + n - 1 of the call, whole sequences or part of one: their
 * partials. */
static int attend(mm_ctx *c, const decode_plan *p, const decode_keys *k, const uint16_t *qf, int r0, int n,
                  float *ml, float *po) {
    const mm_mla_config *g = &c->mla;
    const int NH = g->n_heads, M = n * NH, rows = n < k->rows ? n : k->rows, nseq = n / rows;
    mm_mla_tiles_args a = {qf, ml, po, M, NH, p->HG, p->np + p->no,
                           k->prefix, k->prefix_len, p->pchunk, p->np, k->cache, k->kv_lens, k->kv_len, k->seq_stride,
                           r0 / k->rows, nseq, rows, p->ochunk, p->no, k->rows, r0 % k->rows, k->sinks, k->window};
    const unsigned np = (unsigned)((M + 63) / 64) * (unsigned)p->np;
    const unsigned no = (unsigned)nseq * (unsigned)((rows * NH + 63) / 64) * (unsigned)p->no;
    return mm_launch(c, p->np || (k->rows == 1 && k->window >= k->kv_len) ? K_MLA_ATTN_TILES : K_MLA_ATTN_TILES_W,
                     8 * ((np + 7) / 8) + 8 * ((no + 7) / 8), 1, 1, 512, MM_MLA_TL_LDS, &a);
}

static int decode_run(mm_ctx *c, int layer, const decode_plan *p, const float *q, const decode_keys *k,
                      float *ctx_out, char *ws) {
    const mm_mla_config *g = &c->mla;
    const int NH = g->n_heads, QKN = g->qk_nope_head_dim, VHD = g->v_head_dim, R = p->R;
    uint16_t *qf = (uint16_t *)ws;
    float *ml = (float *)(ws + p->o_ml), *po = (float *)(ws + p->o_po);
    const uint16_t *wukT = c->mla_kvb[layer] + (size_t)NH * (QKN + VHD) * MM_MLA_KVL;
    const uint16_t *wuvf = wukT + (size_t)NH * MM_MLA_KVL * QKN;
    int st;
    for (int r0 = 0, n; r0 < R; r0 += n) {
        n = R - r0 < p->G ? R - r0 : p->G;
        if (k->rows > 1 && n < R) {                   /* whole sequences, or within one */
            const int left = k->rows - r0 % k->rows;
            if (r0 % k->rows == 0 && n >= k->rows) n = n / k->rows * k->rows;
            else if (n > left) n = left;
        }
        const size_t h0 = (size_t)r0 * NH;
        mm_mla_qfrag_args qa = {q + h0 * (QKN + MM_MLA_QKR), wukT, qf, n, NH, QKN,
                                g->softmax_scale * 1.44269504088896341f};
        /* by the call's rows, as below (4 positions of 16 heads: 3.4 us, in blocks of
         * eight heads 4.3; 39 of 20: 5.9 both; 48 of 16: 4.9, 4.6) */
        if (R < 48)
            st = mm_launch(c, K_MLA_QFRAG, MM_MLA_KVL / 64 + 1, (unsigned)NH, (unsigned)(n + 31) / 32, 256, 0, &qa);
        else
            st = mm_launch(c, K_MLA_QFRAG_8, MM_MLA_KVL / 32 + 1, (unsigned)(NH + 7) / 8, (unsigned)(n + 15) / 16, 512, 0, &qa);
        if (st) return st;
        if ((st = attend(c, p, k, qf, r0, n, ml, po))) return st;
        /* blocks of the merge: four waves a position each, a column tile each, for
         * few positions (4 of 16 heads, the same inputs every pass: 5.6 us, with
         * eight waves 6.7); eight waves for
         * more, 4 positions per block as long as every CU has at most one block,
         * else 8 (64 positions: 8.1, with four waves 8.6; 39 of 20 heads and 256
         * columns: 7.8, 4 per block 10.7); from 256 positions on 16 per block and a
         * head's columns together (512: 12.9, 8 per block 17.0, with eight waves 13.4) */
        const int ncol = (VHD + 15) / 16, nw = R <= 16 || R >= 256 ? 4 : 8;
        const int split = R >= 256 ? 1 : (ncol + nw - 1) / nw;
        int ppb = R >= 256 ? 16 : 4, wpp = 1;
        if (R > 16 && R < 256 && (size_t)NH * ((R + 3) / 4) * split > 256) ppb = 8;
        while (2 * wpp * R <= nw) wpp *= 2;          /* by the call's rows: the same bits in groups */
        const int rt = (n + ppb - 1) / ppb;
        mm_mla_merge_uv_args ma = {ml, po, wuvf, ctx_out + h0 * VHD, n, NH, p->HG, VHD, p->np + p->no,
                                   ppb, split, wpp};
        const unsigned blocks = (unsigned)NH * (unsigned)rt * (unsigned)split;
        if ((st = mm_launch(c, nw == 4 ? K_MLA_MERGE_UV4 : K_MLA_MERGE_UV8, blocks, 1, 1, 64 * nw, 0, &ma))) return st;
    }
    return MM_OK;
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

static decode_keys prefix_keys(const uint16_t *prefix, int prefix_len, const uint16_t *cache, int seq_stride,
                               const int32_t *kv_lens, int kv_len) {
    const decode_keys k = {prefix, prefix_len, cache, seq_stride, kv_lens, kv_len, 1, 0, kv_len, kv_len};
    return k;
}

int mm_mla_prefix_decode_workspace(mm_ctx *c, int B, int prefix_len, int kv_len, size_t *bytes) {
    if (!bytes) return mm_fail(MM_ERR_INVALID, "mm_mla_prefix_decode_workspace: NULL argument");
    *bytes = 0;
    const int st = prefix_check(c, "mm_mla_prefix_decode_workspace", B, prefix_len, kv_len);
    if (st || B == 0 || prefix_len + kv_len == 0) return st;
    const decode_keys k = prefix_keys(NULL, prefix_len, NULL, kv_len, NULL, kv_len);
    decode_plan p;
    plan_decode(c, B, &k, &p);
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
    if (prefix_len + kv_len == 0) {                   /* no chunk to merge */
        mm_zero32_args za = {(uint32_t *)ctx_out, (uint64_t)B * c->mla.n_heads * c->mla.v_head_dim};
        return mm_launch(c, K_ZERO32, 256, 1, 1, 256, 0, &za);
    }
    const decode_keys k = prefix_keys(prefix, prefix_len, cache, seq_stride, kv_lens, kv_len);
    decode_plan p;
    plan_decode(c, B, &k, &p);
    char *w;
    if ((st = mm_call_workspace(c, name, ws, ws_bytes, p.bytes, (void **)&w))) return st;
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

/* sinks and window no longer than the cache; the keys that the rows of a tile
 * (as many positions as 64 rows touch) see at most. */
static decode_keys window_keys(const mm_ctx *c, int rows, const uint16_t *cache, int seq_stride,
                               const int32_t *kv_lens, int kv_len, int sinks, int window) {
    if (sinks > kv_len) sinks = kv_len;
    if (window > kv_len) window = kv_len;
    int span = 64 / c->mla.n_heads + 2;
    if (span > rows) span = rows;
    const int own = sinks + window + span - 1;
    const decode_keys k = {NULL, 0, cache, seq_stride, kv_lens, kv_len, rows, sinks, window, own < kv_len ? own : kv_len};
    return k;
}

int mm_mla_window_decode_workspace(mm_ctx *c, int B, int rows, int kv_len, int sinks, int window, size_t *bytes) {
    if (!bytes) return mm_fail(MM_ERR_INVALID, "mm_mla_window_decode_workspace: NULL argument");
    *bytes = 0;
    const int st = window_check(c, "mm_mla_window_decode_workspace", B, rows, kv_len, sinks, window);
    if (st || B == 0) return st;
    const decode_keys k = window_keys(c, rows, NULL, kv_len, NULL, kv_len, sinks, window);
    decode_plan p;
    plan_decode(c, B * rows, &k, &p);
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
    const decode_keys k = window_keys(c, rows, cache, seq_stride, kv_lens, kv_len, sinks, window);
    decode_plan p;
    plan_decode(c, B * rows, &k, &p);
    char *w;
    if ((st = mm_call_workspace(c, name, ws, ws_bytes, p.bytes, (void **)&w))) return st;
    return decode_run(c, layer, &p, q, &k, ctx_out, w);
}
