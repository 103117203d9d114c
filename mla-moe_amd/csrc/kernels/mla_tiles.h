/* mla_tiles.h -- absorbed MLA attention of many rows over common keys (part of
 * mla.hip): the prefix that a decode batch shares with each sequence's own keys,
 * and the rows of a prompt's chunk through a sliding window.
 *
 * A row is one (position, head).  It costs 1,088 products a key, twice over since
 * the fp32 query and the probabilities travel as bf16 pairs.  mm_mla_attn keeps 16
 * rows (one position's heads) per wave, so that each position reads its keys for
 * itself and 16 x 16 tiles are fed from LDS once per 16 rows.  Here a block takes
 * 64 rows over a chunk of their keys on 32 x 32 tiles, one block per CU, its eight
 * waves in three roles (each SIMD holds one of the first four and one of the
 * last), each one 32-key tile behind the other:
 *   waves 0, 1   scores of tile t + 2 over latents 0..287 (32 rows each)
 *   waves 2, 3   scores of tile t + 1 over latents 288..575, added to the former;
 *                softmax; the probabilities as bf16 pairs to LDS
 *   waves 4..7   O += P V of tile t, 64 rows x 160 (4, 5) or 96 (6, 7) latent
 *                columns; and the loads of the tiles to come
 * A score wave keeps its 32 rows' queries over its half of the latents (144
 * registers), an output wave up to 64 x 160 of O (160 registers): neither would
 * fit beside the other, and the softmax of one tile runs beside the products of
 * the others.  One barrier per tile.  Waves 2 and 3 do the softmax, so the output
 * waves on their SIMDs have fewer columns (128 each: 31 us where this takes 29, 64
 * rows of 16 heads over 4,096 keys).
 *
 * The matrix cores bound it: 2,176 cycles of products a tile on each of four
 * SIMDs on average, 64 rows of 16 heads over 32,768 keys 132 to 140 us in all, 1.05
 * to 1.11 PFLOP/s of pair products (a library's product of 8,192^3: 1.21).
 *
 * LDS, per tile of 32 keys: latents 0..287 (576 bytes a row, four tiles of
 * them), 288..511 (448 bytes, three), k_pe (128 bytes, two): a part lives until
 * its last reader.  Rows are 16-byte pieces, piece p of row r in slot p with its
 * low two bits exclusive-ored with r / 4: a wave's reads (32 rows of one piece, or
 * four rows of a 32-column stretch, transposing) then fall on all banks, since
 * both row lengths are odd multiples of 64 bytes.  Rows past the keys are
 * beyond the buffer's range: zeros, no read; their scores are masked.
 *
 * Key order inside a 16-key step of P and V: half h of the lanes holds keys 4 h
 * + {0..3, 8..11}, the keys of its registers after the score product. */
#define TL_R0 18432                /* bytes of one tile: latents 0..287 */
#define TL_R1 14336                /* latents 288..511 */
#define TL_KP 4096                 /* k_pe */
#define TL_O1 (4 * TL_R0)
#define TL_OK (TL_O1 + 3 * TL_R1)
#define TL_OP (TL_OK + 2 * TL_KP)  /* P: two tiles of 64 rows x 32 keys, hi then lo */
#define TL_OX (TL_OP + 2 * 8192)   /* partial scores: two tiles of 64 x 32 floats */
#define TL_OF (TL_OX + 2 * 8192)   /* rescaling factors: two tiles of 64 floats */
#define TL_OG (TL_OF + 2 * 256)    /* [tile % 2][row half]: whether there are some; keys that are not finite */
#define TL_OT (TL_OG + 32)         /* 64 rows' places in the partials */
static_assert(TL_OT + 256 <= MM_MLA_TL_LDS && MM_MLA_TL_LDS <= 163840, "LDS of a block");
typedef __attribute__((address_space(3))) s16x4 *lds_s4;
typedef __attribute__((address_space(3))) i32x4 *lds_w4;
typedef __attribute__((address_space(3))) f32x4 *lds_f4;
typedef __attribute__((address_space(3))) float *lds_f;
typedef __attribute__((address_space(3))) int *lds_i;

/* LDS accesses done, then the block's barrier; loads into LDS stay in flight. */
__device__ __forceinline__ void tl_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/* acc += K Qhi^T + K Qlo^T over 18 steps of 16 latents, K operands at LDS
 * addresses addr(s), three steps' reads ahead of the products (without the scheduling
 * barriers each read sat right before its products). */
template <class Addr>
__device__ __forceinline__ void tl_scores(const i32x4 (&qh)[18], const i32x4 (&ql)[18], f32x16 &acc, Addr addr) {
    i32x4 k[2][3];
#pragma unroll
    for (int i = 0; i < 3; i++) k[0][i] = *(lds_w4)(uintptr_t)addr(i);
#pragma unroll
    for (int b = 0; b < 6; b++) {
        __builtin_amdgcn_sched_barrier(0);
        if (b < 5) {
#pragma unroll
            for (int i = 0; i < 3; i++) k[(b + 1) & 1][i] = *(lds_w4)(uintptr_t)addr(3 * (b + 1) + i);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 3; i++) {
            acc = mfma32(k[b & 1][i], qh[3 * b + i], acc);
            acc = mfma32(k[b & 1][i], ql[3 * b + i], acc);
        }
    }
}

/* Which of a tile's 32 keys hold a value that is not finite (bit r: row r of its
 * three parts in LDS): lane l has half l / 32 of row l % 32, in slots of 16 bytes
 * in whatever order. */
__device__ __forceinline__ uint32_t tl_not_finite(uint32_t r0, uint32_t r1, uint32_t kp) {
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
    uint32_t any = 0;
    auto look = [&](uint32_t p, int n) {
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const i32x4 x = *(lds_w4)(uintptr_t)(p + 16 * i);
#pragma unroll
            for (int k = 0; k < 4; k++) any |= nonfinite2((uint32_t)x[k]);
        }
    };
    look(r0 + (uint32_t)(row * 576 + half * 288), 18);
    look(r1 + (uint32_t)(row * 448 + half * 224), 14);
    look(kp + (uint32_t)(row * 128 + half * 64), 4);
    const uint64_t m = __builtin_amdgcn_ballot_w64(any != 0);
    return (uint32_t)m | (uint32_t)(m >> 32);
}

/* A block's rows and keys. */
struct tl_job {
    const uint16_t *keys;          /* first of the chunk's keys; WIN: the sequence's cache */
    int row0, nrows;               /* flat rows (position, head) of the launch */
    int chunk;                     /* its place among a row's partials */
    int nk;                        /* keys of the chunk */
    /* WIN: the chunk's key v is key v0 + v of the tile's list: the sinks, then
     * from `sinks` on shifted to where the first row's window begins */
    int v0, len, shift, first_row, pos0;   /* pos0: position of the sequence's row 0 in this launch */
};

/* WIN: key of list entry v */
__device__ __forceinline__ int tl_key(const mm_mla_tiles_args &a, const tl_job &j, int v) {
    return v + (v >= a.sinks ? j.shift : 0);
}

template <bool WIN>
__device__ __forceinline__ bool tl_find(const mm_mla_tiles_args &a, tl_job &j) {
    /* both lists in eighths, one per XCD, neighbours (which read the same keys)
     * from one L2: the prefix's blocks chunk by chunk, then the sequences' own */
    const int nrt = (a.M + 63) / 64, nsh = nrt * a.nchunks, psh = (nsh + 7) / 8;
    int i = (int)blockIdx.x;
    if (!WIN && i < 8 * psh) {
        const int trip = i % 8 * psh + i / 8;
        if (trip >= nsh) return false;
        j.chunk = trip / nrt;
        j.row0 = trip % nrt * 64;
        j.nrows = min(64, a.M - j.row0);
        const int k0 = j.chunk * a.chunk;
        j.nk = min(a.chunk, a.nkeys - k0);
        j.keys = a.keys + (size_t)k0 * KVD;
        return true;
    }
    i -= WIN ? 0 : 8 * psh;
    const int rn = a.rows * a.NH, nt = (rn + 63) / 64, nown = a.nseq * nt * a.ochunks, po = (nown + 7) / 8;
    const int trip = i % 8 * po + i / 8;
    if (i >= 8 * po || trip >= nown) return false;
    const int c = trip % a.ochunks, tile = trip / a.ochunks % nt, s = trip / (a.ochunks * nt);
    const int seq = a.seq0 + s;
    const int L = max(min(a.kv_lens ? a.kv_lens[seq] : a.kv_len, a.kv_len), 0);
    j.first_row = 64 * tile;
    j.nrows = min(64, rn - j.first_row);
    j.row0 = s * rn + j.first_row;
    j.chunk = a.nchunks + c;
    j.keys = a.cache + (size_t)seq * a.seq_stride * KVD;
    j.v0 = c * a.ochunk;
    int n = L;
    if (WIN) {
        j.len = L;
        j.pos0 = L - a.all_rows + a.roff;
        const int pa = j.pos0 + j.first_row / a.NH, pb = j.pos0 + (j.first_row + j.nrows - 1) / a.NH;
        const int lo = max(pa - a.window + 1, 0);      /* the first row's window */
        j.shift = lo > a.sinks ? lo - a.sinks : 0;
        n = max(pb + 1 - j.shift, 0);
    } else {
        j.keys += (size_t)min(j.v0, L) * KVD;
    }
    j.nk = min(max(n - j.v0, 0), a.ochunk);
    return true;
}

template <bool WIN>
__device__ __forceinline__ void tl_block(const mm_mla_tiles_args &a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t slds[];
    const uint32_t lds0 = lds_addr(slds);
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, hi = lane >> 5;
    tl_job j;
    if (!tl_find<WIN>(a, j)) return;
    const int nt = (j.nk + 31) / 32;
    const bool two = j.nrows > 32;                     /* rows in both halves */
    if (tid < 64) {                                    /* row (b, h): partial ((b HG + h / 16) pchunks + chunk), line h % 16 */
        const int r = j.row0 + min(tid, j.nrows - 1), b = r / a.NH, h = r - b * a.NH;
        ((lds_i)(uintptr_t)(lds0 + TL_OT))[tid] = ((b * a.HG + (h >> 4)) * a.pchunks + j.chunk) * 16 + (h & 15);
    }

    if (w >= 4) {
        /* ---- O += P V, and the loads ---- */
        const int bw = w - 4, cb = bw < 2 ? 5 * bw : 10 + 3 * (bw - 2);   /* its first column tile of the 16 */
        const rsrc_t rk = raw_rsrc(j.keys, (uint32_t)(WIN ? j.len : j.nk) * KVD * 2);
        /* this wave's nine of a tile's 36 1-KB loads: LDS piece x (16 bytes) of
         * the part is row x / pieces-per-row, slot x % it */
        uint32_t so[9], dl[9];
        int kr[9];                                     /* WIN: the row */
#pragma unroll
        for (int i = 0; i < 9; i++) {
            const bool r0 = i < 4 || (i == 4 && bw < 2);
            const int u = i < 4 ? bw + 4 * i : i == 4 ? (bw < 2 ? 16 + bw : 10 + bw) : i < 8 ? bw + 4 * (i - 5) : bw;
            const int x = 64 * u + lane;
            int r, o;
            if (i == 8) {
                r = x >> 3;
                o = KVL * 2 + 16 * ((x & 7) ^ ((r >> 1) & 7));
            } else {
                const int ppr = r0 ? 36 : 28;
                r = x / ppr;
                const int s = x - r * ppr;
                o = (r0 ? 0 : 576) + 16 * ((s & ~3) | ((s ^ (r >> 2)) & 3));
            }
            so[i] = (uint32_t)(o + (WIN ? 0 : r * KVD * 2));
            kr[i] = r;
            dl[i] = lds0 + (uint32_t)(1024 * u) + (i == 8 ? TL_OK : r0 ? 0 : TL_O1);
        }
        auto load = [&](int i, int t, uint32_t d) {
            uint32_t o;
            if (WIN) {
                const int v = 32 * t + kr[i];          /* past the chunk: out of range */
                o = v < j.nk ? (uint32_t)tl_key(a, j, j.v0 + v) * (KVD * 2) + so[i] : 0xFFFFF000u;
            } else {
                o = so[i] + (uint32_t)t * (32 * KVD * 2);
            }
            lds_dma16_buf(o, rk, dl[i] + d);
        };
        /* latents 0..287 of a tile; 288..575 */
        auto issue0 = [&](int t) {
            const uint32_t d = (uint32_t)(t & 3) * TL_R0;
#pragma unroll
            for (int i = 0; i < 4; i++) load(i, t, d);
            if (bw < 2) load(4, t, d);
        };
        auto issue1 = [&](int t) {
            const uint32_t d = (uint32_t)(t % 3) * TL_R1;
            if (bw >= 2) load(4, t, d);
#pragma unroll
            for (int i = 5; i < 8; i++) load(i, t, d);
            load(8, t, (uint32_t)(t & 1) * TL_KP);
        };
        if (nt > 0) issue0(0);                         /* 4 or 5 loads; with issue1 9 in all */
        if (nt > 1) issue0(1);
        if (nt > 0) issue1(0);
        if (nt > 2) issue0(2);
        if (nt > 1) issue1(1);

        /* transposing reads: lane i of 16-lane group g supplies row 4 (4 s + 2 e
         * + g / 2) + i / 4, 4 columns from 16 (g % 2) + 4 (i % 4) of column tile ct */
        const int i16 = lane & 15, gq = lane >> 4, h = gq >> 1;
        uint32_t v0[2], v1[2];                         /* [e], of latents 0..287 and 288.., column tile 0, s = 0 */
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * e + 4 * h + (i16 >> 2);
            const int low = (2 * (gq & 1) + ((i16 >> 1) & 1)) ^ (2 * e + h);
            v0[e] = lds0 + (uint32_t)(r * 576 + 16 * low + 8 * (i16 & 1));
            v1[e] = lds0 + TL_O1 + (uint32_t)(r * 448 + 16 * low + 8 * (i16 & 1));
        }
        const uint32_t pa = lds0 + TL_OP + (uint32_t)(c32 * 64 + 16 * (hi ^ ((c32 >> 2) & 3)));   /* piece 2 s + hi: s flips bit 1 */
        auto run = [&](auto rtc, auto ctc) {
            constexpr int RT = decltype(rtc)::value, CT = decltype(ctc)::value;   /* row tiles, column tiles */
            f32x16 O[RT][CT] = {};
            for (int t = 0; t < nt; t++) {
                if (t + 3 < nt) issue0(t + 3);
                if (t + 2 < nt) issue1(t + 2);
                const uint32_t d0 = (uint32_t)(t & 3) * TL_R0, d1 = (uint32_t)(t % 3) * TL_R1;
                const uint32_t po = (uint32_t)(t & 1) * 8192;
                const i32x4 flags = *(lds_w4)(uintptr_t)(lds0 + TL_OG + 16 * (t & 1));
                if (WIN) {
                    /* a key that is not finite meets probabilities of zero (rows
                     * that do not see it; those that do have no finite sum): its
                     * values, of which this wave alone reads these columns, are
                     * zeroed */
                    uint32_t bad = (uint32_t)__builtin_amdgcn_readfirstlane(flags[2] | (RT > 1 ? flags[3] : 0));
                    while (bad) {
                        const int r = __builtin_ctz(bad), p = 4 * cb + lane;
                        bad &= bad - 1;
                        if (lane < 4 * CT) {
                            const uint32_t o = p < 36 ? d0 + r * 576 + 16 * ((p & ~3) | ((p ^ (r >> 2)) & 3))
                                                      : TL_O1 + d1 + r * 448 + 16 * (((p - 36) & ~3) | ((p ^ (r >> 2)) & 3));
                            *(lds_w4)(uintptr_t)(lds0 + o) = (i32x4){0, 0, 0, 0};
                        }
                        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    if (__builtin_amdgcn_readfirstlane(flags[rt])) {   /* some row's maximum moved: its factor */
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            const f32x4 f = *(lds_f4)(uintptr_t)(lds0 + TL_OF + (uint32_t)((t & 1) * 256 + 4 * (32 * rt + 8 * g + 4 * hi)));
#pragma unroll
                            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                                for (int i = 0; i < 4; i++) O[rt][ct][4 * g + i] *= f[i];
                        }
                    }
                }
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    i32x4 ph[RT], pl[RT], v[CT];
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const uint32_t p = (pa ^ (uint32_t)(32 * s)) + po + 2048 * rt;
                        ph[rt] = *(lds_w4)(uintptr_t)p;
                        pl[rt] = *(lds_w4)(uintptr_t)(p + 4096);
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        const int col = cb + ct;       /* 32-column tile of the 16 */
                        const uint32_t o = col < 9 ? d0 + 64 * col + 16 * 576 * s : d1 + 64 * (col - 9) + 16 * 448 * s;
                        const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)((col < 9 ? v0[0] : v1[0]) + o));
                        const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)((col < 9 ? v0[1] : v1[1]) + o));
                        v[ct] = __builtin_bit_cast(i32x4, (s16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]});
                    }
                    /* an accumulator's next product CT RT products later */
#pragma unroll
                    for (int lo = 0; lo < 2; lo++)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++)
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) O[rt][ct] = mfma32(lo ? pl[rt] : ph[rt], v[ct], O[rt][ct]);
                }
                __builtin_amdgcn_sched_barrier(0);
                VMCNT_WAIT(0);                         /* the loads of this step, a step's products ago */
                tl_barrier();
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const i32x4 at = *(lds_w4)(uintptr_t)(lds0 + TL_OT + (uint32_t)(4 * (32 * rt + 8 * g + 4 * hi)));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (32 * rt + 8 * g + 4 * hi + i >= j.nrows) continue;
                        float *o = a.part_o + (size_t)(uint32_t)at[i] * KVL + 32 * cb + c32;
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) o[32 * ct] = O[rt][ct][4 * g + i];
                    }
                }
        };
        /* the first barrier: issue0(0) done; the next: issue0(1) and issue1(0);
         * then all */
        if (nt > 2) {
            VMCNT_WAIT(18);
        } else if (nt == 2) {
            VMCNT_WAIT(9);
        } else {
            VMCNT_WAIT(4);
        }
        tl_barrier();
        if (nt > 2) {
            VMCNT_WAIT(9);
        } else if (nt == 2) {
            VMCNT_WAIT(4);
        } else {
            VMCNT_WAIT(0);
        }
        tl_barrier();
        VMCNT_WAIT(0);
        tl_barrier();
        using std::integral_constant;
        if (bw < 2) {
            if (two) run(integral_constant<int, 2>(), integral_constant<int, 5>());
            else run(integral_constant<int, 1>(), integral_constant<int, 5>());
        } else {
            if (two) run(integral_constant<int, 2>(), integral_constant<int, 3>());
            else run(integral_constant<int, 1>(), integral_constant<int, 3>());
        }
        return;
    }

    /* ---- scores ---- */
    const int rh = w & 1, second = w >> 1;             /* row half; latents 288.. */
    if (rh && !two) {
        for (int t = 0; t < nt + 3; t++) tl_barrier();
        return;
    }
    i32x4 qh[18], ql[18];
    {
        const int row = j.row0 + min(32 * rh + c32, j.nrows - 1);
        const uint8_t *p = (const uint8_t *)a.qf + (size_t)(row >> 5) * MM_MLA_QF_TILE + (36 * second + hi) * 512 + 16 * (row & 31);
#pragma unroll
        for (int s = 0; s < 18; s++) {
            qh[s] = *(const i32x4 *)(p + 1024 * s);
            ql[s] = *(const i32x4 *)(p + MM_MLA_QF_TILE / 2 + 1024 * s);
        }
    }
    const int sw = (c32 >> 2) & 3;
    const uint32_t xa = lds0 + TL_OX + (uint32_t)(rh * 4096 + 16 * lane);
    tl_barrier();                                      /* the first tile's latents 0..287 are there */
    if (!second) {
        const uint32_t ka = lds0 + (uint32_t)(c32 * 576);
        const uint32_t e0 = ka + 16 * (hi ^ sw), e1 = ka + 16 * ((2 + hi) ^ sw);   /* steps 0, 2, ..; 1, 3, .. */
        for (int t = 0; t < nt; t++) {
            const uint32_t d = (uint32_t)(t & 3) * TL_R0;
            f32x16 s = {};
            const uint32_t a0 = e0 + d, a1 = e1 + d;
            tl_scores(qh, ql, s, [&](int i) { return (i & 1 ? a1 : a0) + 64 * (i >> 1); });
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(lds_f4)(uintptr_t)(xa + (uint32_t)((t & 1) * 8192 + 1024 * i)) =
                    (f32x4){s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
            tl_barrier();
        }
        tl_barrier();
        tl_barrier();
        return;
    }
    const uint32_t ka = lds0 + TL_O1 + (uint32_t)(c32 * 448), kp = lds0 + TL_OK + (uint32_t)(c32 * 128);
    const uint32_t e0 = ka + 16 * (hi ^ sw), e1 = ka + 16 * ((2 + hi) ^ sw);
    uint32_t pe[4];
#pragma unroll
    for (int s = 0; s < 4; s++) pe[s] = kp + 16 * ((2 * s + hi) ^ ((c32 >> 1) & 7));
    const uint32_t pw = lds0 + TL_OP + (uint32_t)((32 * rh + c32) * 64 + 16 * (hi ^ sw));
    /* WIN: this lane's position, and those of the block's first and last rows */
    const int pos = WIN ? j.pos0 + (j.first_row + min(32 * rh + c32, j.nrows - 1)) / a.NH : 0;
    const int pos_a = WIN ? j.pos0 + j.first_row / a.NH : 0, pos_b = WIN ? j.pos0 + (j.first_row + j.nrows - 1) / a.NH : 0;
    float m = -INFINITY, l = 0.0f;
    tl_barrier();
    for (int t = 0; t < nt; t++) {
        const uint32_t d = (uint32_t)(t % 3) * TL_R1, dk = (uint32_t)(t & 1) * TL_KP;
        f32x16 s1;                                     /* scores in units of ln 2 */
#pragma unroll
        for (int i = 0; i < 4; i++) {                  /* the first half's sums */
            const f32x4 x = *(lds_f4)(uintptr_t)(xa + (uint32_t)((t & 1) * 8192 + 1024 * i));
#pragma unroll
            for (int q = 0; q < 4; q++) s1[4 * i + q] = x[q];
        }
        const uint32_t a0 = e0 + d, a1 = e1 + d;
        tl_scores(qh, ql, s1, [&](int i) { return i < 14 ? (i & 1 ? a1 : a0) + 64 * (i >> 1) : pe[i - 14] + dk; });
        uint32_t bad = 0;
        bool all = true;                               /* uniform: every row sees every key of the tile */
        if (WIN) {
            const int va = j.v0 + 32 * t, vb = va + 31;
            const int ja = tl_key(a, j, max(va, a.sinks)), jb = tl_key(a, j, vb);
            all = 32 * t + 31 < j.nk && jb <= pos_a && (jb < a.sinks || ja > pos_b - a.window);
        } else {
            all = 32 * t + 31 < j.nk;
        }
        float mx = -INFINITY;
        if (!all) {
            bool some = false;                         /* a score that is not finite: of such a key, or such a query */
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int v = 32 * t + 8 * (i >> 2) + 4 * hi + (i & 3);
                bool see = v < j.nk;
                if (WIN) {
                    const int key = tl_key(a, j, j.v0 + v);
                    const bool nf = see && !(fabsf(s1[i]) < INFINITY);
                    see = see && key <= pos && (key < a.sinks || key > pos - a.window);
                    some |= nf;
                    if (nf) s1[i] = __builtin_nanf("");
                }
                if (!see) s1[i] = -INFINITY;
            }
            /* every row's score of a key that is not finite is not, so both halves'
             * waves find the same; all of the tile is in LDS until its output step */
            if (WIN && __builtin_amdgcn_ballot_w64(some)) bad = tl_not_finite(lds0 + (uint32_t)(t & 3) * TL_R0, lds0 + TL_O1 + d, lds0 + TL_OK + dk);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, s1[i]);
        const bool moved = __builtin_amdgcn_ballot_w64(mx > m + XTAU) != 0;
        if (moved) {                                   /* lazy rescaling, as in mm_mla_attn */
            mx = fmaxf(mx, __shfl_xor(mx, 32, MM_WAVE));
            const float mn = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            m = mn;
            if (hi == 0) ((lds_f)(uintptr_t)(lds0 + TL_OF))[(t & 1) * 64 + 32 * rh + c32] = f;
        }
        if (lane == 0) {
            lds_i fl = (lds_i)(uintptr_t)(lds0 + TL_OG + 16 * (t & 1));
            fl[rh] = moved ? 1 : 0;
            if (WIN) fl[2 + rh] = (int)bad;
        }
        const float mz = m == -INFINITY ? 0.0f : m;    /* rows with no key yet: probabilities 0 */
#pragma unroll
        for (int s = 0; s < 2; s++) {
            i32x4 ph, pl;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p0 = __builtin_amdgcn_exp2f(s1[8 * s + 2 * i] - mz), p1 = __builtin_amdgcn_exp2f(s1[8 * s + 2 * i + 1] - mz);
                l += p0 + p1;
                uint32_t vh, vl;
                split_pk(p0, p1, &vh, &vl);
                ph[i] = (int)vh;
                pl[i] = (int)vl;
            }
            const uint32_t p = (pw ^ (uint32_t)(32 * s)) + (uint32_t)((t & 1) * 8192);
            *(lds_w4)(uintptr_t)p = ph;
            *(lds_w4)(uintptr_t)(p + 4096) = pl;
        }
        tl_barrier();
    }
    l += __shfl_xor(l, 32, MM_WAVE);
    if (hi == 0 && 32 * rh + c32 < j.nrows) {
        const uint32_t at = (uint32_t)((lds_i)(uintptr_t)(lds0 + TL_OT))[32 * rh + c32];
        a.part_ml[(size_t)(at >> 4) * 32 + (at & 15)] = m * 0.693147180559945309f;
        a.part_ml[(size_t)(at >> 4) * 32 + 16 + (at & 15)] = l;
    }
    tl_barrier();
}

/* Absorbed queries and q_pe, times softmax scale / ln 2 (scores come out in units
 * of ln 2), as the score waves read them: bf16 pairs in 32-row
 * tiles [hi, lo][72 pieces of 8 latents][32 rows][16 bytes], so that a wave's load
 * is 1 KB.  (From row-major planes each load met 32 lines, 2 us per block.)
 *
 * W_UK comes first, as two 16-row tiles whose rows are latents 8 g + i and 8 g +
 * 4 + i (row 4 g + i), so that a lane ends with the 8 latents of a piece. */
__device__ __forceinline__ void qf_split(const f32x4 &x0, const f32x4 &x1, float f, i32x4 &ph, i32x4 &pl) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t vh, vl;
        split_pk((i < 2 ? x0[2 * i] : x1[2 * i - 4]) * f, (i < 2 ? x0[2 * i + 1] : x1[2 * i - 3]) * f, &vh, &vl);
        ph[i] = (int)vh;
        pl[i] = (int)vl;
    }
}
__device__ __forceinline__ uint8_t *qf_place(const mm_mla_qfrag_args &a, int b, int h, int piece) {
    const size_t r = (size_t)b * a.NH + h;
    return (uint8_t *)a.qf + (r >> 5) * MM_MLA_QF_TILE + 512 * piece + 16 * (r & 31);
}
/* One wave: latents e0 .. e0 + 31 of head h for 16 positions from b0 on (past the
 * last: that again); ph / pl piece e0 / 8 + lane / 16 of position b0 + lane % 16.
 *
 * Both operands come through LDS (`buf`, the wave's own), WIN windows of 64 at a
 * time: a load whose neighbouring lanes are in different rows costs the L1 a
 * request per lane, and the fragments read from memory that way took 10 of 19 us
 * (512 positions of 16 heads).  Rows are 16-byte pieces, W's 8 of them and q's 16;
 * piece p of row r lies in slot p ^ qf_swz(r) or p ^ r, so that the 16 rows of a
 * fragment fall on all banks. */
#define QF_WINDOW 8192
__device__ __forceinline__ int qf_swz(int r) { return (r >> 3 & 3) << 1 | (r >> 1 & 1); }
template <int WIN>
__device__ __forceinline__ void qf_wave(const mm_mla_qfrag_args &a, int h, int b0, int e0, uint8_t *buf, i32x4 &ph, i32x4 &pl) {
    const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
    const uint16_t *wr = a.wukT + ((size_t)h * KVL + e0 + (lane >> 3)) * a.QKN;
    f32x4 y[2] = {};
    for (int k0 = 0; k0 < a.QKN; k0 += 64 * WIN) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   /* the windows before are read */
#pragma unroll
        for (int u = 0; u < WIN; u++) {
            const int k = k0 + 64 * u;
            if (k >= a.QKN) break;                     /* uniform */
            uint8_t *p = buf + u * QF_WINDOW;
#pragma unroll
            for (int i = 0; i < 4; i++)                /* 8 rows of W (a last half window: its end again) */
                lds_dma16(wr + 8 * i * a.QKN + min(k + 8 * ((lane & 7) ^ qf_swz(8 * i + (lane >> 3))), a.QKN - 8), p + 1024 * i);
#pragma unroll
            for (int i = 0; i < 4; i++) {              /* 4 rows of q (a last half window: into q_pe) */
                const int r = 4 * i + g;
                lds_dma16(a.q + ((size_t)min(b0 + r, a.R - 1) * a.NH + h) * (a.QKN + MM_MLA_QKR) + k + 4 * (n16 ^ r), p + 4096 + 1024 * i);
            }
        }
        VMCNT_WAIT(0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < 2 * WIN; u++) {
            if (k0 + 32 * u >= a.QKN) break;
            const uint8_t *p = buf + (u >> 1) * QF_WINDOW, *qp = p + 4096 + 256 * n16;
            const int c = 8 * (u & 1) + 2 * g;
            i32x4 xh, xl;
            qf_split(*(const f32x4 *)(qp + 16 * (c ^ n16)), *(const f32x4 *)(qp + 16 * ((c + 1) ^ n16)), 1.0f, xh, xl);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int r = 8 * (n16 >> 2) + (n16 & 3) + 4 * t;
                const i32x4 wv = *(const i32x4 *)(p + 128 * r + 16 * ((g + 4 * (u & 1)) ^ qf_swz(r)));
                y[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv), __builtin_bit_cast(bf16x8, xh), y[t], 0, 0, 0);
                y[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv), __builtin_bit_cast(bf16x8, xl), y[t], 0, 0, 0);
            }
        }
    }
    qf_split(y[0], y[1], a.scale2, ph, pl);
}

/* Few positions: grid (KVL / 64 slabs and one for q_pe, NH, ceil(R / 32)), wave w
 * latents 32 (w % 2) .. + 31 of the slab for positions 16 (w / 2) .. + 15. */
extern "C" __global__ __launch_bounds__(256) void mm_mla_qfrag(mm_mla_qfrag_args a) {
    __shared__ __attribute__((aligned(1024))) uint8_t qbuf[4][2 * QF_WINDOW];
    const int slab = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    i32x4 ph, pl;
    int b, piece;
    if (slab == KVL / 64) {                            /* q_pe: a piece per thread */
        b = blockIdx.z * 32 + (tid >> 3);
        piece = KVL / 8 + (tid & 7);
        const float *q = a.q + ((size_t)min(b, a.R - 1) * a.NH + h) * (a.QKN + MM_MLA_QKR) + a.QKN + 8 * (tid & 7);
        qf_split(*(const f32x4 *)q, *(const f32x4 *)(q + 4), a.scale2, ph, pl);
    } else {
        const int e0 = 64 * slab + 32 * (w & 1), b0 = blockIdx.z * 32 + 16 * (w >> 1);
        b = b0 + (lane & 15);
        piece = e0 / 8 + (lane >> 4);
        qf_wave<2>(a, h, b0, e0, qbuf[w], ph, pl);
    }
    if (b >= a.R) return;
    uint8_t *p = qf_place(a, b, h, piece);
    *(i32x4 *)p = ph;
    *(i32x4 *)(p + MM_MLA_QF_TILE / 2) = pl;
}

/* More: a block of eight heads (wave w head w), whose 16-byte pieces are one line
 * and leave together through LDS; 32 latents of 16 positions.  One window at a time,
 * so that a CU holds two blocks (512 of 16 heads 15.5 us; two windows 20.4, more
 * positions or latents per block 19).  grid (KVL / 32 and one for q_pe, ceil(NH /
 * 8), ceil(R / 16)). */
extern "C" __global__ __launch_bounds__(512) void mm_mla_qfrag_8(mm_mla_qfrag_args a) {
    __shared__ __attribute__((aligned(1024))) uint8_t qbuf[8][QF_WINDOW];
    typedef i32x4 pieces[2][4][16][8];                 /* [hi, lo][piece][position][head], over the windows */
    static_assert(sizeof(pieces) <= sizeof(qbuf), "a block's pieces");
    pieces &st = *(pieces *)(void *)qbuf;
    const int slab = blockIdx.x, h0 = blockIdx.y * 8, b0 = blockIdx.z * 16;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sh = tid & 7, sb = tid >> 3 & 15, sp = tid >> 7;
    if (slab == KVL / 32) {                            /* q_pe: 8 pieces, 16 positions, 8 heads */
        if (b0 + sb >= a.R || h0 + sh >= a.NH) return;
        const float *q = a.q + ((size_t)(b0 + sb) * a.NH + h0 + sh) * (a.QKN + MM_MLA_QKR) + a.QKN;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int piece = sp + 4 * u;
            i32x4 ph, pl;
            qf_split(*(const f32x4 *)(q + 8 * piece), *(const f32x4 *)(q + 8 * piece + 4), a.scale2, ph, pl);
            uint8_t *p = qf_place(a, b0 + sb, h0 + sh, KVL / 8 + piece);
            *(i32x4 *)p = ph;
            *(i32x4 *)(p + MM_MLA_QF_TILE / 2) = pl;
        }
        return;
    }
    i32x4 ph, pl;
    qf_wave<1>(a, min(h0 + w, a.NH - 1), b0, 32 * slab, qbuf[w], ph, pl);
    __syncthreads();                                   /* the windows are read */
    st[0][lane >> 4][lane & 15][w] = ph;
    st[1][lane >> 4][lane & 15][w] = pl;
    __syncthreads();
    if (b0 + sb < a.R && h0 + sh < a.NH) {
        uint8_t *p = qf_place(a, b0 + sb, h0 + sh, 4 * slab + sp);
        *(i32x4 *)p = st[0][sp][sb][sh];
        *(i32x4 *)(p + MM_MLA_QF_TILE / 2) = st[1][sp][sb][sh];
    }
}

/* A shared prefix, and one position per sequence over its own keys. */
extern "C" __global__ __launch_bounds__(512, 2) void mm_mla_attn_tiles(mm_mla_tiles_args a) { tl_block<false>(a); }
/* Windows with sinks. */
extern "C" __global__ __launch_bounds__(512, 2) void mm_mla_attn_tiles_w(mm_mla_tiles_args a) { tl_block<true>(a); }

/* The chunks' partials of up to 16 positions of one head merged, and their W_UV
 * products: ctx = W_UV sum_c e^(m_c - m) O_c / l, the latent contexts meeting the
 * matrix cores as bf16 pairs from LDS.  One launch and no latent context in memory
 * between.  A 1-D grid of NH * split * ceil(R / ppb) blocks, heads first (column
 * splits merge for themselves); NW waves.
 *
 * Wave w merges positions w, w + NW, ..; in a call of fewer than NW positions
 * `wpp` waves share one, each every wpp-th chunk.  Then each takes every NW-th
 * 16-column tile of the block's columns.  A position without a key: zeros. */
#define MU_ROW 1040                /* bytes of a position's 512 latents in LDS, and 16 */
template <int NW>
__device__ __forceinline__ void merge_uv(const mm_mla_merge_uv_args &a) {
    __shared__ __attribute__((aligned(16))) uint8_t mlds[2 * 16 * MU_ROW];
    __shared__ f32x4 red[NW - 1][2][MM_WAVE];
    const int id = (int)blockIdx.x, h = id % a.NH, sp = id / a.NH % a.split, b0 = id / (a.NH * a.split) * a.ppb;
    const int lane = threadIdx.x & (MM_WAVE - 1);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / MM_WAVE);
    const int nrows = min(a.ppb, a.R - b0);
    const int G = a.wpp;                               /* waves per position */
    const int cg = w % G;
    const int ncol = (a.VHD + 15) / 16, per = (ncol + a.split - 1) / a.split;
    const int ct0 = sp * per, ct1 = min(ct0 + per, ncol);
    const int n16 = lane & 15, kq = 8 * (lane >> 4);
    typedef const __attribute__((address_space(1))) i32x4 *glb_c4;
    /* this wave's first column tile's weights: in flight during the merge */
    i32x4 wv[KVL / 32];
    auto weights = [&](int ct) {
        const uint16_t *p = a.wuvf + ((size_t)h * ncol + ct) * MM_MLA_UVF_TILE + 8 * lane;
#pragma unroll
        for (int s = 0; s < KVL / 32; s++) wv[s] = *(glb_c4)(uintptr_t)(p + 512 * s);
    };
    weights(min(ct0 + w, ncol - 1));

    /* the first 64 chunks' maxima and sums of this wave's positions, all in flight
     * together: lane c has chunk c */
    float mcs[16 / NW], lcs[16 / NW];
#pragma unroll
    for (int i = 0; i < 16 / NW; i++) {
        const size_t pb = ((size_t)(b0 + min(w / G + i * (NW / G), nrows - 1)) * a.HG + (h >> 4)) * a.nchunks;
        const float *ml = a.part_ml + (pb + min(lane, a.nchunks - 1)) * 32 + (h & 15);
        mcs[i] = ml[0];
        lcs[i] = ml[16];
    }
#pragma unroll
    for (int ri = 0; ri < 16 / NW; ri++) {
        /* G > 1: one round, in which waves past the rows (a call's last group of
         * rows) repeat the last one, since all meet at the barrier */
        const int r = w / G + ri * (NW / G);
        if (G > 1 ? ri > 0 : r >= nrows) break;
        const size_t pb = ((size_t)(b0 + min(r, nrows - 1)) * a.HG + (h >> 4)) * a.nchunks;
        const float *ml = a.part_ml + pb * 32 + (h & 15);
        const float *po = a.part_o + (pb * 16 + (h & 15)) * KVL + 4 * lane;
        float mx = mcs[ri];                            /* lanes past the chunks hold the last one's */
        for (int c = MM_WAVE + lane; c < a.nchunks; c += MM_WAVE) mx = fmaxf(mx, ml[(size_t)c * 32]);
        mx = wave_max(mx);
        float l = 0.0f;
        f32x4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
        for (int cb = 0; cb < a.nchunks; cb += MM_WAVE) {
            const int cl = min(cb + lane, a.nchunks - 1);
            const float mc = cb ? ml[(size_t)cl * 32] : mcs[ri], lc = cb ? ml[(size_t)cl * 32 + 16] : lcs[ri];
            const float wc = cb + lane < a.nchunks && mc != -INFINITY ? __expf(mc - mx) : 0.0f;
            l += lc * wc;
            const int n = min(MM_WAVE, a.nchunks - cb);
            constexpr int U = 4;                       /* chunks whose loads are in flight */
            for (int c0 = cg; c0 < n; c0 += U * G) {
                f32x4 v[U][2];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float *p = po + (size_t)(cb + min(c0 + u * G, n - 1)) * 16 * KVL;
                    v[u][0] = *(const f32x4 *)p;
                    v[u][1] = *(const f32x4 *)(p + 256);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int c = c0 + u * G;
                    const float f = c < n ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wc), c & 63)) : 0.0f;
                    s0 += v[u][0] * f;
                    s1 += v[u][1] * f;
                }
            }
        }
        l = wave_sum(l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (G > 1) {
            /* one position per group of G waves: their sums meet in its first */
            if (cg > 0) {
                red[w - 1][0][lane] = s0;
                red[w - 1][1][lane] = s1;
            }
            __syncthreads();
            if (cg == 0)
                for (int u = 1; u < G; u++) {
                    s0 += red[w + u - 1][0][lane];
                    s1 += red[w + u - 1][1][lane];
                }
        }
        if (cg == 0) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const f32x4 s = q ? s1 * inv : s0 * inv;
                uint32_t h0, h1, l0, l1;
                split_pk(s[0], s[1], &h0, &l0);
                split_pk(s[2], s[3], &h1, &l1);
                *(u32x2 *)(mlds + r * MU_ROW + 512 * q + 8 * lane) = (u32x2){h0, h1};
                *(u32x2 *)(mlds + (16 + r) * MU_ROW + 512 * q + 8 * lane) = (u32x2){l0, l1};
            }
        }
    }
    __syncthreads();
    const int ra = min(n16, nrows - 1) * MU_ROW + 2 * kq;
    for (int ct = ct0 + w; ct < ct1; ct += NW) {
        if (ct != ct0 + w) weights(ct);
        f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f}, yl = y;
#pragma unroll
        for (int s = 0; s < KVL / 32; s++) {
            const i32x4 xh = *(const i32x4 *)(mlds + ra + 64 * s), xl = *(const i32x4 *)(mlds + 16 * MU_ROW + ra + 64 * s);
            y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xh), __builtin_bit_cast(bf16x8, wv[s]), y, 0, 0, 0);
            yl = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xl), __builtin_bit_cast(bf16x8, wv[s]), yl, 0, 0, 0);
        }
        const int v = 16 * ct + n16;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 4 * (lane >> 4) + i;
            if (r < nrows && v < a.VHD) a.ctx[((size_t)(b0 + r) * a.NH + h) * a.VHD + v] = y[i] + yl[i];
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void mm_mla_merge_uv_4(mm_mla_merge_uv_args a) { merge_uv<4>(a); }
extern "C" __global__ __launch_bounds__(512) void mm_mla_merge_uv_8(mm_mla_merge_uv_args a) { merge_uv<8>(a); }
