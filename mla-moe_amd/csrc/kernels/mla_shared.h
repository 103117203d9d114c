/* mla_shared.h -- absorbed MLA attention of many rows over one list of keys
 * (part of mla.hip): the prefix that a decode batch shares.
 *
 * A row is one (sequence, head): B NH of them meet every key, 1,088 products a
 * (row, key) pair, twice over since the fp32 query and the probabilities travel
 * as bf16 pairs.  mm_mla_attn keeps 16 rows (one sequence's heads) per wave: each
 * sequence reads the prefix again, and 16 x 16 tiles feed the matrix cores from
 * LDS once per 16 rows.  Here a block takes 64 rows over a chunk of keys, on 32
 * x 32 tiles, one block per CU, its eight waves in three roles (each SIMD holds
 * one wave of the first two and one of the third), each one 32-key tile behind
 * the other:
 *   waves 0, 1   scores of tile t + 2 over latents 0..287 (32 rows each)
 *   waves 2, 3   scores of tile t + 1 over latents 288..575, added to the former;
 *                softmax; the probabilities as bf16 pairs to LDS
 *   waves 4..7   O += P V of tile t, 64 rows x 128 latent columns each; and the
 *                loads of the tiles to come
 * A score wave keeps its 32 rows' queries over its half of the latents (144
 * registers), an output wave its 64 x 128 of O (128 registers): neither would
 * fit beside the other, and the softmax of one tile runs beside the products of
 * the others.  One barrier per tile.
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
#define SH_R0 18432                /* bytes of one tile: latents 0..287 */
#define SH_R1 14336                /* latents 288..511 */
#define SH_KP 4096                 /* k_pe */
#define SH_O1 (4 * SH_R0)
#define SH_OK (SH_O1 + 3 * SH_R1)
#define SH_OP (SH_OK + 2 * SH_KP)  /* P: two tiles of 64 rows x 32 keys, hi then lo */
#define SH_OX (SH_OP + 2 * 8192)   /* partial scores: two tiles of 64 x 32 floats */
#define SH_OF (SH_OX + 2 * 8192)   /* rescaling factors: two tiles of 64 floats */
#define SH_OG (SH_OF + 2 * 256)    /* whether there are some: [tile % 2][row half] */
#define SH_OT (SH_OG + 16)         /* 64 rows' places in the partials */
static_assert(SH_OT + 256 <= MM_MLA_SH_LDS && MM_MLA_SH_LDS <= 163840, "LDS of a block");
typedef __attribute__((address_space(3))) s16x4 *lds_s4;
typedef __attribute__((address_space(3))) i32x4 *lds_w4;
typedef __attribute__((address_space(3))) f32x4 *lds_f4;
typedef __attribute__((address_space(3))) float *lds_f;
typedef __attribute__((address_space(3))) int *lds_i;

/* LDS accesses done, then the block's barrier; loads into LDS stay in flight. */
__device__ __forceinline__ void sh_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

extern "C" __global__ __launch_bounds__(512, 2) void mm_mla_attn_shared(mm_mla_shared_args a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t slds[];
    const uint32_t lds0 = lds_addr(slds);
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, hi = lane >> 5;
    /* chunk-major, an eighth of the list per XCD: a chunk's row tiles read its
     * keys from one L2 */
    const int nrt = (a.M + 63) / 64, ntrip = nrt * a.nchunks, per = (ntrip + 7) / 8;
    const int trip = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || trip >= ntrip) return;
    const int chunk = trip / nrt, row0 = trip % nrt * 64;
    const int k0 = chunk * a.chunk, nk = min(a.chunk, a.nkeys - k0);
    const int nt = (nk + 31) / 32;

    if (tid < 64) {                                    /* row (b, h): partial ((b HG + h / 16) pchunks + chunk), line h % 16 */
        const int r = min(row0 + tid, a.M - 1), b = r / a.NH, h = r - b * a.NH;
        ((lds_i)(uintptr_t)(lds0 + SH_OT))[tid] = ((b * a.HG + (h >> 4)) * a.pchunks + chunk) * 16 + (h & 15);
    }

    if (w >= 4) {
        /* ---- O += P V, and the loads ---- */
        const int bw = w - 4;
        const rsrc_t rk = raw_rsrc(a.keys + (size_t)k0 * KVD, (uint32_t)nk * KVD * 2);
        /* this wave's nine of a tile's 36 1-KB loads: LDS piece x (16 bytes) of
         * the part is row x / pieces-per-row, slot x % it */
        uint32_t so[9], dl[9];
#pragma unroll
        for (int i = 0; i < 9; i++) {
            const bool r0 = i < 4 || (i == 4 && bw < 2);
            const int u = i < 4 ? bw + 4 * i : i == 4 ? (bw < 2 ? 16 + bw : 10 + bw) : i < 8 ? bw + 4 * (i - 5) : bw;
            const int x = 64 * u + lane;
            if (i == 8) {
                const int r = x >> 3, p = (x & 7) ^ ((r >> 1) & 7);
                so[i] = (uint32_t)(r * KVD * 2 + KVL * 2 + 16 * p);
            } else {
                const int ppr = r0 ? 36 : 28, r = x / ppr, s = x - r * ppr;
                const int p = (s & ~3) | ((s ^ (r >> 2)) & 3);
                so[i] = (uint32_t)(r * KVD * 2 + (r0 ? 0 : 576) + 16 * p);
            }
            dl[i] = lds0 + (uint32_t)(1024 * u) + (i == 8 ? SH_OK : r0 ? 0 : SH_O1);
        }
        constexpr uint32_t TB = 32 * KVD * 2;          /* bytes of a tile's rows */
        /* latents 0..287 of tile t0; 288..575 of tile t1 */
        auto issue0 = [&](int t) {
            const uint32_t d = (uint32_t)(t & 3) * SH_R0, o = (uint32_t)t * TB;
#pragma unroll
            for (int i = 0; i < 4; i++) lds_dma16_buf(so[i] + o, rk, dl[i] + d);
            if (bw < 2) lds_dma16_buf(so[4] + o, rk, dl[4] + d);
        };
        auto issue1 = [&](int t) {
            const uint32_t d = (uint32_t)(t % 3) * SH_R1, o = (uint32_t)t * TB;
            if (bw >= 2) lds_dma16_buf(so[4] + o, rk, dl[4] + d);
#pragma unroll
            for (int i = 5; i < 8; i++) lds_dma16_buf(so[i] + o, rk, dl[i] + d);
            lds_dma16_buf(so[8] + o, rk, dl[8] + (uint32_t)(t & 1) * SH_KP);
        };
        issue0(0);
        if (nt > 1) issue0(1);
        issue1(0);
        if (nt > 2) issue0(2);
        if (nt > 1) issue1(1);

        /* transposing reads: lane i of 16-lane group g supplies row 4 (4 s + 2 e
         * + g / 2) + i / 4, 4 columns from 16 (g % 2) + 4 (i % 4) of column tile ct */
        const int i16 = lane & 15, gq = lane >> 4, h = gq >> 1;
        uint32_t va[4][2][2];                          /* [ct][s][e], without the tile's place */
#pragma unroll
        for (int ct = 0; ct < 4; ct++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int col4 = 4 * bw + ct;      /* 32-column tile of the 16 */
                    const bool r0 = col4 < 9;
                    const int r = 16 * s + 8 * e + 4 * h + (i16 >> 2);
                    const int low = (2 * (gq & 1) + ((i16 >> 1) & 1)) ^ (2 * e + h);
                    va[ct][s][e] = lds0 + (r0 ? 0 : SH_O1) + (uint32_t)(r * (r0 ? 576 : 448) + 64 * (r0 ? col4 : col4 - 9) + 16 * low + 8 * (i16 & 1));
                }
        const uint32_t pa = lds0 + SH_OP + (uint32_t)(c32 * 64 + 16 * (hi ^ ((c32 >> 2) & 3)));   /* piece 2 s + hi: s flips bit 1 */
        f32x16 O[2][4] = {};
        VMCNT_WAIT(0);
        sh_barrier();                                  /* the first tiles are there */
        sh_barrier();
        sh_barrier();
        for (int t = 0; t < nt; t++) {
            if (t + 3 < nt) issue0(t + 3);
            if (t + 2 < nt) issue1(t + 2);
            const uint32_t d0 = (uint32_t)(t & 3) * SH_R0, d1 = (uint32_t)(t % 3) * SH_R1;
            const uint32_t po = (uint32_t)(t & 1) * 8192;
            i32x4 ph[2][2], pl[2][2];                  /* [s][row tile] */
            i32x4 v[2][4];
#pragma unroll
            for (int s = 0; s < 2; s++) {
#pragma unroll
                for (int rt = 0; rt < 2; rt++) {
                    const uint32_t p = (pa ^ (uint32_t)(32 * s)) + po + 2048 * rt;
                    ph[s][rt] = *(lds_w4)(uintptr_t)p;
                    pl[s][rt] = *(lds_w4)(uintptr_t)(p + 4096);
                }
#pragma unroll
                for (int ct = 0; ct < 4; ct++) {
                    const uint32_t d = 4 * bw + ct < 9 ? d0 : d1;
                    const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(va[ct][s][0] + d));
                    const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(va[ct][s][1] + d));
                    v[s][ct] = __builtin_bit_cast(i32x4, (s16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]});
                }
            }
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                const int moved = __builtin_amdgcn_readfirstlane(((lds_i)(uintptr_t)(lds0 + SH_OG))[2 * (t & 1) + rt]);
                if (moved) {                           /* some row's maximum moved: its factor */
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const f32x4 f = *(lds_f4)(uintptr_t)(lds0 + SH_OF + (uint32_t)((t & 1) * 256 + 4 * (32 * rt + 8 * g + 4 * hi)));
#pragma unroll
                        for (int ct = 0; ct < 4; ct++)
#pragma unroll
                            for (int i = 0; i < 4; i++) O[rt][ct][4 * g + i] *= f[i];
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int ct = 0; ct < 4; ct++)
#pragma unroll
                    for (int rt = 0; rt < 2; rt++) {
                        O[rt][ct] = mfma32(ph[s][rt], v[s][ct], O[rt][ct]);
                        O[rt][ct] = mfma32(pl[s][rt], v[s][ct], O[rt][ct]);
                    }
            VMCNT_WAIT(0);                             /* the loads of this step, a step's products ago */
            sh_barrier();
        }
#pragma unroll
        for (int rt = 0; rt < 2; rt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const i32x4 at = *(lds_w4)(uintptr_t)(lds0 + SH_OT + (uint32_t)(4 * (32 * rt + 8 * g + 4 * hi)));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (row0 + 32 * rt + 8 * g + 4 * hi + i >= a.M) continue;
                    float *o = a.part_o + (size_t)(uint32_t)at[i] * KVL + 128 * bw + c32;
#pragma unroll
                    for (int ct = 0; ct < 4; ct++) o[32 * ct] = O[rt][ct][4 * g + i];
                }
            }
        return;
    }

    /* ---- scores ---- */
    const int rh = w & 1, second = w >> 1;             /* row half; latents 288.. */
    const int row = min(row0 + 32 * rh + c32, a.M - 1);
    i32x4 qh[18], ql[18];
    {
        const uint16_t *p = a.qhl + (size_t)row * 2 * KVL + 288 * second + 8 * hi;
#pragma unroll
        for (int s = 0; s < 14; s++) {
            qh[s] = *(const i32x4 *)(p + 16 * s);
            ql[s] = *(const i32x4 *)(p + KVL + 16 * s);
        }
        if (second) {
            const float *qp = a.q + (size_t)row * (a.QKN + MM_MLA_QKR) + a.QKN + 8 * hi;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const f32x4 x0 = *(const f32x4 *)(qp + 16 * s), x1 = *(const f32x4 *)(qp + 16 * s + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t vh, vl;
                    split_pk(j < 2 ? x0[2 * j] : x1[2 * j - 4], j < 2 ? x0[2 * j + 1] : x1[2 * j - 3], &vh, &vl);
                    qh[14 + s][j] = (int)vh;
                    ql[14 + s][j] = (int)vl;
                }
            }
        } else {
#pragma unroll
            for (int s = 14; s < 18; s++) {
                qh[s] = *(const i32x4 *)(p + 16 * s);
                ql[s] = *(const i32x4 *)(p + KVL + 16 * s);
            }
        }
    }
    const int sw = (c32 >> 2) & 3;
    const uint32_t xa = lds0 + SH_OX + (uint32_t)(rh * 4096 + 16 * lane);
    sh_barrier();                                      /* the first tiles are there */
    if (!second) {
        const uint32_t ka = lds0 + (uint32_t)(c32 * 576);
        const uint32_t e0 = ka + 16 * (hi ^ sw), e1 = ka + 16 * ((2 + hi) ^ sw);   /* steps 0, 2, ..; 1, 3, .. */
        for (int t = 0; t < nt; t++) {
            const uint32_t d = (uint32_t)(t & 3) * SH_R0;
            f32x16 s1 = {}, s2 = {};
#pragma unroll
            for (int s = 0; s < 18; s++) {
                const i32x4 k = *(lds_w4)(uintptr_t)((s & 1 ? e1 : e0) + d + 64 * (s >> 1));
                s1 = mfma32(k, qh[s], s1);
                s2 = mfma32(k, ql[s], s2);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(lds_f4)(uintptr_t)(xa + (uint32_t)((t & 1) * 8192 + 1024 * j)) =
                    (f32x4){s1[4 * j] + s2[4 * j], s1[4 * j + 1] + s2[4 * j + 1], s1[4 * j + 2] + s2[4 * j + 2], s1[4 * j + 3] + s2[4 * j + 3]};
            sh_barrier();
        }
        sh_barrier();
        sh_barrier();
        return;
    }
    const uint32_t ka = lds0 + SH_O1 + (uint32_t)(c32 * 448), kp = lds0 + SH_OK + (uint32_t)(c32 * 128);
    const uint32_t e0 = ka + 16 * (hi ^ sw), e1 = ka + 16 * ((2 + hi) ^ sw);
    uint32_t pe[4];
#pragma unroll
    for (int s = 0; s < 4; s++) pe[s] = kp + 16 * ((2 * s + hi) ^ ((c32 >> 1) & 7));
    const uint32_t pw = lds0 + SH_OP + (uint32_t)((32 * rh + c32) * 64 + 16 * (hi ^ sw));
    const float scale2 = a.scale * 1.44269504088896341f;   /* scores in units of ln 2 */
    float m = -INFINITY, l = 0.0f;
    sh_barrier();
    for (int t = 0; t < nt; t++) {
        const uint32_t d = (uint32_t)(t % 3) * SH_R1, dk = (uint32_t)(t & 1) * SH_KP;
        f32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = *(lds_f4)(uintptr_t)(xa + (uint32_t)((t & 1) * 8192 + 1024 * j));
        f32x16 s1 = {}, s2 = {};
#pragma unroll
        for (int s = 0; s < 18; s++) {
            const i32x4 k = s < 14 ? *(lds_w4)(uintptr_t)((s & 1 ? e1 : e0) + d + 64 * (s >> 1)) : *(lds_w4)(uintptr_t)(pe[s - 14] + dk);
            s1 = mfma32(k, qh[s], s1);
            s2 = mfma32(k, ql[s], s2);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s1[i] = (s1[i] + s2[i] + x[i >> 2][i & 3]) * scale2;
            if (t == nt - 1 && 32 * t + 8 * (i >> 2) + 4 * hi + (i & 3) >= nk) s1[i] = -INFINITY;
            mx = fmaxf(mx, s1[i]);
        }
        const bool moved = __builtin_amdgcn_ballot_w64(mx > m + XTAU) != 0;
        if (moved) {                                   /* lazy rescaling, as in mm_mla_attn */
            mx = fmaxf(mx, __shfl_xor(mx, 32, MM_WAVE));
            const float mn = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            m = mn;
            if (hi == 0) ((lds_f)(uintptr_t)(lds0 + SH_OF))[(t & 1) * 64 + 32 * rh + c32] = f;
        }
        if (lane == 0) ((lds_i)(uintptr_t)(lds0 + SH_OG))[2 * (t & 1) + rh] = moved ? 1 : 0;
        const float mz = m == -INFINITY ? 0.0f : m;
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
        sh_barrier();
    }
    l += __shfl_xor(l, 32, MM_WAVE);
    if (hi == 0 && row0 + 32 * rh + c32 < a.M) {
        const uint32_t at = (uint32_t)((lds_i)(uintptr_t)(lds0 + SH_OT))[32 * rh + c32];
        a.part_ml[(size_t)(at >> 4) * 32 + (at & 15)] = m * 0.693147180559945309f;
        a.part_ml[(size_t)(at >> 4) * 32 + 16 + (at & 15)] = l;
    }
    sh_barrier();
}
