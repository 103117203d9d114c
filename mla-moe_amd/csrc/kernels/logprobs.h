/* logprobs.h -- log probabilities of given tokens, entropies and top
 * alternatives of rows of logits (part of lm_head.hip).
 *
 * For a row x with maximum m (held by one element; equal ones count again):
 *   R = sum over the others of e^(x_i - m),  U = the same sum of e^(x_i - m) (x_i - m)
 *   log p_t = (x_t - m) - log1p(R),  entropy = log1p(R) - U / (1 + R)
 * Keeping the maximum's own 1 out of the sum leaves no cancellation: a token
 * of probability 1 - 1e-9 has its log probability and the row its entropy to
 * full precision.  U <= 0, so the entropy adds two non-negative terms.
 *
 * One pass over the logits; bound by reading them (4 bytes each, about 16
 * instructions per element against the ~30 that fit beside the memory's
 * rate).  A wave takes chunks of 1,024 elements of its block's segment, two in
 * flight, every lane with an (m, R, U) of its own; they meet by pairs at the
 * end.  The n_top largest are kept beside, as 64-bit keys whose order is (value
 * descending, index ascending): a list in LDS, compacted by rank, and the key that
 * an element must beat.  A wave meets few such elements after its first chunk,
 * which starts from the n_top-th of the lanes' maxima.  All of this is written
 * once per kernel, in loops: unrolled over a chunk's elements it was instructions
 * to fetch (one row, 20 alternatives: 13 + 7 us, in loops 9 + 5; without any 4 +
 * 2, so that the selection still is most of a short call). */
#define LP_VPL 16                  /* elements per lane and chunk */
#define LP_CHUNK (LP_VPL * MM_WAVE)
#define LP_WAVES 4
#define LP_LIST 128                /* list entries of a wave: compacted past 64, 64 more fit */
#define LP_DMIN (-200.0f)          /* below it e^d is 0: keeps 0 * -inf out of U */
static_assert(MM_LP_TOP_MAX <= 32 && LP_WAVES * MM_LP_TOP_MAX <= LP_LIST, "the waves' lists meet in one");
static_assert(MM_LP_SEG_MAX <= MM_WAVE, "the final merge: a lane per segment");

struct lp_stat {
    float m, R, U;                 /* no element: -inf, -1 (1 + R = 0), 0 */
};

__device__ __forceinline__ lp_stat lp_merge(const lp_stat &a, const lp_stat &b) {
    const bool ab = a.m >= b.m;
    const float mh = ab ? a.m : b.m, ml = ab ? b.m : a.m;
    const float Rh = ab ? a.R : b.R, Rl = ab ? b.R : a.R;
    const float Uh = ab ? a.U : b.U, Ul = ab ? b.U : a.U;
    const float d = ml - mh, w = ml == -INFINITY ? 0.0f : __expf(d), s = 1.0f + Rl;
    return {mh, Rh + s * w, Uh + w * (Ul + fmaxf(d, LP_DMIN) * s)};
}

/* Whole numbers in the order of the values (-0 as 0), and back. */
__device__ __forceinline__ uint32_t lp_ord(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (uint32_t)((int32_t)u >> 31 | (int32_t)0x80000000);
}
__device__ __forceinline__ float lp_val(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
#define LP_ORD_NINF 0x007fffffu    /* lp_ord(-inf): nothing that is listed is below */
__device__ __forceinline__ uint64_t lp_key(float v, int i) { return (uint64_t)lp_ord(v) << 32 | (uint32_t)~i; }

/* A wave's best entries: `cnt` keys in `l` (LDS, this wave's), and the key that an
 * element must be above, and its value not below tv, to be one. */
struct lp_top {
    uint64_t *l;
    int cnt, k;
    uint64_t t;
    float tv;
    /* the k best of the cnt entries, sorted, to the front: an entry's rank is
     * the number of entries above it */
    __device__ __forceinline__ void compact() {
        const int lane = threadIdx.x & (MM_WAVE - 1), n = cnt;
        asm volatile("" ::: "memory");
        const uint64_t k0 = l[lane], k1 = l[64 + lane];
        int r0 = 0, r1 = 0;
        for (int j = 0; j < n; j += 8) {
            uint64_t b[8];
#pragma unroll
            for (int u = 0; u < 8; u++) b[u] = l[j + u];   /* (n <= LP_LIST, a multiple of 8) */
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const bool in = j + u < n;
                r0 += in && b[u] > k0 ? 1 : 0;
                r1 += in && b[u] > k1 ? 1 : 0;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (lane < n && r0 < k) l[r0] = k0;
        if (64 + lane < n && r1 < k) l[r1] = k1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        cnt = min(n, k);
        if (cnt == k) {
            t = l[k - 1];
            tv = lp_val((uint32_t)(t >> 32));
        }
    }
    /* one key per lane; ok: there is one */
    __device__ __forceinline__ void offer(uint64_t key, bool ok) {
        const bool c = ok && key > t;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(c);
        const int at = cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        if (c) l[at] = key;
        cnt += __builtin_popcountll(mask);
        if (cnt > 64) compact();
    }
    /* a value that at least k of the lanes' values (-inf: none) are not below:
     * the k-th largest, its last 14 bits cleared */
    __device__ __forceinline__ void threshold(float v) {
        const uint32_t o = lp_ord(v);
        uint32_t p = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit >= 1u << 14; bit >>= 1)
            if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(o >= (p | bit))) >= k) p |= bit;
        p = max(p, LP_ORD_NINF);
        t = ((uint64_t)p << 32) - 1;
        tv = lp_val(p);
    }
};

/* A lane's chunk into its (m, R, U). */
__device__ __forceinline__ void lp_add(lp_stat &s, const float (&x)[LP_VPL], float mc) {
    const float mn = fmaxf(s.m, mc), m0 = mn == -INFINITY ? 0.0f : mn;
    float E[2] = {0.0f, 0.0f}, V[2] = {0.0f, 0.0f}, C = 0.0f;
#pragma unroll
    for (int j = 0; j < LP_VPL; j++) {
        const float d = x[j] - m0, e = __expf(d);
        E[j & 1] += d == 0.0f ? 0.0f : e;
        C += d == 0.0f ? 1.0f : 0.0f;
        V[j & 1] = __builtin_fmaf(e, fmaxf(d, LP_DMIN), V[j & 1]);
    }
    const float w = s.m == -INFINITY ? 0.0f : __expf(s.m - mn), old = 1.0f + s.R;
    const float es = E[0] + E[1];
    s.U = w * (s.U + fmaxf(s.m - mn, LP_DMIN) * old) + (V[0] + V[1]);
    s.R = mc > s.m ? old * w + es + (C - 1.0f) : s.R + es + C;
    s.m = mn;
}

/* The row's answers from its whole (m, R, U) and list; lanes of one wave. */
__device__ __forceinline__ void lp_finish(const mm_logprobs_args &a, int t, const lp_stat &s, const lp_top &top) {
    const int lane = threadIdx.x & (MM_WAVE - 1);
    const float lz = log1pf(s.R);
    if (lane == 0) {
        if (a.logprob) {
            const int g = a.targets[t];
            a.logprob[t] = g >= 0 && g < a.n ? (a.logits[(size_t)t * a.stride + g] - s.m) - lz : __builtin_nanf("");
        }
        if (a.entropy) a.entropy[t] = lz - s.U / (1.0f + s.R);
    }
    if (lane < a.n_top) {
        const bool is = lane < top.cnt;
        const uint64_t key = top.l[lane];
        const size_t o = (size_t)t * a.n_top + lane;
        if (a.top_idx) a.top_idx[o] = is ? (int)~(uint32_t)key : -1;
        if (a.top_logprob) a.top_logprob[o] = is ? (lp_val((uint32_t)(key >> 32)) - s.m) - lz : __builtin_nanf("");
    }
}

/* One block per (row t, segment): a 1-D grid of T * nseg blocks.  V: elements
 * per load (4 where every row is 16-byte aligned). */
template <int V>
__device__ __forceinline__ void lp_block(const mm_logprobs_args &a) {
    __shared__ uint64_t ls[LP_WAVES][LP_LIST];
    __shared__ lp_stat ws[LP_WAVES];
    __shared__ int wc[LP_WAVES];
    const int t = (int)(blockIdx.x / (unsigned)a.nseg), seg = (int)(blockIdx.x % (unsigned)a.nseg);
    const int lane = threadIdx.x & (MM_WAVE - 1);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / MM_WAVE);
    const float *x = a.logits + (size_t)t * a.stride;
    const int n = a.n, s0 = seg * a.seg, s1 = (int)min((int64_t)s0 + a.seg, (int64_t)n);
    typedef float vec __attribute__((ext_vector_type(4)));
    /* element j of this lane in the chunk at c is c + at(j); a chunk that the row
     * ends in is read an element at a time, at clamped indices */
    auto at = [&](int j) { return V * (MM_WAVE * (j / V) + lane) + j % V; };
    auto load = [&](int c, float (&v)[LP_VPL]) {
        if (V == 4 && c + LP_CHUNK <= n) {             /* uniform */
#pragma unroll
            for (int u = 0; u < LP_VPL / 4; u++) {
                const vec d = *(const vec *)(x + c + 4 * (MM_WAVE * u + lane));
#pragma unroll
                for (int q = 0; q < 4; q++) v[4 * u + q] = d[q];
            }
        } else {
#pragma unroll
            for (int j = 0; j < LP_VPL; j++) v[j] = x[min(c + at(j), n - 1)];
        }
    };
    lp_stat st = {-INFINITY, -1.0f, 0.0f};
    lp_top top = {ls[w], 0, a.n_top, 0, -INFINITY};
    constexpr int STEP = LP_WAVES * LP_CHUNK;
    const int c0 = s0 + w * LP_CHUNK;
    if (c0 < s1) {
        float v[LP_VPL], nx[LP_VPL];
        load(c0, v);
        for (int c = c0;; c += STEP) {
            const bool more = c + STEP < s1;
            if (more) load(c + STEP, nx);
            if (c + LP_CHUNK > s1) {                   /* uniform: the row ends in it */
#pragma unroll
                for (int j = 0; j < LP_VPL; j++)
                    if (c + at(j) >= s1) v[j] = -INFINITY;
            }
            float mc = v[0];
#pragma unroll
            for (int j = 1; j < LP_VPL; j++) mc = fmaxf(mc, v[j]);
            mc = fmaxf(mc, -INFINITY);                 /* a lane of NaNs only */
            lp_add(st, v, mc);
            if (a.n_top) {
                if (c == c0) top.threshold(mc);
                uint32_t cand = 0;                     /* this lane's elements that may be listed */
#pragma unroll
                for (int j = 0; j < LP_VPL; j++) cand |= v[j] >= top.tv ? 1u << j : 0u;
                while (__builtin_amdgcn_ballot_w64(cand != 0)) {
                    const int j = __builtin_ctz(cand | 1u << (LP_VPL - 1));
                    float e = v[0];
#pragma unroll
                    for (int u = 1; u < LP_VPL; u++) e = j == u ? v[u] : e;
                    const int i = c + V * (MM_WAVE * (j / V) + lane) + j % V;
                    top.offer(lp_key(e, i), cand != 0 && i < s1);
                    cand &= cand - 1;
                }
            }
            if (!more) break;
#pragma unroll
            for (int j = 0; j < LP_VPL; j++) v[j] = nx[j];
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const lp_stat o = {__shfl_xor(st.m, off, MM_WAVE), __shfl_xor(st.R, off, MM_WAVE), __shfl_xor(st.U, off, MM_WAVE)};
        st = lp_merge(st, o);
    }
    /* each wave's list, then (turn 1, wave 0 alone) the waves' lists in one, at
     * most LP_LIST entries */
#pragma unroll 1
    for (int turn = 0; turn < 2; turn++) {
        if (top.cnt) top.compact();
        if (turn) break;
        if (lane == 0) {
            ws[w] = st;
            wc[w] = top.cnt;
        }
        __syncthreads();
        if (w > 0) return;
        for (int u = 1; u < LP_WAVES; u++) {
            st = lp_merge(st, ws[u]);
            const int nu = wc[u];
            if (lane < nu) ls[0][top.cnt + lane] = ls[u][lane];
            top.cnt += nu;
        }
    }
    if (a.nseg == 1) {
        lp_finish(a, t, st, top);
        return;
    }
    const size_t p = blockIdx.x;
    if (lane == 0) *(f32x4 *)(a.part_s + 4 * p) = (f32x4){st.m, st.R, st.U, __int_as_float(top.cnt)};
    if (lane < top.cnt) a.part_k[p * a.n_top + lane] = top.l[lane];
}

extern "C" __global__ __launch_bounds__(64 * LP_WAVES) void mm_logprobs(mm_logprobs_args a) { lp_block<4>(a); }
/* rows that are not 16-byte aligned */
extern "C" __global__ __launch_bounds__(64 * LP_WAVES) void mm_logprobs_1(mm_logprobs_args a) { lp_block<1>(a); }

/* One wave per row merges its segments: lane s has segment s. */
extern "C" __global__ __launch_bounds__(64) void mm_logprobs_final(mm_logprobs_args a) {
    __shared__ uint64_t ls[LP_LIST];
    const int t = blockIdx.x, lane = threadIdx.x;
    const size_t p = (size_t)t * a.nseg + min(lane, a.nseg - 1);
    const f32x4 ps = *(const f32x4 *)(a.part_s + 4 * p);
    const uint64_t *pk = a.part_k + p * a.n_top;
    constexpr int U = 4;                               /* list entries read together */
    uint64_t key[U];
    if (a.n_top)
#pragma unroll
        for (int u = 0; u < U; u++) key[u] = pk[min(u, a.n_top - 1)];
    lp_stat st = {ps.x, ps.y, ps.z};
    int have = __float_as_int(ps.w);
    if (lane >= a.nseg) {
        st = {-INFINITY, -1.0f, 0.0f};
        have = 0;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const lp_stat o = {__shfl_xor(st.m, off, MM_WAVE), __shfl_xor(st.R, off, MM_WAVE), __shfl_xor(st.U, off, MM_WAVE)};
        st = lp_merge(st, o);
    }
    lp_top top = {ls, 0, a.n_top, 0, -INFINITY};
    if (a.n_top) {
        top.threshold(have ? lp_val((uint32_t)(key[0] >> 32)) : -INFINITY);
        /* the lists are sorted: past the first entry that nobody takes nothing follows */
#pragma unroll 1
        for (int j = 0; j < a.n_top; j++) {
            const bool ok = j < have;
            if (!__builtin_amdgcn_ballot_w64(ok && key[0] > top.t)) break;
            top.offer(key[0], ok);
#pragma unroll
            for (int u = 0; u + 1 < U; u++) key[u] = key[u + 1];
            key[U - 1] = pk[min(j + U, a.n_top - 1)];
        }
        if (top.cnt) top.compact();
    }
    lp_finish(a, t, st, top);
}
