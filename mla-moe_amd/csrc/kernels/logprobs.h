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
 * end.  The n_top largest are kept beside: a list in LDS, sorted by (value
 * descending, index ascending), and its last entry as the threshold that an
 * element must beat; a wave meets few such elements after its first chunk,
 * whose threshold is the n_top-th of the lanes' maxima.
 */
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

/* (v, i) before (bv, bi): larger, or equal at a lower index */
__device__ __forceinline__ bool lp_before(float v, int i, float bv, int bi) {
    return v > bv || (v == bv && i < bi);
}

/* A wave's best entries: `cnt` of them in lv / li (LDS, this wave's), and what
 * an element must come before to be one. */
struct lp_top {
    float *lv;
    int *li;
    int cnt, k;
    float tv;
    int ti;
    /* the k best of the cnt entries, sorted, to the front: each entry's rank
     * is the number of entries before it */
    __device__ __forceinline__ void compact() {
        const int lane = threadIdx.x & (MM_WAVE - 1);
        const int n = cnt;
        asm volatile("" ::: "memory");
        const float v0 = lv[min(lane, LP_LIST - 1)], v1 = lv[64 + lane];
        const int i0 = li[lane], i1 = li[64 + lane];
        int r0 = 0, r1 = 0;
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const float bv = lv[j];
            const int bi = li[j];
            r0 += lp_before(bv, bi, v0, i0) ? 1 : 0;
            r1 += lp_before(bv, bi, v1, i1) ? 1 : 0;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (lane < n && r0 < k) {
            lv[r0] = v0;
            li[r0] = i0;
        }
        if (64 + lane < n && r1 < k) {
            lv[r1] = v1;
            li[r1] = i1;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        cnt = min(n, k);
        if (cnt == k) {
            tv = lv[k - 1];
            ti = li[k - 1];
        }
    }
    /* one element per lane; ok: there is one */
    __device__ __forceinline__ void offer(float v, int i, bool ok) {
        const bool c = ok && lp_before(v, i, tv, ti);
        const uint64_t mask = __builtin_amdgcn_ballot_w64(c);
        if (!mask) return;
        const int at = cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        if (c) {
            lv[at] = v;
            li[at] = i;
        }
        cnt += __builtin_popcountll(mask);
        if (cnt > 64) compact();
    }
    /* the k-th largest of the lanes' values (-inf: none): at least k elements
     * are not below it */
    __device__ __forceinline__ void threshold(float v) {
        const int lane = threadIdx.x & (MM_WAVE - 1);
        int r = 0;
#pragma unroll
        for (int l = 0; l < MM_WAVE; l++) {
            const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
            r += lp_before(o, l, v, lane) ? 1 : 0;
        }
        const uint64_t at = __builtin_amdgcn_ballot_w64(r == k - 1);
        tv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), __builtin_ctzll(at)));
        ti = 0x7fffffff;
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
        const size_t o = (size_t)t * a.n_top + lane;
        if (a.top_idx) a.top_idx[o] = is ? top.li[lane] : -1;
        if (a.top_logprob) a.top_logprob[o] = is ? (top.lv[lane] - s.m) - lz : __builtin_nanf("");
    }
}

/* One block per (row t, segment): a 1-D grid of T * nseg blocks.  V: elements
 * per load (4 where every row is 16-byte aligned). */
template <int V>
__device__ __forceinline__ void lp_block(const mm_logprobs_args &a) {
    __shared__ float lv[LP_WAVES][LP_LIST];
    __shared__ int li[LP_WAVES][LP_LIST];
    __shared__ lp_stat ws[LP_WAVES];
    __shared__ int wc[LP_WAVES];
    const int t = (int)(blockIdx.x / (unsigned)a.nseg), seg = (int)(blockIdx.x % (unsigned)a.nseg);
    const int lane = threadIdx.x & (MM_WAVE - 1);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / MM_WAVE);
    const float *x = a.logits + (size_t)t * a.stride;
    const int n = a.n, s0 = seg * a.seg, s1 = (int)min((int64_t)s0 + a.seg, (int64_t)n);
    constexpr int NL = LP_VPL / V;
    typedef float vec __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    /* element j of this lane in the chunk at c: c + V (64 (j / V) + lane) + j % V.
     * With V = 4 the loads stop at the row's last whole vector; its up to 3
     * further elements are offered on their own below. */
    const int nv = V == 1 ? n : n / V * V;
    auto load = [&](int c, float (&v)[LP_VPL]) {
#pragma unroll
        for (int u = 0; u < NL; u++) {
            const int i = c + V * (MM_WAVE * u + lane);
            if (V == 1) {
                v[u] = x[min(i, n - 1)];
            } else {
                const vec d = *(const vec *)(x + min(i, nv - V));
#pragma unroll
                for (int q = 0; q < V; q++) v[V * u + q] = d[q];
            }
        }
    };
    lp_stat st = {-INFINITY, -1.0f, 0.0f};
    lp_top top = {lv[w], li[w], 0, a.n_top, -INFINITY, 0x7fffffff};
    const int e1 = min(s1, nv);                       /* chunks cover [s0, e1) */
    auto take = [&](int c, float (&v)[LP_VPL], bool first) {
        if (c + LP_CHUNK > e1) {                      /* uniform: the segment's last chunk */
#pragma unroll
            for (int j = 0; j < LP_VPL; j++)
                if (c + V * (MM_WAVE * (j / V) + lane) + j % V >= e1) v[j] = -INFINITY;
        }
        float mc = v[0];
#pragma unroll
        for (int j = 1; j < LP_VPL; j++) mc = fmaxf(mc, v[j]);
        mc = fmaxf(mc, -INFINITY);                    /* a lane of NaNs only */
        lp_add(st, v, mc);
        if (a.n_top == 0) return;
        if (first) top.threshold(mc);
        if (!__builtin_amdgcn_ballot_w64(mc >= top.tv)) return;
#pragma unroll
        for (int j = 0; j < LP_VPL; j++) {
            const int i = c + V * (MM_WAVE * (j / V) + lane) + j % V;
            if (__builtin_amdgcn_ballot_w64(v[j] >= top.tv)) top.offer(v[j], i, i < e1);
        }
    };
    constexpr int STEP = LP_WAVES * LP_CHUNK;
    const int c0 = s0 + w * LP_CHUNK;
    if (c0 < e1) {
        float va[LP_VPL], vb[LP_VPL];
        load(c0, va);
        for (int c = c0; c < e1; c += 2 * STEP) {
            load(c + STEP, vb);                       /* past the end: clamped, not used */
            take(c, va, c == c0);
            if (c + STEP >= e1) break;
            load(c + 2 * STEP, va);
            take(c + STEP, vb, false);
        }
    }
    if (V > 1 && nv < n && s1 == n && w == 0) {       /* the row's last n % V elements */
        const bool ok = lane < n - nv;
        const float v = ok ? x[min(nv + lane, n - 1)] : -INFINITY;
        float one[LP_VPL];
#pragma unroll
        for (int j = 0; j < LP_VPL; j++) one[j] = j == 0 ? v : -INFINITY;
        lp_add(st, one, fmaxf(v, -INFINITY));
        if (a.n_top) top.offer(v, nv + lane, ok);
    }
    if (top.cnt) top.compact();
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const lp_stat o = {__shfl_xor(st.m, off, MM_WAVE), __shfl_xor(st.R, off, MM_WAVE), __shfl_xor(st.U, off, MM_WAVE)};
        st = lp_merge(st, o);
    }
    if (lane == 0) {
        ws[w] = st;
        wc[w] = top.cnt;
    }
    __syncthreads();
    if (w > 0) return;
    for (int u = 1; u < LP_WAVES; u++) st = lp_merge(st, ws[u]);
    for (int u = 1; u < LP_WAVES; u++) {              /* the waves' lists, at most LP_LIST entries */
        const int nu = wc[u];
        if (lane < nu) {
            lv[0][top.cnt + lane] = lv[u][lane];
            li[0][top.cnt + lane] = li[u][lane];
        }
        top.cnt += nu;
    }
    if (top.cnt) top.compact();
    if (a.nseg == 1) {
        lp_finish(a, t, st, top);
        return;
    }
    const size_t p = blockIdx.x;
    if (lane == 0) {
        float *ps = a.part_s + 4 * p;
        ps[0] = st.m;
        ps[1] = st.R;
        ps[2] = st.U;
        ps[3] = __int_as_float(top.cnt);
    }
    if (lane < top.cnt) {
        a.part_v[p * a.n_top + lane] = top.lv[lane];
        a.part_i[p * a.n_top + lane] = top.li[lane];
    }
}

extern "C" __global__ __launch_bounds__(64 * LP_WAVES) void mm_logprobs(mm_logprobs_args a) { lp_block<4>(a); }
/* rows that are not 16-byte aligned */
extern "C" __global__ __launch_bounds__(64 * LP_WAVES) void mm_logprobs_1(mm_logprobs_args a) { lp_block<1>(a); }

/* One wave per row merges its segments: lane s has segment s. */
extern "C" __global__ __launch_bounds__(64) void mm_logprobs_final(mm_logprobs_args a) {
    __shared__ float lv[LP_LIST];
    __shared__ int li[LP_LIST];
    const int t = blockIdx.x, lane = threadIdx.x;
    const size_t p = (size_t)t * a.nseg + min(lane, a.nseg - 1);
    const f32x4 ps = *(const f32x4 *)(a.part_s + 4 * p);
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
    lp_top top = {lv, li, 0, a.n_top, -INFINITY, 0x7fffffff};
    if (a.n_top) {
        const float *pv = a.part_v + p * a.n_top;
        const int32_t *pi = a.part_i + p * a.n_top;
        top.threshold(have ? pv[0] : -INFINITY);
        for (int j = 0; j < a.n_top; j++) {           /* the lists are sorted: past the last taker nothing follows */
            const bool ok = j < have;
            const float v = ok ? pv[j] : -INFINITY;
            const int i = ok ? pi[j] : 0x7fffffff;
            if (!__builtin_amdgcn_ballot_w64(ok && lp_before(v, i, top.tv, top.ti))) break;
            top.offer(v, i, ok);
        }
        if (top.cnt) top.compact();
    }
    lp_finish(a, t, st, top);
}
