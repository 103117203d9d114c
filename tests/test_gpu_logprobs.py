"""Log probabilities, entropies and top alternatives of rows of logits against
64-bit numpy, and the calls that are refused.

Tolerances count fp32 roundings (half a step, 2^-24 relative): a term e^d of R
carries (2 |d| + 2) of them (d, its product with log2 e, the exponential), its
way through the sums at most 8 + n / 4096 + 12 more (a lane's chunk, its chunks,
the merges); with n <= 102,400 and the weighted |d| of these rows below 16 that
is under 96 steps of R, which move log1p(R) by at most 96 R / (1 + R).  A log
probability adds two rounded terms, an entropy U with as many steps of its own.
"""
import ctypes as C

import numpy as np
import pytest

import mlamoe
from hip_graph import Graph

STEP = 2.0 ** -24


def ref(row, targets_row, n_top):
    """(logprob, its tolerance, entropy, its tolerance, top indices, top log
    probabilities, their tolerances) of one row in 64 bits."""
    x = row.astype(np.float64)
    order = [i for i in np.lexsort((np.arange(x.size), -(x + 0.0))) if x[i] == x[i]][:n_top]
    if np.isnan(x).any() or x.max() in (np.inf, -np.inf):
        nan = np.nan
        return nan, 0.0, nan, 0.0, order, [nan] * len(order), [0.0] * len(order)
    m, am = x.max(), int(np.argmax(x))
    d = np.delete(x, am) - m
    e = np.exp(d)
    R, U = e.sum(), np.where(e > 0, e * np.where(np.isfinite(d), d, 0.0), 0.0).sum()
    lz = np.log1p(R)
    base = 96.0 * R / (1.0 + R)
    H = lz - U / (1.0 + R)

    def lp(i):
        v = x[i] - m
        return v - lz, STEP * (base + 4.0 * (abs(v) + lz)) if np.isfinite(v) else 0.0
    t = targets_row
    own = lp(t) if 0 <= t < x.size else (np.nan, 0.0)
    tops = [lp(i) for i in order]
    return own[0], own[1], H, STEP * (base + 128.0 * H), order, [v for v, _ in tops], [v for _, v in tops]


def same(got, want, tol, what):
    if np.isnan(want):
        assert np.isnan(got), what
    elif np.isinf(want):
        assert got == want, what
    else:
        assert abs(float(got) - want) <= tol, (what, got, want, tol)


def check(ctx, logits, targets, n_top, n=None):
    T, stride = logits.shape
    n = stride if n is None else n
    print(f"logprobs T={T} n={n} stride={stride} top={n_top}", flush=True)
    lp, H, idx, tlp = ctx.token_logprobs(logits, targets, n_top, n)
    for t in range(T):
        w, wt, h, ht, order, tops, ttol = ref(logits[t, :n], int(targets[t]), n_top)
        same(lp[t], w, wt, ("logprob", t))
        same(H[t], h, ht, ("entropy", t))
        assert list(idx[t, :len(order)]) == order, ("top", t)
        for j, (v, tol) in enumerate(zip(tops, ttol)):
            same(tlp[t, j], v, tol, ("top_logprob", t, j))
        assert np.all(idx[t, len(order):] == -1) and np.all(np.isnan(tlp[t, len(order):])), ("rest", t)
    return lp, H, idx, tlp


@pytest.fixture(scope="module")
def ctx():
    c = mlamoe.Context(0)
    yield c
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,pad,top", [
    (1, 1, 0, 1), (1, 2, 0, 2), (1, 3, 0, 1), (2, 3, 2, 3), (3, 5, 0, 5), (1, 63, 0, 32), (2, 64, 0, 32), (4, 65, 3, 20),
    (3, 1023, 0, 7), (3, 1025, 1, 7), (2, 4095, 1, 20), (2, 4096, 0, 20), (2, 4097, 3, 20), (1, 4100, 0, 1), (5, 8193, 7, 32),
    (1, 32003, 29, 5), (7, 32003, 0, 5), (1, 102400, 0, 20), (3, 102400, 0, 0), (1100, 4099, 1, 3), (1030, 640, 0, 1)])
def test_shapes(ctx, T, n, pad, top):
    """Lengths around a vector, a lane's chunk, a wave's, a block's pass and a
    segment; rows that are and are not 16-byte aligned; one and several
    segments per row; NaN in the padding, which is not part of a row."""
    rng = np.random.default_rng(1000 * T + n + top)
    x = (rng.standard_normal((T, n + pad)) * 3.0).astype(np.float32)
    x[:, n:] = np.nan
    check(ctx, x, rng.integers(0, n, T), top, n)


@pytest.mark.gpu
def test_odd_base(ctx):
    """Logits that begin at an odd float of an allocation."""
    rng = np.random.default_rng(5)
    n, off = 5003, 3
    x = rng.standard_normal(n).astype(np.float32)
    buf = ctx.to_device(np.concatenate([np.full(off, np.nan, np.float32), x, np.full(5, np.nan, np.float32)]))
    t, lp, idx = ctx.to_device(np.array([17], np.int32)), ctx.empty((1,), np.float32), ctx.empty((1, 4), np.int32)
    buf.ptr += 4 * off
    ctx.token_logprobs_dev(1, buf, n, n, t, lp, None, 4, idx, None)
    buf_lp, got = lp.download(), idx.download()
    buf.ptr -= 4 * off
    w, wt, _, _, order, _, _ = ref(x, 17, 4)
    same(buf_lp[0], w, wt, "logprob")
    assert list(got[0]) == order


@pytest.mark.gpu
@pytest.mark.parametrize("n", [70, 1500, 9001])
def test_rows_that_are_special(ctx, n):
    """Masked vocabularies (-inf, the type's lowest value), one token left, none
    left, NaN, +inf, all equal, -0 beside 0, ascending and descending rows,
    rows of one certain token."""
    rng = np.random.default_rng(n)
    r = []
    base = (rng.standard_normal(n) * 2.0).astype(np.float32)
    masked = np.full(n, -np.inf, np.float32)
    masked[[3, 40, n - 1]] = [1.0, 2.0, 1.5]
    one = np.full(n, -np.inf, np.float32)
    one[n // 2] = -7.0
    low = np.full(n, np.finfo(np.float32).min, np.float32)
    low[[5, n - 2]] = [0.25, 0.5]
    nan, inf = base.copy(), base.copy()
    nan[n // 3] = np.nan
    inf[n // 4] = np.inf
    zeros = np.where(np.arange(n) % 3 == 0, np.float32(-0.0), np.float32(0.0))
    sure = base.copy()
    sure[n - 1] = 40.0
    surer = np.full(n, -30.0, np.float32)
    surer[1] = 0.0
    top = np.where(np.arange(n) < n - 5, np.nan, base).astype(np.float32)
    big = base * np.float32(1e37)
    r = [masked, one, np.full(n, -np.inf, np.float32), low, nan, inf, np.full(n, np.inf, np.float32), np.full(n, 1.25, np.float32),
         zeros, np.sort(base), np.sort(base)[::-1], sure, surer, top, np.full(n, np.nan, np.float32), big,
         np.where(np.arange(n) % 2 == 0, -np.inf, base)]
    x = np.stack([np.asarray(v, np.float32) for v in r])
    targets = np.array([40, 0, 5, 5, 1, 1, 1, n - 1, 0, 0, 0, n - 1, 1, n - 1, 2, 9, 0])
    check(ctx, x, targets, 20)


@pytest.mark.gpu
def test_small_probabilities_are_exact(ctx):
    """One token of probability 1 - 1e-9: its log probability and the entropy
    to full relative precision (a sum that held the 1 would give 0)."""
    n = 1000
    x = np.full((1, n), -27.0, np.float32)
    x[0, 10] = 0.0
    lp, H, idx, _ = ctx.token_logprobs(x, [10], 1)
    R = 999.0 * np.exp(-27.0)
    assert idx[0, 0] == 10
    # 96 steps of R as above; |d| = 27: 56 of them in each term
    assert abs(lp[0] / -np.log1p(R) - 1.0) < 128 * STEP
    assert abs(H[0] / (np.log1p(R) + 27.0 * R / (1 + R)) - 1.0) < 192 * STEP


@pytest.mark.gpu
def test_targets_outside(ctx):
    x = np.random.default_rng(3).standard_normal((4, 100)).astype(np.float32)
    lp, H, _, _ = ctx.token_logprobs(x, [-1, 100, 2147483647, 99], 0)
    assert np.all(np.isnan(lp[:3])) and np.isfinite(lp[3]) and np.all(np.isfinite(H))


@pytest.mark.gpu
@pytest.mark.parametrize("T,n", [(2, 3001), (2, 50000)])
def test_outputs_on_their_own(ctx, T, n):
    """Each output alone is what it is among all, bit for bit, and nothing else
    is written; the logits stay as they were."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((T, n)).astype(np.float32)
    t = rng.integers(0, n, T).astype(np.int32)
    full = ctx.token_logprobs(x, t, 6)
    dl, dt = ctx.to_device(x), ctx.to_device(t)
    shapes = {"logprob": ((T,), np.float32), "entropy": ((T,), np.float32), "top_idx": ((T, 6), np.int32), "top_logprob": ((T, 6), np.float32)}
    for (name, (shape, dtype)), want in zip(shapes.items(), full):
        guard = np.full(int(np.prod(shape)) + 8, 77, dtype)
        out = ctx.to_device(guard)
        ctx.token_logprobs_dev(T, dl, n, n, dt if name == "logprob" else None, n_top=6 if "top" in name else 0, **{name: out})
        got = out.download()
        assert np.array_equal(got[:-8].reshape(shape).view(np.uint32), want.view(np.uint32)), name
        assert np.all(got[-8:] == 77), name
    assert np.array_equal(dl.download(), x)


@pytest.mark.gpu
def test_top_is_the_argmax(ctx):
    """The first alternative is mm_argmax_dev's token, ties included."""
    rng = np.random.default_rng(8)
    x = rng.integers(-20, 20, (9, 7001)).astype(np.float32)
    _, _, idx, _ = ctx.token_logprobs(x, None, 1)
    assert np.array_equal(idx[:, 0], ctx.argmax(x))


@pytest.mark.gpu
def test_far_rows(ctx):
    """Rows past 2^31 bytes of a padded array."""
    n, stride, T = 130, 1 << 20, 600
    x = ctx.alloc(4 * T * stride)
    ctx.fill(x, T * stride, mlamoe.MM_FILL_F32_NORMAL, 4)
    t, lp, idx = ctx.to_device(np.full(T, 7, np.int32)), ctx.empty((T,), np.float32), ctx.empty((T, 2), np.int32)
    ctx.token_logprobs_dev(T, x, stride, n, t, lp, None, 2, idx, None)
    got, tops, base = lp.download(), idx.download(), x.ptr
    for r in (0, 511, 512, 513, T - 1):
        x.ptr = base + 4 * stride * r
        row = x.download(np.float32, (n,))
        x.ptr = base
        w, wt, _, _, order, _, _ = ref(row, 7, 2)
        same(got[r], w, wt, r)
        assert tops[r].tolist() == order


@pytest.mark.gpu
def test_captured(ctx):
    """Two graphs with workspaces of their own, replayed in turn between eager
    calls: every replay gives the eager result of the inputs it meets; without
    a workspace a captured call is refused."""
    T, n, k = 3, 60000, 9
    nbytes = mlamoe.token_logprobs_workspace(T, n, k)
    assert nbytes > 0
    x = [ctx.empty((T, n), np.float32) for _ in range(2)]
    tg = ctx.to_device(np.arange(T, dtype=np.int32))
    outs = [[ctx.empty((T,), np.float32), ctx.empty((T,), np.float32), ctx.empty((T, k), np.int32), ctx.empty((T, k), np.float32)]
            for _ in range(3)]
    ws = [ctx.alloc(nbytes) for _ in range(2)]

    def call(i, o, w):
        ctx.token_logprobs_dev(T, x[i], n, n, tg, o[0], o[1], k, o[2], o[3], w)

    def record(i):
        with pytest.raises(mlamoe.MMError) as e:
            call(i, outs[i], None)
        assert e.value.status == -5
        call(i, outs[i], ws[i])
    graphs = [Graph(ctx, lambda i=i: record(i)) for i in range(2)]
    for rep in range(4):
        for i, v in enumerate(x):
            ctx.fill(v, T * n, mlamoe.MM_FILL_F32_NORMAL, 10 * rep + i)
        for g in graphs:
            g.replay()
        for i in range(2):
            call(i, outs[2], None)
            for a, b in zip(outs[i], outs[2]):
                assert np.array_equal(a.download().view(np.uint32), b.download().view(np.uint32)), (rep, i)
    for g in graphs:
        g.close()


@pytest.mark.gpu
def test_refusals(ctx):
    L = mlamoe.lib()
    x, o = ctx.to_device(np.zeros((2, 64), np.float32)), ctx.to_device(np.full(64, 5.0, np.float32))

    def call(T=2, lg=x.ptr, stride=64, n=64, tg=None, lp=None, H=o.ptr, k=0, ti=None, tv=None, ws=None, nb=0):
        return L.mm_token_logprobs_dev(ctx.h, T, lg, stride, n, tg, lp, H, k, ti, tv, ws, nb)
    assert call(lg=None) == -1 and call(T=-1) == -1 and call(n=0) == -1 and call(stride=63) == -1
    assert call(k=65) == -1 and call(k=-1) == -1 and call(k=33) == -2 and call(lg=x.ptr + 2) == -1
    assert call(lp=o.ptr) == -1                                   # no targets
    big = ctx.empty((1, 9000), np.float32)
    assert call(T=1, lg=big.ptr, stride=9000, n=9000, ws=o.ptr, nb=8) == -1    # a workspace too small
    assert call(T=1, lg=big.ptr, stride=9000, n=9000, ws=o.ptr + 4, nb=1 << 20) == -1
    assert call(T=0, lg=None) == 0 and call(H=None) == 0
    assert np.all(o.download() == 5.0)


def test_refusals_without_a_gpu():
    L = mlamoe.lib()
    assert L.mm_token_logprobs_dev(None, 1, None, 1, 1, None, None, None, 0, None, None, None, 0) == -1
    assert L.mm_token_logprobs_workspace(1, 10, 1, None) == -1
    b = C.c_size_t(7)
    for T, n, k, want in ((-1, 10, 1, -1), (1, 0, 0, -1), (1, 10, 11, -1), (1, 100, 33, -2), (1, (1 << 30) + 1, 1, -2), (0, 10, 1, 0)):
        assert L.mm_token_logprobs_workspace(T, n, k, C.byref(b)) == want, (T, n, k)
        assert b.value == 0
    assert mlamoe.token_logprobs_workspace(4000, 102400, 20) == 0     # a row a block: none needed
    assert mlamoe.token_logprobs_workspace(1, 102400, 20) > 0


def test_more_rows_than_a_grid_holds_are_refused():
    b = C.c_size_t(7)
    assert mlamoe.lib().mm_token_logprobs_workspace((1 << 23) + 1, 10, 1, C.byref(b)) == -2 and b.value == 0
    assert mlamoe.token_logprobs_workspace(1 << 23, 10, 1) == 0


@pytest.mark.gpu
def test_host_form_refuses_arrays_too_short(ctx):
    x = np.zeros((3, 64), np.float32)
    for call in (lambda: ctx.token_logprobs(x, [1, 2], 1), lambda: ctx.token_logprobs(x, [1, 2, 3], 1, 65), lambda: ctx.token_logprobs(x[:1], None, 1, 100)):
        with pytest.raises(mlamoe.MMError) as e:
            call()
        assert e.value.status == -1
