"""Absorbed decode over a shared prefix and through a sliding window with sinks,
against the attention's formula in 64-bit numpy on the same bf16 cache.

Tolerances.  A bf16 rounding is off by at most half a step, 2^-8 of a value, so
an fp32 operand that travels as a bf16 pair by 2^-16.

Each value: the absorbed query as a product's result and as an operand, 2^-15; a
score sums 2 x 576 products in fp32, taken as the root of that many roundings of
2^-24, under 2^-18 -- in all under 1.25 x 2^-15 of sum |q c| scale.  With ds the
largest such error of a row, a weight is off by 2 ds of itself and by its pair's
2^-16, the latent context as an operand by 2^-16: under (2 ds + 1.25 x 2^-15)
sum_r |W_UV| sum_k a_k |c_k| in all.

The whole row, since that bound lets roundings add up that do not: independent
roundings of at most 2^-16 add in squares, each with a third of its largest
square.  A score is off by sqrt(2 / 3) 2^-16 sqrt(sum (q c)^2) scale =: sqrt(2 / 3)
2^-16 s, a weight by twice that, its pair and the latent context's by 2^-16 / sqrt(3)
each: under (2 + 2 s) 2^-16 of the row's norm.  A product that lost its low
halves would be off by 2^-9 of it.
"""
import ctypes as C

import numpy as np
import pytest

import mlamoe
from hip_graph import Graph
from mlamoe import synth

KVL, QKR = 512, 64
NAN16 = np.uint16(0x7FC0)


def attend(q, kv_b, keys, NH, QKN, VHD):
    """One row q [NH, QKN + QKR] over keys [n, KVL + QKR] (fp64): ctx [NH, VHD],
    its tolerance per value and that of its norm."""
    w = kv_b.reshape(NH, QKN + VHD, KVL)
    if keys.shape[0] == 0:
        return np.zeros((NH, VHD)), np.zeros((NH, VHD)), 0.0
    scale = 1.0 / np.sqrt(QKN + QKR)
    qa = np.einsum("hd,hdr->hr", q[:, :QKN], w[:, :QKN])
    full = np.concatenate([qa, q[:, QKN:]], 1)
    s = full @ keys.T * scale
    # the absorbed query is itself a sum: its error counts by its terms
    mag = np.concatenate([np.einsum("hd,hdr->hr", np.abs(q[:, :QKN]), np.abs(w[:, :QKN])), np.abs(q[:, QKN:])], 1)
    ds = 1.25 * 2.0 ** -15 * (mag @ np.abs(keys).T).max(1) * scale
    a = np.exp(s - s.max(1, keepdims=True))
    a /= a.sum(1, keepdims=True)
    lat, lmag = a @ keys[:, :KVL], a @ np.abs(keys[:, :KVL])
    out = np.einsum("hvr,hr->hv", w[:, QKN:], lat)
    rms = np.sqrt((full ** 2 @ (keys ** 2).T).max()) * scale
    return (out, (2.0 * ds[:, None] + 1.25 * 2.0 ** -15) * np.einsum("hvr,hr->hv", np.abs(w[:, QKN:]), lmag),
            (2.0 + 2.0 * rms) * 2.0 ** -16)


def close(got, want, what):
    want, tol, norm = want
    assert np.all(np.isfinite(got)), what
    bad = np.abs(got - want) - tol
    assert bad.max() <= 0, (what, float(np.abs(got - want).max()), float(tol.max()))
    off = np.linalg.norm(got - want)
    assert off <= norm * np.linalg.norm(want), (what, off / np.linalg.norm(want), norm)


def near(a, b):
    """Two forms of one product, each within the row bound (s is under 3 here)."""
    assert np.linalg.norm(a - b) <= 2 * 8 * 2.0 ** -16 * np.linalg.norm(b)


def f64(a):
    return synth.bf16_to_f32(a).astype(np.float64)


def weights(rng, NH, QKN, VHD):
    return synth.normal_bf16(rng, (NH * (QKN + VHD), KVL), 0.02)


def loaded(NH, QKN=128, VHD=128, seed=0):
    ctx = mlamoe.Context(0)
    kv_b = weights(np.random.default_rng(seed), NH, QKN, VHD)
    ctx.mla_init(NH, QKN, QKR, KVL, VHD)
    ctx.mla_load_layer(0, kv_b)
    return ctx, f64(kv_b)


def poisoned(rng, B, L, lens):
    """Caches whose rows past each length are NaN."""
    c = synth.normal_bf16(rng, (B, L, KVL + QKR), 1.0)
    for b, n in enumerate(lens):
        c[b, max(n, 0):] = NAN16
    return c


def prefix_case(NH, B, P, L, lens=None, QKN=128, VHD=128, seed=1, qstd=2.0):
    print(f"prefix NH={NH} B={B} P={P} L={L} lens={lens}", flush=True)
    rng = np.random.default_rng(seed)
    q = synth.normal_f32(rng, (B, NH, QKN + QKR), qstd)
    prefix = synth.normal_bf16(rng, (P, KVL + QKR), 1.0) if P else None
    n = list(lens) if lens is not None else [L] * B
    cache = poisoned(rng, B, L, n) if L else None
    ctx, kv_b = loaded(NH, QKN, VHD, seed)
    with ctx:
        got = ctx.mla_prefix_decode(0, q, prefix, cache, lens)
    for b in range(B):
        own = cache[b, :min(max(n[b], 0), L)] if L else np.zeros((0, KVL + QKR), np.uint16)
        keys = np.concatenate([f64(prefix), f64(own)]) if P else f64(own)
        close(got[b].reshape(NH, VHD), attend(q[b].astype(np.float64), kv_b, keys, NH, QKN, VHD), ("ctx", b))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("P", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 513, 1000])
def test_prefix_lengths(P):
    prefix_case(16, 5, P, 7, seed=P)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2, 3, 4, 5, 8, 9, 17, 33, 64])
def test_prefix_batches(B):
    prefix_case(16, B, 700, 40, [40 - 5 * b % 40 for b in range(B)], seed=100 + B)


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,QKN,VHD", [(1, 3, 128, 128), (3, 7, 32, 40), (8, 2, 128, 128), (15, 9, 64, 16), (17, 5, 128, 128), (20, 23, 192, 256), (40, 3, 128, 128)])
def test_prefix_heads(NH, B, QKN, VHD):
    prefix_case(NH, B, 333, 50, [(37 * b) % 51 for b in range(B)], QKN, VHD, seed=NH)


@pytest.mark.gpu
@pytest.mark.parametrize("P,L,lens", [(100, 0, None), (0, 90, None), (0, 90, [0, 90, 1, 0, -5]), (64, 90, [0, 0, 0, 0, 0]), (33, 90, [0, 500, -1, 2147483647, 17]), (0, 0, None)])
def test_prefix_empty_parts(P, L, lens):
    """No prefix, no own rows, lengths outside [0, kv_len]: rows without any key
    give zeros."""
    got = prefix_case(16, 5, P, L, lens, seed=7 + P + L)
    if not P:
        for b, n in enumerate(lens if lens is not None else [L] * 5):
            assert (np.abs(got[b]).max() == 0) == (n <= 0)


@pytest.mark.gpu
@pytest.mark.parametrize("B,P,L", [(64, 4097, 130), (3, 40000, 5), (130, 1111, 20), (520, 260, 9)])
def test_prefix_large(B, P, L):
    prefix_case(16, B, P, L, [L - b % L for b in range(B)], seed=B + P)


@pytest.mark.gpu
def test_prefix_peaked_scores():
    """Scores tens apart: running maxima move, in the prefix and after it."""
    prefix_case(16, 9, 900, 60, seed=31, qstd=30.0)


@pytest.mark.gpu
def test_prefix_is_the_whole_cache():
    """A prefix and own rows are what mm_mla_absorbed_decode_dev computes of
    them in one cache."""
    rng = np.random.default_rng(11)
    NH, B, P, L = 16, 6, 777, 60
    lens = np.array([60, 1, 33, 16, 59, 2], np.int32)
    q = synth.normal_f32(rng, (B, NH, 192))
    prefix, cache = synth.normal_bf16(rng, (P, 576), 1.0), synth.normal_bf16(rng, (B, L, 576), 1.0)
    ctx, _ = loaded(NH)
    with ctx:
        a = ctx.mla_prefix_decode(0, q, prefix, cache, lens)
        whole = np.concatenate([np.broadcast_to(prefix, (B, P, 576)), cache], 1)
        b = ctx.mla_absorbed_decode(0, q, whole, P + L, lens + P, want_probs=False)[0]
    near(a, b)


@pytest.mark.gpu
def test_prefix_rows_in_groups(monkeypatch):
    """Partials over the cap: the rows go in groups, the same bits."""
    a = prefix_case(16, 21, 300, 80, [80 - 3 * b for b in range(21)], seed=40)
    monkeypatch.setenv("MLAMOE_MLA_PART_MAX", str(1 << 20))
    b = prefix_case(16, 21, 300, 80, [80 - 3 * b for b in range(21)], seed=40)
    assert np.array_equal(a, b)


def window_case(NH, B, rows, L, sinks, window, lens=None, QKN=128, VHD=128, seed=2, qstd=2.0):
    print(f"window NH={NH} B={B} rows={rows} L={L} sinks={sinks} window={window} lens={lens}", flush=True)
    rng = np.random.default_rng(seed)
    q = synth.normal_f32(rng, (B, rows, NH, QKN + QKR), qstd)
    n = list(lens) if lens is not None else [L] * B
    cache = poisoned(rng, B, L, n)
    for b in range(B):                    # keys that no row sees
        first = min(max(n[b], 0), L) - rows + 1 - window
        if first > sinks:
            cache[b, sinks:first] = NAN16
    ctx, kv_b = loaded(NH, QKN, VHD, seed)
    with ctx:
        got = ctx.mla_window_decode(0, q, cache, sinks, window, lens)
    for b in range(B):
        for r in range(rows):
            p = min(max(n[b], 0), L) - rows + r
            at = np.arange(max(p + 1, 0))
            keys = f64(cache[b, at[(at < sinks) | (at > p - window)]])
            close(got[b, r].reshape(NH, VHD), attend(q[b, r].astype(np.float64), kv_b, keys, NH, QKN, VHD), ("ctx", b, r))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("sinks,window", [(0, 1), (0, 16), (1, 1), (4, 100), (4, 64), (17, 33), (0, 999), (4, 1000), (64, 5000), (1000, 1), (3000, 7), (4, 2147483647)])
def test_window_sizes(sinks, window):
    window_case(16, 3, 1, 1000, sinks, window, [1000, 5, 640], seed=sinks + window % 1000)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 3, 4, 5, 8, 17, 70])
def test_window_rows(rows):
    """Drafted tokens and prompt chunks: each row its own window."""
    window_case(16, 2, rows, 400, 4, 90, [400, 150], seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,lens", [(1, [0, 1, 2, -3, 99, 100]), (5, [0, 1, 4, 5, 6, 100])])
def test_window_rows_before_the_start(rows, lens):
    """Sequences shorter than their rows: rows before position 0 give zeros."""
    got = window_case(16, 6, rows, 100, 2, 10, lens, seed=50)
    for b, n in enumerate(lens):
        for r in range(rows):
            assert (np.abs(got[b, r]).max() == 0) == (min(max(n, 0), 100) - rows + r < 0)


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,rows,QKN,VHD", [(3, 4, 1, 32, 40), (20, 13, 3, 192, 256), (17, 2, 9, 128, 128), (40, 2, 2, 128, 128)])
def test_window_heads(NH, B, rows, QKN, VHD):
    window_case(NH, B, rows, 700, 7, 211, [700 - 41 * b for b in range(B)], QKN, VHD, seed=60 + NH)


@pytest.mark.gpu
@pytest.mark.parametrize("B,rows,L,window", [(64, 1, 2500, 2100), (1, 200, 900, 256), (3, 180, 500, 130), (1, 520, 600, 64)])
def test_window_large(B, rows, L, window):
    window_case(16, B, rows, L, 4, window, [L - (7 * b) % (L // 4) for b in range(B)], seed=70 + B + rows)


@pytest.mark.gpu
def test_window_peaked_scores():
    window_case(16, 2, 6, 800, 4, 300, seed=77, qstd=30.0)


@pytest.mark.gpu
def test_window_that_sees_all_is_the_absorbed_decode():
    rng = np.random.default_rng(12)
    lens = np.array([300, 17, 1], np.int32)
    q, cache = synth.normal_f32(rng, (3, 1, 16, 192)), synth.normal_bf16(rng, (3, 300, 576), 1.0)
    ctx, _ = loaded(16)
    with ctx:
        a = ctx.mla_window_decode(0, q, cache, 0, 300, lens)[:, 0]
        b = ctx.mla_absorbed_decode(0, q[:, 0], cache, 300, lens, want_probs=False)[0]
    near(a, b)


@pytest.mark.gpu
def test_window_rows_in_groups(monkeypatch):
    """Partials over the cap: groups that cut a sequence's rows, the same bits."""
    lens = [900, 333, 40]
    a = window_case(16, 3, 7, 900, 4, 700, lens, seed=80)
    monkeypatch.setenv("MLAMOE_MLA_PART_MAX", str(3 << 20))
    b = window_case(16, 3, 7, 900, 4, 700, lens, seed=80)
    assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B", [(64, 2), (128, 1), (32, 2), (64, 3)])
def test_few_rows_in_groups(monkeypatch, NH, B):
    """Few rows of many heads, whose merge shares a row's chunks between waves:
    one row per group, the same bits."""
    a = prefix_case(NH, B, 1500, 40, [40 - b for b in range(B)], QKN=64, VHD=32, seed=43)
    w = window_case(NH, 1, B, 700, 3, 500, QKN=64, VHD=32, seed=44)
    monkeypatch.setenv("MLAMOE_MLA_PART_MAX", "1")
    assert np.array_equal(a, prefix_case(NH, B, 1500, 40, [40 - b for b in range(B)], QKN=64, VHD=32, seed=43))
    assert np.array_equal(w, window_case(NH, 1, B, 700, 3, 500, QKN=64, VHD=32, seed=44))


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,QKN,VHD", [(5, 3, 96, 24), (20, 50, 96, 40), (9, 60, 160, 272), (16, 49, 32, 16), (3, 260, 224, 100)])
def test_prefix_query_layouts(NH, B, QKN, VHD):
    """Query dimensions that end inside a window of 64, few and many positions,
    heads that do not fill a block."""
    prefix_case(NH, B, 70, 9, [b % 10 for b in range(B)], QKN, VHD, seed=300 + NH)


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,rows,L,sinks,window,lens", [
    (16, 2, 20, 7, 2, 5, [7, 3]), (1, 1, 150, 200, 3, 40, None), (1, 3, 70, 65, 0, 1, [65, 64, 1]),
    (128, 1, 2, 33, 1, 16, None), (16, 1, 1, 1, 0, 1, None), (6, 2, 25, 90, 90, 3, [90, 31])])
def test_window_odd_shapes(NH, B, rows, L, sinks, window, lens):
    """More rows than keys, one head (64 positions a tile), many heads, a single key."""
    window_case(NH, B, rows, L, sinks, window, lens, 64, 48, seed=400 + NH + rows)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [0x7FC0, 0x7F80, 0xFF80])
def test_window_keys_that_are_not_finite(bad):
    """A drafted position whose cache row is not finite: the rows before it,
    which do not see it, are what they are without it; the rows that see it have
    no finite value.  So does a key that has left some rows' windows."""
    NH, B, rows, L, sinks, window = 16, 2, 9, 300, 2, 70
    rng = np.random.default_rng(45)
    q = synth.normal_f32(rng, (B, rows, NH, 192), 2.0)
    cache = synth.normal_bf16(rng, (B, L, KVL + QKR), 1.0)
    clean = cache.copy()
    new, old = L - rows + 5, L - rows + 3 - window + 1           # rows 5.. see `new`, rows ..3 `old`
    cache[0, new] = np.uint16(bad)
    cache[1, old] = np.uint16(bad)
    ctx, _ = loaded(NH)
    with ctx:
        got, want = ctx.mla_window_decode(0, q, cache, sinks, window), ctx.mla_window_decode(0, q, clean, sinks, window)
    for r in range(rows):
        for b, sees in ((0, r >= 5), (1, r <= 3)):
            if sees:
                assert not np.isfinite(got[b, r]).any(), (b, r)
            else:
                assert np.array_equal(got[b, r], want[b, r]), (b, r)


@pytest.mark.gpu
def test_far_caches():
    """Own rows past 2^32 bytes of the caches."""
    NH, B, stride, P = 16, 260, 16384, 100
    rng = np.random.default_rng(90)
    ctx, kv_b = loaded(NH)
    with ctx:
        cache = ctx.alloc(B * stride * 1152)
        ctx.fill(cache, B * stride * 576, mlamoe.MM_FILL_BF16_NORMAL, 3)
        q, prefix = synth.normal_f32(rng, (B, NH, 192)), synth.normal_bf16(rng, (P, 576), 1.0)
        lens = np.full(B, 9, np.int32)
        dq, dp, dl, out = ctx.to_device(q), ctx.to_device(prefix), ctx.to_device(lens), ctx.empty((B, NH * 128), np.float32)
        ctx.mla_prefix_decode_dev(0, B, dq, dp, P, cache, stride, 20, out, dl)
        got = out.download()
        dl.upload(np.full(B, stride, np.int32))
        ctx.mla_window_decode_dev(0, B, 1, dq, cache, stride, stride, 2, 5, out, dl)
        win, base = out.download(), cache.ptr
        for b in (0, 1, 227, 228, B - 1):
            cache.ptr = base + b * stride * 1152
            own = cache.download(np.uint16, (stride, 576))
            cache.ptr = base
            for got_b, keys in ((got, np.concatenate([prefix, own[:9]])), (win, np.concatenate([own[:2], own[-5:]]))):
                close(got_b[b].reshape(NH, 128), attend(q[b].astype(np.float64), kv_b, f64(keys), NH, 128, 128), b)


@pytest.mark.gpu
def test_captured():
    """A graph of both calls, with workspaces of their own, replayed between
    eager calls on new queries and cache rows: the eager result every time;
    without a workspace a captured call is refused."""
    NH, B, P, L, rows = 16, 6, 500, 64, 3
    rng = np.random.default_rng(91)
    ctx, _ = loaded(NH)
    with ctx:
        dq, dw = ctx.empty((B, NH, 192), np.float32), ctx.empty((B // rows, rows, NH, 192), np.float32)
        dp, dc = ctx.empty((P, 576), np.uint16), ctx.empty((B, L, 576), np.uint16)
        dl = ctx.to_device(np.array([64, 1, 0, 33, 16, 63], np.int32))
        out = [ctx.empty((B, NH * 128), np.float32) for _ in range(4)]
        w1 = ctx.alloc(ctx.mla_prefix_decode_workspace(B, P, L))
        w2 = ctx.alloc(ctx.mla_window_decode_workspace(B // rows, rows, L, 2, 20))

        def prefix(o, w):
            ctx.mla_prefix_decode_dev(0, B, dq, dp, P, dc, L, L, o, dl, w)

        def window(o, w):
            ctx.mla_window_decode_dev(0, B // rows, rows, dw, dc, L, L, 2, 20, o, dl, w)

        def record():
            for call, o, w in ((prefix, out[0], w1), (window, out[1], w2)):
                with pytest.raises(mlamoe.MMError) as e:
                    call(o, None)
                assert e.value.status == -5
                call(o, w)
        g = Graph(ctx, record)
        for rep in range(4):
            dq.upload(synth.normal_f32(rng, (B, NH, 192)))
            dw.upload(synth.normal_f32(rng, (B // rows, rows, NH, 192)))
            dp.upload(synth.normal_bf16(rng, (P, 576), 1.0))
            dc.upload(synth.normal_bf16(rng, (B, L, 576), 1.0))
            g.replay()
            prefix(out[2], None)
            window(out[3], None)
            for a, b in zip(out[:2], out[2:]):
                assert np.array_equal(a.download(), b.download()), rep
        g.close()


@pytest.mark.gpu
def test_callers_stream_and_rows_behind():
    """On a stream of the caller's: the same bits as on the context's, and
    nothing behind the last row or the workspace is written."""
    NH, B, P, L = 16, 5, 260, 33
    rng = np.random.default_rng(92)
    q, prefix = synth.normal_f32(rng, (B, NH, 192)), synth.normal_bf16(rng, (P, 576), 1.0)
    cache, lens = synth.normal_bf16(rng, (B, L, 576), 1.0), np.array([33, 0, 7, 32, 1], np.int32)
    ctx, _ = loaded(NH)
    hip = C.CDLL("libamdhip64.so")
    stream = C.c_void_p()
    hip.hipStreamCreateWithFlags.argtypes = [C.POINTER(C.c_void_p), C.c_uint]
    hip.hipStreamDestroy.argtypes = [C.c_void_p]
    with ctx:
        a, w = ctx.mla_prefix_decode(0, q, prefix, cache, lens), ctx.mla_window_decode(0, q[:, None], cache, 1, 9, lens)
        dq, dp, dc, dl = (ctx.to_device(v) for v in (q, prefix, cache, lens))
        need = max(ctx.mla_prefix_decode_workspace(B, P, L), ctx.mla_window_decode_workspace(B, 1, L, 1, 9))
        out, ws = ctx.to_device(np.full((B + 2, NH * 128), 7.0, np.float32)), ctx.to_device(np.full(need + 4096, 7, np.uint8))
        size = ws.nbytes
        ctx.sync()
        assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
        ctx.set_stream(stream)
        for want, call in ((a, lambda: ctx.mla_prefix_decode_dev(0, B, dq, dp, P, dc, L, L, out, dl, ws)),
                           (w[:, 0], lambda: ctx.mla_window_decode_dev(0, B, 1, dq, dc, L, L, 1, 9, out, dl, ws))):
            ws.nbytes = need
            call()
            ws.nbytes = size
            got = out.download()
            assert np.array_equal(got[:B], want) and np.all(got[B:] == 7.0)
            assert np.all(ws.download()[need:] == 7)
        ctx.set_stream(None)
        ctx.sync()
    assert hip.hipStreamDestroy(stream) == 0


@pytest.mark.gpu
def test_refusals():
    L = mlamoe.lib()
    with mlamoe.Context(0) as bare:
        assert L.mm_mla_prefix_decode_dev(bare.h, 0, 1, None, None, 0, None, 0, None, 0, None, None, 0) == -5
        assert L.mm_mla_window_decode_dev(bare.h, 0, 1, 1, None, None, 1, None, 1, 0, 1, None, None, 0) == -5
    ctx, _ = loaded(16)
    with ctx:
        q, p, c = ctx.empty((2, 16, 192), np.float32), ctx.empty((8, 576), np.uint16), ctx.empty((2, 8, 576), np.uint16)
        o = ctx.to_device(np.full((2, 16 * 128), 3.0, np.float32))

        def pre(layer=0, B=2, q=q.ptr, p=p.ptr, P=8, c=c.ptr, stride=8, n=8, o=o.ptr, ws=None, nb=0):
            return L.mm_mla_prefix_decode_dev(ctx.h, layer, B, q, p, P, c, stride, None, n, o, ws, nb)

        def win(layer=0, B=2, rows=1, q=q.ptr, c=c.ptr, stride=8, n=8, s=1, w=4, o=o.ptr, ws=None, nb=0):
            return L.mm_mla_window_decode_dev(ctx.h, layer, B, rows, q, c, stride, None, n, s, w, o, ws, nb)
        assert pre(layer=1) == -5 and pre(layer=-1) == -5 and win(layer=1) == -5
        assert pre(B=-1) == -1 and pre(P=-1) == -1 and pre(n=-1) == -1 and pre(stride=7) == -1
        assert pre(q=None) == -1 and pre(p=None) == -1 and pre(c=None) == -1 and pre(o=None) == -1
        assert pre(q=q.ptr + 4) == -1 and pre(p=p.ptr + 2) == -1 and pre(c=c.ptr + 8) == -1
        assert pre(B=(1 << 20) + 1) == -2 and pre(P=262145) == -2 and pre(n=262145, stride=262145) == -2
        assert pre(ws=o.ptr, nb=64) == -1 and pre(ws=o.ptr + 4, nb=1 << 30) == -1
        assert win(B=-1) == -1 and win(rows=0) == -1 and win(n=0) == -1 and win(stride=7) == -1 and win(s=-1) == -1 and win(w=0) == -1
        assert win(q=None) == -1 and win(c=None) == -1 and win(o=None) == -1 and win(q=q.ptr + 8) == -1 and win(c=c.ptr + 4) == -1
        assert win(B=1 << 19, rows=3) == -2 and win(n=262145, stride=262145) == -2 and win(ws=o.ptr, nb=64) == -1
        assert pre(B=0, q=None, o=None) == 0 and win(B=0, q=None, c=None, o=None) == 0
        assert np.all(o.download() == 3.0)


def test_refusals_without_a_gpu():
    L = mlamoe.lib()
    b = C.c_size_t(7)
    assert L.mm_mla_prefix_decode_dev(None, 0, 1, None, None, 0, None, 0, None, 0, None, None, 0) == -1
    assert L.mm_mla_window_decode_dev(None, 0, 1, 1, None, None, 1, None, 1, 0, 1, None, None, 0) == -1
    assert L.mm_mla_prefix_decode_workspace(None, 1, 1, 1, C.byref(b)) == -1 and b.value == 0
    assert L.mm_mla_window_decode_workspace(None, 1, 1, 1, 1, 1, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("NH,rows,head,row,what", [
    (16, 1, 5, 0, "nope"), (16, 9, 0, 4, "nope"), (16, 9, 15, 8, "rope"), (20, 7, 19, 0, "rope"), (3, 4, 1, 2, "nope"),
    (16, 9, 3, 5, "inf"), (16, 1, 15, 0, "large"), (20, 7, 2, 3, "large")])
def test_window_query_that_is_not_finite(NH, rows, head, row, what):
    """One head's query of one position is not finite, or so large that scores
    overflow: every other head and position has its own result."""
    B, L, sinks, window = 2, 300, 2, 70
    rng = np.random.default_rng(46)
    q = synth.normal_f32(rng, (B, rows, NH, 192), 2.0)
    cache = synth.normal_bf16(rng, (B, L, KVL + QKR), 1.0)
    if what == "nope":
        q[0, row, head, 7] = np.nan
    elif what == "rope":
        q[0, row, head, 150] = np.nan
    elif what == "inf":
        q[0, row, head, 128:130] = np.inf, -np.inf
    else:
        q[0, row, head, 128:] = 3e38
    ctx, kv_b = loaded(NH)
    with ctx:
        got = ctx.mla_window_decode(0, q, cache, sinks, window)
    got = got.reshape(B, rows, NH, 128)
    at = np.arange(L)
    for b in range(B):
        for r in range(rows):
            p = L - rows + r
            keys = f64(cache[b, at[(at <= p) & ((at < sinks) | (at > p - window))]])
            for h in range(NH):
                if (b, r, h) == (0, row, head):
                    assert what == "large" or not np.isfinite(got[b, r, h]).any()
                    continue
                w = kv_b.reshape(NH, 256, KVL)[h]
                close(got[b, r, h:h + 1], attend(q[b, r, h:h + 1].astype(np.float64), w, keys, 1, 128, 128), (b, r, h))


@pytest.mark.gpu
@pytest.mark.parametrize("NH,rows,bad", [(16, 9, 5), (20, 5, 4), (16, 2, 1), (3, 8, 3), (16, 40, 17)])
def test_window_position_that_is_not_finite(NH, rows, bad):
    """A drafted or prompt position whose hidden state was not finite: neither is
    its query nor its cache row.  The positions before it do not see it, and are
    what they are without it; those from it on have no finite value."""
    B, L, sinks, window = 2, 300, 2, 70
    rng = np.random.default_rng(47)
    q = synth.normal_f32(rng, (B, rows, NH, 192), 2.0)
    cache = synth.normal_bf16(rng, (B, L, KVL + QKR), 1.0)
    clean, at = cache.copy(), np.arange(L)
    q[1, bad], cache[1, L - rows + bad] = np.nan, NAN16
    ctx, kv_b = loaded(NH)
    with ctx:
        got = ctx.mla_window_decode(0, q, cache, sinks, window)
    for b in range(B):
        for r in range(rows):
            if b == 1 and r >= bad:
                assert not np.isfinite(got[b, r]).any(), (b, r)
                continue
            p = L - rows + r
            keys = f64(clean[b, at[(at <= p) & ((at < sinks) | (at > p - window))]])
            close(got[b, r].reshape(NH, 128), attend(q[b, r].astype(np.float64), kv_b, keys, NH, 128, 128), (b, r))


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,VHD", [(16, 3, 128), (3, 40, 24), (128, 1, 16)])
def test_no_keys_at_all(NH, B, VHD):
    """No prefix and no own row: zeros without a workspace, captured too, and
    nothing behind the last row."""
    ctx, _ = loaded(NH, 64, VHD)
    with ctx:
        assert ctx.mla_prefix_decode_workspace(B, 0, 0) == 0
        q = ctx.to_device(np.full((B, NH, 64 + QKR), np.nan, np.float32))
        outs = [ctx.to_device(np.full((B + 1, NH * VHD), 7.0, np.float32)) for _ in range(2)]
        ctx.mla_prefix_decode_dev(0, B, q, None, 0, None, 0, 0, outs[0])
        g = Graph(ctx, lambda: ctx.mla_prefix_decode_dev(0, B, q, None, 0, None, 0, 0, outs[1]))
        for _ in range(3):
            g.replay()
        for o in outs:
            got = o.download()
            assert np.all(got[:B] == 0.0) and np.all(got[B] == 7.0)
        g.close()


@pytest.mark.gpu
def test_workspace_stays_within_the_cap(monkeypatch):
    """Queries and partials of the rows in flight together, however many rows."""
    for cap in (None, 1 << 28):
        if cap:
            monkeypatch.setenv("MLAMOE_MLA_PART_MAX", str(cap))
        for NH in (16, 20, 3):
            with mlamoe.Context(0) as ctx:
                ctx.mla_init(NH, 128, QKR, KVL, 128)
                most = (cap or 512 << 20) + 2304 * 32 + 512      # a last tile of queries, alignment
                for rows in (1, 1000, 14600, 1 << 20):
                    for p, own in ((4096, 0), (33, 7), (0, 1), (100000, 300)):
                        assert 0 < ctx.mla_prefix_decode_workspace(rows, p, own) <= most, (cap, NH, rows, p, own)
                    for n, w in ((8192, 4096), (50, 7)):
                        assert 0 < ctx.mla_window_decode_workspace(1, rows, n, 4, w) <= most, (cap, NH, rows, n, w)
                        assert 0 < ctx.mla_window_decode_workspace(rows, 1, n, 4, w) <= most, (cap, NH, rows, n, w)


@pytest.mark.gpu
@pytest.mark.parametrize("NH,B,QKN,VHD", [(20, 130, 96, 40), (3, 300, 32, 16)])
def test_many_rows_in_groups(monkeypatch, NH, B, QKN, VHD):
    """As above with the query layout and merge of many rows, and lengths that
    differ from sequence to sequence."""
    lens = [(7 * b) % 51 for b in range(B)]
    a = prefix_case(NH, B, 210, 50, lens, QKN, VHD, seed=500 + NH)
    w = window_case(NH, 2, B // 2, 400, 5, 90, [400, 311], QKN, VHD, seed=501 + NH)
    monkeypatch.setenv("MLAMOE_MLA_PART_MAX", str(9 << 20))
    assert np.array_equal(a, prefix_case(NH, B, 210, 50, lens, QKN, VHD, seed=500 + NH))
    assert np.array_equal(w, window_case(NH, 2, B // 2, 400, 5, 90, [400, 311], QKN, VHD, seed=501 + NH))


@pytest.mark.gpu
def test_host_forms_refuse_arrays_too_short():
    """Lengths, rows and heads that the kernels would read past."""
    ctx, _ = loaded(16)
    q, pre, c = np.zeros((3, 16, 192), np.float32), np.zeros((5, 576), np.uint16), np.zeros((3, 8, 576), np.uint16)
    with ctx:
        for call in (lambda: ctx.mla_prefix_decode(0, q, pre, c, [1, 2]), lambda: ctx.mla_prefix_decode(0, q, pre, c[:2]),
                     lambda: ctx.mla_prefix_decode(0, q[:, :15], pre, c), lambda: ctx.mla_prefix_decode(0, q[..., :128], pre, c),
                     lambda: ctx.mla_prefix_decode(0, q, pre[:, :512], c), lambda: ctx.mla_prefix_decode(0, q, pre, c[..., :512]),
                     lambda: ctx.mla_window_decode(0, q[:, None], c[:2], 0, 4), lambda: ctx.mla_window_decode(0, q[:, None], c, 0, 4, [1]),
                     lambda: ctx.mla_window_decode(0, q, c, 0, 4), lambda: ctx.mla_window_decode(0, q[:, None, :8], c, 0, 4),
                     lambda: ctx.mla_window_decode(0, q[:, None], c[..., :512], 0, 4)):
            with pytest.raises(mlamoe.MMError) as e:
                call()
            assert e.value.status == -1
