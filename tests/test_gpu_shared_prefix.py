"""Decode steps of sequences behind a shared prefix, from the layer's front to the
tokens' log probabilities, as a serving loop makes them; and the prompt's last
rows through a window.  Each stage is compared on its own inputs: what the front
writes with mm_mla_front_dev on whole caches (the same operations: the same bits),
attention and log probabilities with their 64-bit formulas and tolerances
(test_gpu_mla_decode.py, test_gpu_logprobs.py)."""
import numpy as np
import pytest

import mlamoe
import test_gpu_logprobs as lp
import test_gpu_mla_decode as md
from hip_graph import Graph
from mlamoe import synth

H, NH, QKN, VHD, QKD, KVD, VOCAB, TOP = 512, 4, 64, 64, 128, 576, 5003, 5
P, OWN = 70, 6


class Model:
    def __init__(self, ctx, seed):
        self.ctx = ctx
        self.w = synth.attn_layer(seed, H, NH, QKN, 64, 512, VHD)
        rng = np.random.default_rng(seed + 1)
        self.embed, self.head = synth.normal_f32(rng, (VOCAB, H), 1.0), synth.normal_bf16(rng, (VOCAB, H), 0.1)
        ctx.mla_init(NH, QKN, 64, 512, VHD)
        ctx.mla_front_init(H, mlamoe.rope_inv_freq(64, 10000.0))
        ctx.mla_load_layer(0, self.w["kv_b"])
        self.kv_b = md.f64(self.w["kv_b"])
        self.front, self.keep = ctx.front_weights(self.w)
        self.o_proj, self.norm, self.lm = (ctx.to_device(v) for v in (self.w["o_proj"], self.w["in_norm"], self.head))

    def prompt(self, rng):
        """P tokens of one sequence: its cache and queries."""
        cache, q = self.ctx.empty((P, KVD), np.uint16), np.empty((P, NH, QKD), np.float32)
        pos, dq = self.ctx.empty((1,), np.int32), self.ctx.empty((1, NH * QKD), np.float32)
        x = self.ctx.empty((1, H), np.float32)
        for p in range(P):
            x.upload(self.embed[rng.integers(VOCAB)][None])
            pos.upload(np.array([p], np.int32))
            self.ctx.mla_front_dev(1, x, self.front, pos, dq, cache, P)
            q[p] = dq.download().reshape(NH, QKD)
        return cache, q


class Step:
    """A decode step of B sequences and its buffers."""

    def __init__(self, m, B, prefix):
        c = self.c = m.ctx
        self.m, self.B, self.prefix = m, B, prefix
        self.x, self.q, self.o = c.empty((B, H), np.float32), c.empty((B, NH * QKD), np.float32), c.empty((B, NH * VHD), np.float32)
        self.cache, self.pos, self.lens = c.empty((B, OWN, KVD), np.uint16), c.empty((B,), np.int32), c.empty((B,), np.int32)
        self.logits, self.tokens = c.empty((B, VOCAB), np.float32), c.empty((B,), np.int32)
        self.lp, self.ent = c.empty((B,), np.float32), c.empty((B,), np.float32)
        self.ti, self.tl = c.empty((B, TOP), np.int32), c.empty((B, TOP), np.float32)
        self.w1 = c.alloc(c.mla_prefix_decode_workspace(B, P, OWN))
        self.w2 = c.alloc(mlamoe.token_logprobs_workspace(B, VOCAB, TOP))

    def run(self):
        c, m = self.c, self.m
        c.mla_front_prefix_dev(self.B, self.x, m.front, self.pos, P, self.q, self.cache, OWN)
        c.mla_prefix_decode_dev(0, self.B, self.q, self.prefix, P, self.cache, OWN, OWN, self.o, self.lens, self.w1)
        c.matmul_dev(self.x, self.o, m.o_proj, H, NH * VHD, self.B, mlamoe.MM_MATMUL_ACCUMULATE)
        c.lm_head_dev(self.B, self.x, m.norm, 1e-6, m.lm, VOCAB, H, self.logits, self.tokens)
        c.token_logprobs_dev(self.B, self.logits, VOCAB, VOCAB, self.tokens, self.lp, self.ent, TOP, self.ti, self.tl, self.w2)

    def outputs(self):
        return [b.download() for b in (self.q, self.cache, self.o, self.logits, self.tokens, self.lp, self.ent, self.ti, self.tl)]


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 3, 9])
def test_decode_behind_a_prefix(B):
    print(f"shared prefix B={B}", flush=True)
    rng = np.random.default_rng(B)
    with mlamoe.Context(0) as ctx:
        m = Model(ctx, 5)
        prefix, _ = m.prompt(rng)
        s = Step(m, B, prefix)
        s.cache.upload(np.full((B, OWN, KVD), md.NAN16))
        whole = ctx.to_device(np.concatenate([np.broadcast_to(prefix.download(), (B, P, KVD)), np.zeros((B, OWN, KVD), np.uint16)], 1))
        q2 = ctx.empty((B, NH * QKD), np.float32)
        start = np.arange(B) % 2                                  # every other sequence a step behind
        token = rng.integers(VOCAB, size=B)
        for step in range(4):
            own = np.maximum(step + 1 - start, 0)                 # rows after this step; 0: pos is in the prefix, none written
            s.x.upload(m.embed[token])
            s.pos.upload((P + own - 1).astype(np.int32))
            s.lens.upload(own.astype(np.int32))
            ctx.mla_front_dev(B, s.x, m.front, s.pos, q2, whole, P + OWN)
            s.run()
            q, cache, o, logits, tokens, lps, ent, ti, tl = s.outputs()
            assert np.array_equal(q, q2.download())
            rows = whole.download()[:, P:]
            for b in range(B):
                assert np.array_equal(cache[b, :own[b]], rows[b, :own[b]])
                assert np.all(cache[b, own[b]:] == md.NAN16)
                keys = np.concatenate([md.f64(prefix.download()), md.f64(cache[b, :own[b]])])
                md.close(o[b].reshape(NH, VHD), md.attend(q[b].reshape(NH, QKD).astype(np.float64), m.kv_b, keys, NH, QKN, VHD), (step, b))
                want = lp.ref(logits[b], tokens[b], TOP)
                lp.same(lps[b], want[0], want[1], "logprob")
                lp.same(ent[b], want[2], want[3], "entropy")
                assert list(ti[b]) == want[4] and ti[b, 0] == tokens[b] and tl[b, 0] == lps[b]
            token = tokens


@pytest.mark.gpu
def test_step_captured():
    """The step in a graph, replayed between eager steps on other tokens."""
    rng = np.random.default_rng(77)
    with mlamoe.Context(0) as ctx:
        m = Model(ctx, 6)
        prefix, _ = m.prompt(rng)
        a, b = Step(m, 7, prefix), Step(m, 7, prefix)
        for s in (a, b):                                          # the context's workspace at its size
            s.cache.upload(np.zeros((7, OWN, KVD), np.uint16))
            s.x.upload(m.embed[:7])
            s.pos.upload(np.full(7, P, np.int32))
            s.lens.upload(np.ones(7, np.int32))
            s.run()
        g = Graph(ctx, a.run)
        for rep in range(1, 5):
            x = m.embed[rng.integers(VOCAB, size=7)]
            for s, run in ((a, g.replay), (b, b.run)):
                s.x.upload(x)
                s.pos.upload(np.full(7, P + rep, np.int32))
                s.lens.upload(np.full(7, rep + 1, np.int32))
                run()
            for u, v in zip(a.outputs(), b.outputs()):
                assert np.array_equal(u, v), rep
        g.close()


@pytest.mark.gpu
def test_prompt_rows_through_a_window():
    rng = np.random.default_rng(78)
    rows, sinks, window = 11, 3, 20
    with mlamoe.Context(0) as ctx:
        m = Model(ctx, 7)
        prefix, q = m.prompt(rng)
        dq, out = ctx.to_device(q[P - rows:]), ctx.empty((rows, NH * VHD), np.float32)
        ctx.mla_window_decode_dev(0, 1, rows, dq, prefix, P, P, sinks, window, out)
        got, keys = out.download(), md.f64(prefix.download())
        for r in range(rows):
            p, at = P - rows + r, np.arange(P)
            see = (at <= p) & ((at < sinks) | (at > p - window))
            md.close(got[r].reshape(NH, VHD), md.attend(q[p].astype(np.float64), m.kv_b, keys[see], NH, QKN, VHD), r)


@pytest.mark.gpu
def test_front_refusals():
    L = mlamoe.lib()
    with mlamoe.Context(0) as ctx:
        m = Model(ctx, 8)
        b = ctx.empty((4, H), np.float32)
        assert L.mm_mla_front_prefix_dev(ctx.h, 1, b.ptr, m.front, b.ptr, -1, b.ptr, b.ptr, 1, None) == -1
        assert L.mm_mla_front_prefix_dev(ctx.h, 1, None, m.front, b.ptr, 1, b.ptr, b.ptr, 1, None) == -1
        assert L.mm_mla_front_prefix_dev(ctx.h, 1, b.ptr, m.front, b.ptr, 1, b.ptr, b.ptr, 0, None) == -1
        assert L.mm_mla_front_prefix_dev(ctx.h, 0, None, None, None, 1, None, None, 0, None) == 0


def test_front_refusals_without_a_gpu():
    assert mlamoe.lib().mm_mla_front_prefix_dev(None, 1, None, None, None, 0, None, None, 1, None) == -1
