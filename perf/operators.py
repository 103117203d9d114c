"""Decoding many continuations of one prompt, as cases that can be timed and
whose results can be compared: absorbed attention over a prefix that the whole
batch shares, absorbed attention of long sessions through a sliding window with
a few first tokens kept, and the log probabilities, entropies and top
alternatives that rank the continuations.

Head dimensions and the vocabulary are DeepSeek-V2-Lite's and GLM-4.7-Flash's.
listed() names the fixed cases, draw() gives more of the same ranges; prepare()
makes a case's inputs from a seed, run() is one pass -- through the library's
entry points where `own` is true, else in elementary fp32 torch operations --,
exact() the same results in 64 bits.
"""
import math
import os
import random
import sys
import weakref

import torch

own = False

KVL, QKR = 512, 64                # latent and rope parts of a cache row
KVD = KVL + QKR
# heads: (nope, value) dimensions per head
DIMS = {16: (128, 128), 20: (192, 256)}
VOCAB = 102400


def listed():
    return [
        # four samples of one short question, a few tokens in: latency
        {"name": "prefix_b4_p512", "kind": "prefix", "heads": 16, "batch": 4, "prefix": 512, "own": 40, "ragged": False},
        # a batch answering questions about one document, replies of different lengths
        {"name": "prefix_b64_p4096", "kind": "prefix", "heads": 16, "batch": 64, "prefix": 4096, "own": 256, "ragged": True},
        # the other head geometry, nothing a multiple of a tile
        {"name": "prefix_b23_p7777_h20", "kind": "prefix", "heads": 20, "batch": 23, "prefix": 7777, "own": 301, "ragged": True},
        # many samples (a reward model's group) of one long context
        {"name": "prefix_b64_p32768", "kind": "prefix", "heads": 16, "batch": 64, "prefix": 32768, "own": 128, "ragged": False},
        # one long interactive session: latency
        {"name": "window_b1_l4096_w1024", "kind": "window", "heads": 16, "batch": 1, "rows": 1, "length": 4096, "sinks": 4, "window": 1024, "ragged": False},
        # a decode batch of long sessions, some still shorter than their window
        {"name": "window_b64_l16384_w4096", "kind": "window", "heads": 16, "batch": 64, "rows": 1, "length": 16384, "sinks": 4, "window": 4096, "ragged": True},
        # odd sizes, three drafted tokens verified at once
        {"name": "window_b13_r3_l5001_w611_h20", "kind": "window", "heads": 20, "batch": 13, "rows": 3, "length": 5001, "sinks": 7, "window": 611, "ragged": True},
        # a prompt's chunk through the window
        {"name": "window_b1_r512_l6000_w1024", "kind": "window", "heads": 16, "batch": 1, "rows": 512, "length": 6000, "sinks": 4, "window": 1024, "ragged": False},
        # the token just sampled, with the alternatives a client asked for: latency
        {"name": "logprobs_t1_top20", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "pad": 0, "top": 20},
        # a decode batch
        {"name": "logprobs_t64_top5", "kind": "logprobs", "rows": 64, "vocab": VOCAB, "pad": 0, "top": 5},
        # another vocabulary, of odd size, in rows padded to whole cache lines
        {"name": "logprobs_t257_v32003", "kind": "logprobs", "rows": 257, "vocab": 32003, "pad": 29, "top": 1},
        # a prompt scored whole
        {"name": "logprobs_t2048_top8", "kind": "logprobs", "rows": 2048, "vocab": VOCAB, "pad": 0, "top": 8},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "window", "logprobs"])
    if kind == "logprobs":
        v = rng.choice([VOCAB, _between(rng, 1000, VOCAB)])
        return {"kind": kind, "rows": _between(rng, 1, 2048), "vocab": v, "pad": rng.choice([0, rng.randint(1, 127)]), "top": rng.choice([0, 1, rng.randint(2, 32)])}
    heads = rng.choice([16, 16, 20])
    c = {"kind": kind, "heads": heads, "batch": _between(rng, 1, 64 if heads == 16 else 48)}
    if kind == "prefix":
        return {**c, "prefix": _between(rng, 32, 32768), "own": _between(rng, 1, 512), "ragged": rng.random() < 0.6}
    rows = rng.choice([1, 1, rng.randint(2, 8), _between(rng, 9, 512)])
    c["batch"] = min(c["batch"], max(1, 512 // rows))
    return {**c, "rows": rows, "length": _between(rng, rows, 16384), "sinks": rng.choice([0, 4, rng.randint(1, 64)]),
            "window": _between(rng, 16, 4096 if rows <= 8 else 1024), "ragged": rng.random() < 0.6}


# ---- inputs ----------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _lengths(c):
    """Cache rows of each sequence: all of the longest, or spread evenly from
    it down to a twentieth."""
    n, b = c["own"] if c["kind"] == "prefix" else c["length"], c["batch"]
    lens = [n - (n - n // 20) * j // b for j in range(b)] if c["ragged"] else [n] * b
    return [max(x, c.get("rows", 1)) for x in lens]


def _cache(g, shape):
    """Latent cache rows (normalised c_kv, rotated k_pe), bf16."""
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)


def _inputs(c, seed):
    g = _gen(seed)
    if c["kind"] == "logprobs":
        t, n = c["rows"], c["vocab"]
        logits = _normal(g, (t, n + c["pad"]), 2.5)
        # the target is among the likelier tokens, and a few tokens stand out
        targets = torch.randint(0, n, (t,), generator=g, device="cuda", dtype=torch.int32)
        peaks = torch.randint(0, n, (t, 4), generator=g, device="cuda")
        logits.scatter_add_(1, peaks, _normal(g, (t, 4), 4.0).abs() + 8.0)
        picked = torch.rand((t,), generator=g, device="cuda") < 0.7
        targets = torch.where(picked, peaks[:, 0].to(torch.int32), targets)
        return {"logits": logits, "targets": targets}
    nh, b = c["heads"], c["batch"]
    nope, vdim = DIMS[nh]
    lens = _lengths(c)
    random.Random(seed).shuffle(lens)
    d = {"kv_b": _normal(g, (nh * (nope + vdim), KVL), 0.02).to(torch.bfloat16),
         "q": _normal(g, (b, c.get("rows", 1), nh, nope + QKR), 2.0),
         "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    d["cache"] = _cache(g, (b, max(lens), KVD))
    if c["kind"] == "prefix":
        d["prefix"] = _cache(g, (c["prefix"], KVD))
    return d


# ---- the handles a program keeps ----------------------------------------------------


class _Dev:
    """A tensor as the binding's device buffer."""

    def __init__(self, t):
        self.t, self.ptr, self.shape = t, t.data_ptr(), tuple(t.shape)


_programs = {}
_LAYERS = 256                     # a state's attention weights are a layer of its program


class _Program:
    """A context for one head geometry, its work on one stream.  Its layers are
    given back with it, when it has handed out all and no state of it is left."""

    def __init__(self, heads):
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mla-moe_amd"))
        import mlamoe
        self.ctx, self.layers, self.stream = mlamoe.Context(0), 0, torch.cuda.Stream()
        self.ctx.set_stream(self.stream.cuda_stream)
        self.ctx.mla_init(heads, DIMS[heads][0], QKR, KVL, DIMS[heads][1], n_layers=_LAYERS)
        weakref.finalize(self, _Program._close, self.ctx, self.stream).atexit = False

    @staticmethod
    def _close(ctx, stream):
        stream.synchronize()
        ctx.close()


def _program(heads):
    if heads not in _programs or _programs[heads].layers == _LAYERS:
        _programs[heads] = _Program(heads)
    return _programs[heads]


def prepare(case, seed):
    c = dict(case)
    st = {"case": c, **_inputs(c, seed)}
    if own:
        torch.cuda.synchronize()
        program = st["program"] = _program(c.get("heads", 16))
        ctx = st["ctx"] = program.ctx
        f32 = dict(dtype=torch.float32, device="cuda")
        if c["kind"] == "logprobs":
            t, k = c["rows"], c["top"]
            st["out"] = {"logprob": torch.zeros(t, **f32), "entropy": torch.zeros(t, **f32),
                         "top": torch.zeros((t, k), dtype=torch.int32, device="cuda"), "top_logprob": torch.zeros((t, k), **f32)}
        else:
            st["layer"] = program.layers
            program.layers += 1
            ctx.mla_load_layer(st["layer"], _Dev(st["kv_b"]), 4)          # 4: device pointers
            b, r, nh, _ = st["q"].shape
            st["out"] = torch.zeros((b, r, nh, DIMS[nh][1]), **f32)
        st["dev"] = {k: _Dev(v) for k, v in {**st, **(st["out"] if c["kind"] == "logprobs" else {})}.items() if isinstance(v, torch.Tensor)}
    torch.cuda.synchronize()
    return st


def run(st):
    c = st["case"]
    if own:
        ctx, d = st["ctx"], st["dev"]
        if c["kind"] == "prefix":
            ctx.mla_prefix_decode_dev(st["layer"], c["batch"], d["q"], d["prefix"], c["prefix"], d["cache"], d["cache"].shape[1],
                                      d["cache"].shape[1], d["out"], kv_lens=d["lens"])
        elif c["kind"] == "window":
            ctx.mla_window_decode_dev(st["layer"], c["batch"], c["rows"], d["q"], d["cache"], d["cache"].shape[1], d["cache"].shape[1],
                                      c["sinks"], c["window"], d["out"], kv_lens=d["lens"])
        else:
            ctx.token_logprobs_dev(c["rows"], d["logits"], c["vocab"] + c["pad"], c["vocab"], d["targets"], d["logprob"], d["entropy"],
                                   c["top"], d["top"], d["top_logprob"])
        return st["out"]
    return {"prefix": _plain_prefix, "window": _plain_window, "logprobs": _plain_logprobs}[c["kind"]](st)


# ---- the plain forms -----------------------------------------------------------------


def _absorbed(q, kv_b):
    """q [.., NH, nope + rope] -> [.., NH, KVD]: the query against cache rows."""
    nh = q.shape[-2]
    nope, vdim = DIMS[nh]
    w = kv_b.float().view(nh, nope + vdim, KVL)[:, :nope]
    qn = q[..., :nope].reshape(-1, nh, nope).transpose(0, 1)
    qa = torch.matmul(qn, w).transpose(0, 1).reshape(*q.shape[:-1], KVL)
    return torch.cat([qa, q[..., nope:]], -1) * (nope + QKR) ** -0.5


def _values(clat, kv_b):
    """clat [.., NH, KVL] -> [.., NH, vdim]."""
    nh = clat.shape[-2]
    nope, vdim = DIMS[nh]
    w = kv_b.float().view(nh, nope + vdim, KVL)[:, nope:].transpose(1, 2).contiguous()
    c = clat.reshape(-1, nh, KVL).transpose(0, 1)
    return torch.matmul(c, w).transpose(0, 1).reshape(*clat.shape[:-1], vdim)


def _plain_prefix(st):
    q, lens = _absorbed(st["q"], st["kv_b"]), st["lens"]
    b, _, nh, _ = q.shape
    shared, cache = st["prefix"].float(), st["cache"].float()
    s0 = torch.matmul(q.reshape(b * nh, KVD), shared.t()).view(b, nh, -1)
    s1 = torch.matmul(q.view(b, nh, KVD), cache.transpose(1, 2))
    at = torch.arange(cache.shape[1], device="cuda")
    s1 = torch.where(at[None, None, :] < lens[:, None, None], s1, -torch.inf)
    m = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    p0, p1 = torch.exp(s0 - m), torch.exp(s1 - m)
    o = torch.matmul(p0.view(b * nh, -1), shared[:, :KVL]).view(b, nh, KVL) + torch.matmul(p1, cache[..., :KVL])
    o = o / (p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True))
    return _values(o.view(b, 1, nh, KVL), st["kv_b"])


def _plain_window(st):
    c, lens = st["case"], st["lens"]
    q = _absorbed(st["q"], st["kv_b"])
    b, r, nh, _ = q.shape
    cache, sinks, w = st["cache"], c["sinks"], c["window"]
    u = min(w + r - 1, cache.shape[1])
    # the first keys, then the keys of the rows' windows
    start = (lens.long() - u).clamp(min=0)
    sink_at = torch.arange(min(sinks, cache.shape[1]), device="cuda")[None, :].expand(b, -1)
    at = torch.cat([sink_at, start[:, None] + torch.arange(u, device="cuda")], 1)
    first = torch.arange(at.shape[1], device="cuda")[None, :] < sink_at.shape[1]
    keys = cache[torch.arange(b, device="cuda")[:, None], at].float()
    pos = lens.long()[:, None] - r + torch.arange(r, device="cuda")        # [b, r]
    near = (at[:, None, :] <= pos[:, :, None]) & (at[:, None, :] > pos[:, :, None] - w)
    seen = torch.where(first[:, None, :], (at[:, None, :] <= pos[:, :, None]), near & (at[:, None, :] >= sinks))
    s = torch.matmul(q.reshape(b, r * nh, KVD), keys.transpose(1, 2)).view(b, r, nh, -1)
    s = torch.where(seen[:, :, None, :], s, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p.view(b, r * nh, -1), keys[..., :KVL]).view(b, r, nh, KVL) / p.sum(-1, keepdim=True)
    return _values(o, st["kv_b"])


def _plain_logprobs(st):
    c = st["case"]
    n, k = c["vocab"], c["top"]
    x = st["logits"][:, :n]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    lz = torch.log(z)
    logprob = torch.gather(d, 1, st["targets"].long()[:, None]) - lz
    entropy = lz - (e * d).sum(-1, keepdim=True) / z
    # whole numbers in the order of the logits, of equal ones the lowest index first
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = bits.long() * (1 << 32) + (n - 1 - torch.arange(n, device="cuda"))
    top = n - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
    return {"logprob": logprob[:, 0], "entropy": entropy[:, 0], "top": top.to(torch.int32), "top_logprob": torch.gather(d, 1, top) - lz}


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    c = dict(case)
    if c["kind"] == "logprobs":
        t, n, k = c["rows"], c["vocab"], c["top"]
        # the logits once; an exponential, two products and three sums for each
        return {"bytes": float(4 * t * n + t * (12 + 8 * k)), "flops": 6.0 * t * n}
    nh, b, r = c["heads"], c["batch"], c.get("rows", 1)
    nope, vdim = DIMS[nh]
    lens = _lengths(c)
    if c["kind"] == "prefix":
        keys, pairs = c["prefix"] + sum(lens), b * c["prefix"] + sum(lens)
    else:
        s, w = c["sinks"], c["window"]
        keys = sum(n if n <= s + w + r - 1 else s + w + r - 1 for n in lens)
        pairs = sum(min(p + 1, s + w) for n in lens for p in range(n - r, n))
    nbytes = 2 * KVD * keys + 2 * nh * (nope + vdim) * KVL + 4 * b * r * nh * (nope + QKR + vdim)
    return {"bytes": float(nbytes), "flops": 2.0 * nh * (pairs * (KVD + KVL) + b * r * KVL * (nope + vdim))}


# ---- the same results in 64 bits -----------------------------------------------------------


def exact(case, seed):
    c = dict(case)
    st = _inputs(c, seed)
    if c["kind"] == "logprobs":
        n, k = c["vocab"], c["top"]
        found = {"logprob": [], "entropy": [], "top": [], "top_logprob": []}
        for x in torch.split(st["logits"][:, :n], 256):
            at = sum(len(v) for v in found["logprob"])
            p = torch.log_softmax(x.double(), -1)
            tp = p.gather(1, st["targets"][at:at + len(x)].long()[:, None])
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
            found["logprob"].append(tp[:, 0])
            found["entropy"].append(torch.special.entr(p.exp()).sum(-1))
            found["top"].append(order.to(torch.int32))
            found["top_logprob"].append(p.gather(1, order))
        return {name: torch.cat(v) for name, v in found.items()}
    q, kv_b, cache = st["q"].double(), st["kv_b"].double(), st["cache"]
    lens, out = st["lens"].tolist(), []
    if c["kind"] == "prefix":
        # every head's keys and values of the prefix once, for all sequences
        nh, b = c["heads"], c["batch"]
        nope, vdim = DIMS[nh]
        w, shared = kv_b.view(nh, nope + vdim, KVL), st["prefix"].double()
        longest = max(lens)
        mine = cache[:, :longest].double()
        ok = torch.arange(longest, device="cuda")[None, :] < st["lens"][:, None]
        res = torch.empty((b, 1, nh, vdim), dtype=torch.float64, device="cuda")
        for h in range(nh):
            kv0, kv1 = shared[:, :KVL] @ w[h].t(), mine[..., :KVL] @ w[h].t()
            qh = q[:, 0, h]
            s0 = qh[:, :nope] @ kv0[:, :nope].t() + qh[:, nope:] @ shared[:, KVL:].t()
            s1 = (qh[:, None, :nope] * kv1[..., :nope]).sum(-1) + (qh[:, None, nope:] * mine[..., KVL:]).sum(-1)
            a = torch.softmax(torch.cat([s0, s1.masked_fill(~ok, float("-inf"))], 1) / math.sqrt(nope + QKR), -1)
            res[:, 0, h] = a[:, :len(shared)] @ kv0[:, nope:] + (a[:, len(shared):, None] * kv1[..., nope:]).sum(1)
        return res
    r, nh = c["rows"], c["heads"]
    nope, vdim = DIMS[nh]
    w = kv_b.view(nh, nope + vdim, KVL)
    for b, n in enumerate(lens):
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        at = torch.arange(n, device="cuda")[None, :]
        seen = (at <= pos) & ((at < c["sinks"]) | (at > pos - c["window"]))
        some = seen.any(0)
        keys, seen = cache[b, :n][some].double(), seen[:, some]
        res = torch.empty((r, nh, vdim), dtype=torch.float64, device="cuda")
        for h in range(nh):
            kv = keys[:, :KVL] @ w[h].t()                                  # [keys, nope + vdim]
            s = (q[b, :, h, :nope] @ kv[:, :nope].t() + q[b, :, h, nope:] @ keys[:, KVL:].t()) / math.sqrt(nope + QKR)
            res[:, h] = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ kv[:, nope:]
        out.append(res)
    return torch.stack(out)
