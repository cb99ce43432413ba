"""The token-generation operators together, as they are used: cache.PagedKV and vlm.CachedLM on the GPU.

A prompt, single-token steps, a fork, drafted tokens taken back, a freed sequence and a compaction, against a float64
model of the same layers (oracle/cache_oracle.py for the cache's rounding, the weights in the form that each step uses).
Layer outputs pass through bf16 at every step, so they are compared by cosine, >= 0.999 as the decoder layer's test."""

import numpy as np
import pytest

from oracle import bfp16_oracle as O
from oracle import cache_oracle as C
from oracle import vlm_oracle as VO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from redline_tiny_b200 import cache, ops, vlm
    assert torch.cuda.is_available()
    return torch, ops, vlm, cache, torch.device("cuda:0")


class Model:
    """float64 decoder layers with a cache per sequence that rounds as the 8-bit blocks do."""

    def __init__(self, weights, cfg, few, group):
        self.cfg, self.few = cfg, few
        self.w4, self.bfp, self.norm = [], [], []
        for lw in weights["layers"]:
            lw = {k: v.cpu().numpy() for k, v in lw.items()}
            mats = {"qkv": lw["qkv"], "o": lw["o"], "gate": lw["gate"].T, "up": lw["up"].T, "down": lw["down"]}
            self.bfp.append({n: VO.decode_b(m) for n, m in mats.items()})
            q = {n: C.quantize_w4(np.ascontiguousarray(m), group) for n, m in mats.items()}
            self.w4.append({n: (c.astype(np.float64) - 8) * np.repeat(s.astype(np.float64), group, 0) for n, (c, s) in q.items()})
            self.norm.append(lw)

    def new(self):
        blocks = 40
        def one():
            return C.Cache(np.full((blocks, self.cfg.kv_heads, 16, 128), 128, np.uint8),
                           np.zeros((blocks, self.cfg.kv_heads, 1), np.uint8))
        return {"len": 0, "kv": [(one(), one()) for _ in self.norm]}

    def copy(self, seq):
        def dup(c):
            return C.Cache(c.codes.copy(), c.exps.copy())
        return {"len": seq["len"], "kv": [(dup(k), dup(v)) for k, v in seq["kv"]]}

    def step(self, seqs, xs, cos, sin):
        """xs: rows per sequence (the form of the weights goes by all rows of the step)."""
        cfg, mats = self.cfg, self.w4 if sum(len(x) for x in xs) <= self.few else self.bfp
        table = np.arange(40)
        outs = []
        for seq, x in zip(seqs, xs):
            n = len(x)
            if n == 0:
                outs.append(np.zeros((0, cfg.hidden)))
                continue
            pos = seq["len"] + np.arange(n)
            seq["len"] += n
            x = x.astype(np.float64)
            for lw, m, (kc, vc) in zip(self.norm, mats, seq["kv"]):
                qkv = VO.rms(x, lw["w_in"]) @ m["qkv"]
                H, Hk = cfg.heads, cfg.kv_heads
                q, k, v = (t.reshape(n, -1, 128) for t in np.split(qkv, [H * 128, (H + Hk) * 128], 1))
                q = VO.rope_pairs(VO.rms(q, lw["q_norm"]).transpose(1, 0, 2), cos[pos], sin[pos]).transpose(1, 0, 2)
                k = VO.rope_pairs(VO.rms(k, lw["k_norm"]).transpose(1, 0, 2), cos[pos], sin[pos]).transpose(1, 0, 2)
                kc.append(table, seq["len"], k.astype(np.float32))
                vc.append(table, seq["len"], v.astype(np.float32))
                o, _ = C.attention(q, kc.read(table, seq["len"]), vc.read(table, seq["len"]), pos)
                x = x + o.reshape(n, -1) @ m["o"]
                h = VO.rms(x, lw["w_post"])
                g = h @ m["gate"]
                x = x + (g / (1 + np.exp(-g)) * (h @ m["up"])) @ m["down"]
            outs.append(x)
        return np.concatenate(outs)


@pytest.mark.parametrize("dims,few,page", [(dict(hidden=512, heads=4, kv_heads=2, ffn=1024, layers=2), 64, 16),
                                           (dict(hidden=1024, heads=8, kv_heads=2, ffn=2048, layers=1), 16, 64),
                                           (dict(hidden=512, heads=4, kv_heads=2, ffn=1024, layers=1), 0, 32)])
def test_generation(env, dims, few, page):
    torch, ops, vlm, cache, dev = env
    cfg = vlm.LMConfig(**dims)
    w = vlm.random_lm_weights(cfg, seed=3)
    kv = cache.PagedKV(cfg.layers, 80, cfg.kv_heads, page)
    lm = vlm.CachedLM(cfg, w, kv, few=few, group=64)
    ref = Model(w, cfg, few, 64)
    ang = np.arange(640)[:, None] * (1e6 ** (-np.arange(64) / 64.0))[None]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    d_cos, d_sin = torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev)
    rng = np.random.default_rng(4)
    state = {}

    def step(seqs, counts):
        batch = kv.batch(seqs)
        batch.extend(counts)
        xs = [O.bf16_round(rng.standard_normal((n, cfg.hidden)).astype(np.float32)) for n in counts]
        pos = np.concatenate([np.arange(kv.length(s) - n, kv.length(s)) for s, n in zip(seqs, counts)]).astype(np.int64)
        x = torch.from_numpy(np.concatenate(xs)).to(dev).to(torch.bfloat16)
        got = lm.forward(x, batch, d_cos[pos], d_sin[pos]).float().cpu().numpy()
        ops.device_status()
        want = ref.step([state[s] for s in seqs], xs, cos, sin)
        for r in range(len(want)):
            c = float(got[r] @ want[r] / np.linalg.norm(got[r]) / np.linalg.norm(want[r]))
            assert c >= 0.999, f"row {r}: cosine {c:.6f}"

    a, b = kv.new(), kv.new()
    state[a], state[b] = ref.new(), ref.new()
    step([a, b], [70, 33])                       # prompts
    for _ in range(3):
        step([a, b], [1, 1])
    c = kv.fork(a)
    state[c] = ref.copy(state[a])
    step([a, b, c], [1, 1, 1])                   # the fork's page is copied here
    step([c, a], [5, 2])                         # drafted tokens
    kv.truncate(c, kv.length(c) - 3)             # and three taken back
    state[c]["len"] -= 3
    step([a, c], [1, 1])
    kv.free(a)
    del state[a]
    assert kv.compact() > 0 or kv.free_pages > 0
    step([b, c], [1, 20])
    kv.resize(kv.pool.pages - kv.free_pages)
    with pytest.raises(cache.OutOfPages):
        kv.batch([b]).extend([500])
    assert kv.free_pages == 0


def test_two_streams_and_two_graphs(env):
    """Steps of two batches captured into graphs and replayed on two streams at once give what they give alone."""
    torch, ops, vlm, cache, dev = env
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    kv = cache.PagedKV(1, 64, 2, 16)
    q, k, batches, alone, graphs, outs = [], [], [], [], [], []
    for i in range(2):
        seqs = [kv.new() for _ in range(3)]
        batches.append(kv.batch(seqs))
        batches[i].extend([100 + 30 * i, 5, 60])
        T = 165 + 30 * i
        k.append(torch.randn(T, 2, 128, generator=g, device=dev).to(torch.bfloat16))
        q.append(torch.randn(T, 8, 128, generator=g, device=dev).to(torch.bfloat16))
        ops.kv_append(kv.pool, 0, k[i], k[i], *batches[i].args)
        alone.append(ops.kv_attention(q[i], kv.pool, 0, *batches[i].args))
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.kv_attention(q[i], kv.pool, 0, *batches[i].args))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    ops.device_status()
    for i in range(2):
        assert torch.equal(outs[i], alone[i])


def test_refusals(env):
    torch, ops, vlm, cache, dev = env
    cfg = vlm.LMConfig(hidden=256, heads=2, kv_heads=1, ffn=256, layers=1)
    kv = cache.PagedKV(1, 8, 1, 16)
    lm = vlm.CachedLM(cfg, vlm.random_lm_weights(cfg), kv, few=8)
    batch = kv.batch([kv.new()])
    batch.extend([3])
    x, rope = torch.zeros((2, 256), dtype=torch.bfloat16, device=dev), torch.zeros((2, 64), device=dev)
    with pytest.raises(ValueError, match="2 rows"):
        lm.forward(x, batch, rope, rope)
    other = cache.PagedKV(1, 8, 1, 16)
    step = other.batch([other.new()])
    step.extend([2])
    with pytest.raises(ValueError, match="another cache"):
        lm.forward(x, step, rope, rope)
    with pytest.raises(ValueError, match="layers"):
        vlm.CachedLM(vlm.LMConfig(hidden=256, heads=2, kv_heads=2, ffn=256), {"layers": []}, kv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=dev)
        for call in (lambda: batch.extend([1]), kv.compact, lambda: kv.resize(4)):
            with pytest.raises(RuntimeError, match="captured"):
                call()


def test_one_row_views_with_odd_strides(env):
    """A single row or head, whose stride says nothing, is taken with any stride."""
    torch, ops, vlm, cache, dev = env
    kv = cache.PagedKV(1, 8, 1, 16)
    batch = kv.batch([kv.new()])
    batch.extend([1])
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    x = torch.randn((1, 1, 128), generator=g, device=dev).to(torch.bfloat16)
    ops.kv_append(kv.pool, 0, x, x, *batch.args)
    want = ops.kv_attention(x, kv.pool, 0, *batch.args)
    odd = torch.as_strided(x, (1, 1, 128), (3, 5, 1))
    out = torch.as_strided(torch.zeros(256, dtype=torch.bfloat16, device=dev), (1, 128), (7, 1))
    assert torch.equal(ops.kv_attention(odd, kv.pool, 0, *batch.args, out=out), want)
    ops.device_status()
