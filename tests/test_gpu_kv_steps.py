"""Runs of the paged cache and of the cached decoder layers on the GPU that are held bit for bit: sequences that fork, draft,
take back, move and shrink against a model of each sequence alone, and captured decode steps against eager ones."""

import copy

import numpy as np
import pytest

from oracle import bfp16_oracle as O
from oracle import cache_oracle as C
from test_gpu_kv_cache import bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from redline_tiny_b200 import _lib, cache, ops, vlm
    assert torch.cuda.is_available()
    return torch, ops, _lib, cache, vlm, torch.device("cuda:0")


class Sequence:
    """The blocks of one sequence, to itself."""

    def __init__(self, layers, hkv):
        self.length = 0
        self.kv = [[C.Cache(np.full((12, hkv, 16, 128), 128, np.uint8), np.zeros((12, hkv, 1), np.uint8)) for _ in range(2)]
                   for _ in range(layers)]

    def append(self, layer, k, v):
        for cache, x in zip(self.kv[layer], (k, v)):
            cache.append(range(12), self.length, x)


@pytest.mark.parametrize("page,layers,hkv", [(16, 2, 2), (64, 3, 1)])
def test_sequences_hold_what_they_were_given(env, page, layers, hkv):
    """kv_read of every sequence after each step equals its model, in every layer: the copies of shared pages and the moves of
    compact and resize carry codes and exponents, and no sequence writes into another's pages."""
    torch, ops, L, cache, vlm, dev = env
    kv = cache.PagedKV(layers, 40, hkv, page)
    rng = np.random.default_rng(page)
    model = {}

    def check():
        ops.device_status()
        for s, m in model.items():
            one = kv.batch([s])
            one.extend([0])
            table, lens, _ = one.args
            for layer in range(layers):
                got = ops.kv_read(kv.pool, layer, table, lens, torch.zeros(1, dtype=torch.int32, device=dev), m.length + 3)
                for t, want in zip(got, m.kv[layer]):
                    t = t[0].float().cpu().numpy()
                    assert np.array_equal(t[:m.length], want.read(range(12), m.length)), (s, layer)
                    assert not t[m.length:].any()
        ops.device_status()

    def step(seqs, counts):
        batch = kv.batch(seqs)
        batch.extend(counts)
        for s, n in zip(seqs, counts):
            model[s].length += n
        for layer in range(layers):
            x = [O.bf16_round((rng.standard_normal((sum(counts), hkv, 128)) * 2.0 ** rng.integers(-6, 7, (sum(counts), 1, 1)))
                              .astype(np.float32)) for _ in range(2)]
            ops.kv_append(kv.pool, layer, *(bf16(torch, a, dev) for a in x), *batch.args)
            at = 0
            for s, n in zip(seqs, counts):
                if n:
                    model[s].append(layer, x[0][at:at + n], x[1][at:at + n])
                at += n
        check()

    def fork(s):
        t = kv.fork(s)
        model[t] = copy.deepcopy(model[s])
        return t

    z, a, b = (kv.new() for _ in range(3))
    model.update({s: Sequence(layers, hkv) for s in (z, a, b)})
    step([z], [66])
    step([a, b], [70, 33])
    step([a, b], [1, 1])
    c, d = fork(a), fork(a)
    moved = kv.pages(a)[-1]
    step([c], [1])                                       # a shared page, in its middle: c gets a copy
    assert kv.pages(a)[-1] == moved and kv.pages(c)[-1] != moved
    step([d, a, c], [4, 1, 3])                           # drafted tokens
    kv.truncate(d, kv.length(d) - 3)                     # and three taken back
    model[d].length -= 3
    step([d], [1])
    e = fork(d)
    kv.truncate(e, 66)                                   # into a page that others hold
    model[e].length = 66
    step([e, d], [5, 0])
    for s in (a, z):
        kv.free(s)
        del model[s]
    step([b, c], [1, 1])
    live = sum(1 for r in kv.refs if r)
    above = sum(1 for p, r in enumerate(kv.refs) if r and p >= live)
    assert above > 0 and kv.compact() == above           # pages above the live count are moved into the holes
    check()
    step([c, e], [1, 17])
    kv.resize(kv.pool.pages - kv.free_pages)
    check()
    with pytest.raises(cache.OutOfPages):
        kv.batch([b]).extend([500])
    kv.resize(40)
    check()
    step([b, c, d, e], [1, 2, 3, 4])


@pytest.mark.parametrize("few", [64, 0])
def test_a_captured_step_of_the_layers(env, few):
    """CachedLM.forward captured once and replayed after each extend gives, and leaves in the cache, what eager steps do."""
    torch, ops, L, cache, vlm, dev = env
    cfg = vlm.LMConfig(hidden=256, heads=4, kv_heads=2, ffn=384, layers=2)
    weights = vlm.random_lm_weights(cfg, seed=2)
    g = torch.Generator(device=dev)
    g.manual_seed(9)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    prompt = randn(50, 256).to(torch.bfloat16)
    steps = [(randn(2, 256).to(torch.bfloat16), randn(2, 64), randn(2, 64)) for _ in range(20)]
    rope = randn(50, 64), randn(50, 64)
    kvs = [cache.PagedKV(2, 16, 2, 16) for _ in range(2)]
    lms = [vlm.CachedLM(cfg, weights, kv, few=few) for kv in kvs]
    batches = []
    for kv, lm in zip(kvs, lms):
        batches.append(kv.batch([kv.new(), kv.new()], max_pages=8))
        batches[-1].extend([37, 13])
        lm.forward(prompt, batches[-1], *rope)
    x, cos, sin = (torch.empty_like(t) for t in steps[0])
    graph, out = None, None
    for i, (xi, ci, si) in enumerate(steps):
        for batch in batches:
            batch.extend([1, 1])
        want = lms[0].forward(xi, batches[0], ci, si)
        for t, v in zip((x, cos, sin), (xi, ci, si)):
            t.copy_(v)
        if graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                lms[1].forward(x, batches[1], cos, sin)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = lms[1].forward(x, batches[1], cos, sin)
        graph.replay()
        assert torch.equal(out, want), f"step {i}"
    ops.device_status()
    for layer in range(2):
        start = torch.zeros(2, dtype=torch.int32, device=dev)
        a, b = (ops.kv_read(kv.pool, layer, *batch.args[:2], start, 60) for kv, batch in zip(kvs, batches))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("M", [9, 16, 17, 24, 25, 32, 33, 48, 49, 64])
@pytest.mark.parametrize("K,N,G", [(40000, 130, 32), (1696, 9601, 32)])
def test_products_longer_than_a_panel_of_x(env, M, K, N, G):
    """More k tiles a share than shared memory holds of x, with K split over a cluster and not, ragged in K and N."""
    torch, ops, L, cache, vlm, dev = env
    rng = np.random.default_rng(M + K)
    x = O.bf16_round((rng.standard_normal((M, K)) * 3).astype(np.float32))
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = O.bf16_round((rng.standard_normal((K // G, N)) * 0.02).astype(np.float32))
    w = ops.Weight4.from_codes(torch.from_numpy(codes).to(dev), bf16(torch, scales, dev))
    got = ops.linear_w4(bf16(torch, x, dev), w, out_dtype=torch.float32)
    ops.device_status()
    # the oracle's product and bound (fp32 sum of K products), on the GPU in 64 bits
    wd = (torch.from_numpy(codes).to(dev).double() - 8) * torch.from_numpy(scales).to(dev).double().repeat_interleave(G, 0)
    xd = torch.from_numpy(x).to(dev).double()
    off = (got.double() - xd @ wd).abs() - (K * 2.0 ** -23 * (xd.abs() @ wd.abs()) + 1e-30)
    assert torch.isfinite(got).all() and off.max() <= 0
