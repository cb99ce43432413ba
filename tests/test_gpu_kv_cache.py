"""GPU parity of the 8-bit paged cache (rl_kv_append, rl_kv_read, rl_kv_copy_pages) and of the attention over it
(rl_kv_attention) against oracle/cache_oracle.py.

Codes and exponents are held bit for bit. Attention: |o - ref| <= the oracle's bound (fp16 weights, fp32 scores) plus
half a bf16 step, 2^-8 |ref|, of the output's rounding."""

import numpy as np
import pytest

from oracle import bfp16_oracle as O
from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from redline_tiny_b200 import _lib, ops
    assert torch.cuda.is_available()
    return torch, ops, _lib, torch.device("cuda:0")


@pytest.fixture(params=["split", "prompt", "cluster"])
def path(request, env):
    """Every kernel of kv_attention takes every shape."""
    ops = env[1]
    before = ops.set_kv_attention_path({"split": 1, "prompt": 2, "cluster": 3}[request.param])
    yield request.param
    ops.set_kv_attention_path(before)


def bf16(torch, a, dev):
    return torch.from_numpy(O.bf16_bits(np.asarray(a, np.float32)).view(np.int16)).to(dev).view(torch.bfloat16)


class Case:
    """A pool with a batch of sequences over shuffled pages, and the oracle's copy of it."""

    def __init__(self, torch, ops, dev, kv, new, hkv, page, layers=1, layer=0, seed=0, spare=2, wide=0):
        rng = np.random.default_rng(seed)
        self.rng, self.kv, self.new, self.hkv, self.page, self.layer = rng, kv, new, hkv, page, layer
        need = [-(-a // page) for a in kv]
        self.pages = sum(need) + spare
        perm = rng.permutation(self.pages)
        self.width = max(max(need), 1) + wide
        self.table = np.full((len(kv), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.free = perm[at:]
        shape = (layers, self.pages, hkv, page, 128)
        codes = [np.clip(np.rint(rng.standard_normal(shape) * 30) + 128, 0, 255).astype(np.uint8) for _ in range(2)]
        exps = [rng.integers(124, 131, (*shape[:3], page // 16)).astype(np.uint8) for _ in range(2)]
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.start[-1])
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.pool = ops.KVPool(t(codes[0]), t(codes[1]), t(exps[0]), t(exps[1]))
        self.d_table, self.d_len, self.d_start = t(self.table), t(np.asarray(kv, np.int32)), t(self.start)
        self.k = C.Cache(codes[0][layer].copy(), exps[0][layer].copy())
        self.v = C.Cache(codes[1][layer].copy(), exps[1][layer].copy())

    def args(self):
        return self.pool, self.layer, self.d_table, self.d_len, self.d_start

    def oracle(self, q, limits=None, present=None):
        o, tol = np.zeros(q.shape), np.zeros(q.shape)
        for b, (a, n) in enumerate(zip(self.kv, self.new)):
            r = slice(self.start[b], self.start[b + 1])
            lim = a - n + np.arange(n) if limits is None else np.minimum(limits[r], a - 1)
            o[r], tol[r] = C.attention(q[r].astype(np.float64), self.k.read(self.table[b], a),
                                       self.v.read(self.table[b], a), lim, None if present is None else present[b])
        return o, tol


def same_pool(case):
    lay = case.layer
    for got, want in ((case.pool.k, case.k.codes), (case.pool.v, case.v.codes), (case.pool.k_exp, case.k.exps),
                      (case.pool.v_exp, case.v.exps)):
        assert np.array_equal(got[lay].cpu().numpy(), want)


def check_attention(got, ref, tol):
    got = got.float().cpu().numpy().reshape(ref.shape).astype(np.float64)
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - tol - 2.0 ** -8 * np.abs(ref)
    assert off.max() <= 0, f"largest excess {off.max():.3e}"


APPENDS = [  # kv lengths (new tokens counted), new tokens, K/V heads, page
    ([1], [1], 1, 16), ([16], [1], 2, 16), ([17], [1], 2, 16), ([33, 1, 64], [1, 1, 1], 8, 32),
    ([100, 7, 64, 65], [50, 7, 64, 1], 2, 64), ([40, 20, 90], [0, 20, 33], 1, 128), ([300], [299], 3, 256),
    ([31, 31], [16, 15], 2, 16), ([1] * 40, [1] * 40, 2, 16), ([2900, 1300], [2899, 1300], 2, 64),
]


@pytest.mark.parametrize("kv,new,hkv,page", APPENDS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append(env, kv, new, hkv, page, dtype):
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, kv, new, hkv, page, layers=2, layer=1, seed=len(kv) * 7 + page)
    x = [(c.rng.standard_normal((c.T, hkv, 128)) * 4.0 ** c.rng.integers(-4, 4, (c.T, 1, 1))).astype(np.float32)
         for _ in range(2)]
    if dtype == "bf16":
        x = [O.bf16_round(a) for a in x]
        k, v = (bf16(torch, a, dev) for a in x)
    else:
        k, v = (torch.from_numpy(a).to(dev) for a in x)
    other = c.pool.k[0].clone(), c.pool.v_exp[0].clone()
    for b in range(len(kv)):
        r = slice(c.start[b], c.start[b + 1])
        c.k.append(c.table[b], kv[b], x[0][r])
        c.v.append(c.table[b], kv[b], x[1][r])
    for again in range(2):                       # writing the same tokens again changes nothing
        ops.kv_append(c.pool, 1, k, v, c.d_table, c.d_len, c.d_start)
        ops.device_status()
        same_pool(c)
    assert torch.equal(other[0], c.pool.k[0]) and torch.equal(other[1], c.pool.v_exp[0])
    first = torch.tensor([max(0, a - 20) for a in kv], dtype=torch.int32, device=dev)
    kr, vr = ops.kv_read(c.pool, 1, c.d_table, c.d_len, first, 23)
    ops.device_status()
    for got, cache in ((kr, c.k), (vr, c.v)):
        for b, a in enumerate(kv):
            want = np.zeros((23, hkv, 128))
            seq = cache.read(c.table[b], a)[max(0, a - 20):]
            want[:len(seq)] = seq
            assert np.array_equal(got[b].float().cpu().numpy(), want)


def test_append_values_at_the_edges(env):
    """Ties, the largest and smallest magnitudes, subnormals, zero blocks; a NaN or an infinity poisons its block."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [64], [64], 1, 64)
    x = np.zeros((64, 1, 128), np.float32)
    x[0:16] = np.arange(2048).reshape(16, 1, 128) * 0.5 - 512       # halves: ties
    x[16:32] = np.float32(3.3e38) * np.linspace(-1, 1, 2048).reshape(16, 1, 128)
    x[32:48] = np.float32(1e-45) * np.arange(2048).reshape(16, 1, 128)
    k, v = torch.from_numpy(x).to(dev), torch.from_numpy(-x).to(dev)
    ops.kv_append(c.pool, 0, k, v, c.d_table, c.d_len, c.d_start)
    c.k.append(c.table[0], 64, x)
    c.v.append(c.table[0], 64, -x)
    ops.device_status()
    same_pool(c)
    for bad in (np.nan, np.inf, -np.inf):
        x[20, 0, 5] = bad
        ops.kv_append(c.pool, 0, torch.from_numpy(x).to(dev), v, c.d_table, c.d_len, c.d_start)
        kr, vr = ops.kv_read(c.pool, 0, c.d_table, c.d_len, torch.zeros(1, dtype=torch.int32, device=dev), 64)
        nan = torch.isnan(kr).cpu().numpy()[0]
        assert nan[16:32].all() and not nan[:16].any() and not nan[32:].any() and not torch.isnan(vr).any()
    ops.device_status()


@pytest.mark.parametrize("layout", ["heads_first", "transposed_v", "offset"])
def test_append_strided(env, layout):
    """k (H, T, 128), V^T (H, 128, ldv) as qkv_post leaves them, and rows inside a larger buffer at an odd offset."""
    torch, ops, L, dev = env
    kv, new, hkv = [70, 19], [41, 2], 2
    c = Case(torch, ops, dev, kv, new, hkv, 32, seed=3)
    x = [O.bf16_round(c.rng.standard_normal((c.T, hkv, 128)).astype(np.float32)) for _ in range(2)]
    k, v = (bf16(torch, a, dev) for a in x)
    if layout == "heads_first":
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    elif layout == "transposed_v":
        vt = torch.zeros((hkv, 128, 128), dtype=torch.bfloat16, device=dev)
        vt[:, :, :c.T] = v.permute(1, 2, 0)
        v = vt.permute(2, 0, 1)[:c.T]
    else:
        buf = torch.zeros((c.T, hkv, 259), dtype=torch.bfloat16, device=dev)
        buf[:, :, 1:129], buf[:, :, 130:258] = k, v
        k, v = buf[:, :, 1:129], buf[:, :, 130:258]
    ops.kv_append(c.pool, 0, k, v, c.d_table, c.d_len, c.d_start)
    ops.device_status()
    for b in range(2):
        r = slice(c.start[b], c.start[b + 1])
        c.k.append(c.table[b], kv[b], x[0][r])
        c.v.append(c.table[b], kv[b], x[1][r])
    same_pool(c)


def test_append_token_by_token(env):
    """A sequence written one token at a time, with growing and shrinking magnitudes, equals the oracle's."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [40], [1], 2, 16)
    x = (c.rng.standard_normal((40, 2, 128)) * 2.0 ** c.rng.integers(-9, 9, (40, 1, 1))).astype(np.float32)
    for t in range(40):
        ops.kv_append(c.pool, 0, torch.from_numpy(x[t:t + 1]).to(dev), torch.from_numpy(x[t:t + 1]).to(dev), c.d_table,
                      torch.tensor([t + 1], dtype=torch.int32, device=dev), c.d_start)
        for cache in (c.k, c.v):
            cache.append(c.table[0], t + 1, x[t:t + 1])
    ops.device_status()
    same_pool(c)


ATTENDS = [  # kv lengths, new tokens, heads, K/V heads, page
    ([1], [1], 1, 1, 16), ([15], [1], 4, 2, 16), ([16], [1], 4, 1, 16), ([17], [1], 8, 1, 32), ([63], [1], 3, 3, 64),
    ([64], [1], 4, 2, 64), ([65], [1], 6, 2, 128), ([1000], [1], 4, 1, 64), ([777, 1, 300, 16, 513], [1] * 5, 8, 2, 64),
    ([70, 5, 200], [4, 5, 1], 4, 2, 16), ([50, 64, 90], [0, 3, 0], 4, 1, 16), ([130], [130], 4, 2, 32),
    ([257, 40], [100, 40], 8, 2, 16), ([90, 33], [60, 33], 12, 1, 256), ([2500], [3], 16, 1, 64),
    ([40 + 13 * i for i in range(50)], [1 + i % 3 for i in range(50)], 4, 2, 16),
    ([400, 130, 700], [300, 130, 129], 6, 2, 64), ([128, 256, 129], [64, 64, 65], 4, 1, 32),
]


@pytest.mark.parametrize("kv,new,H,hkv,page", ATTENDS)
def test_attention(env, path, kv, new, H, hkv, page):
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, kv, new, hkv, page, layers=2, layer=1, seed=sum(kv) + H, wide=len(kv) % 3)
    q = O.bf16_round((c.rng.standard_normal((c.T, H, 128)) * 2).astype(np.float32))
    out = torch.full((c.T + 2, H * 128 + 8), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.kv_attention(bf16(torch, q, dev), *c.args(), out=out[1:c.T + 1, :H * 128])
    ops.device_status()
    check_attention(got, *c.oracle(q))
    assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[:, H * 128:] == 7).all()
    again = ops.kv_attention(bf16(torch, q, dev), *c.args())
    assert torch.equal(again, got)


def test_attention_sharp_and_wide_scores(env, path):
    """Large logits (one key dominates, the maximum rises along the sequence) and rows of very different magnitude."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [400, 90], [2, 9], 2, 32, seed=5)
    q = c.rng.standard_normal((c.T, 4, 128)) * np.array([1e-6, 1.0, 30.0, 300.0])[None, :, None]
    q = O.bf16_round(q.astype(np.float32))
    got = ops.kv_attention(bf16(torch, q, dev), *c.args())
    ops.device_status()
    check_attention(got, *c.oracle(q))


def test_attention_blocks_of_very_different_scale(env, path):
    """V and K blocks from 2^-40 to 2^40 and all-zero ones, in every order."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [700, 300], [1, 3], 2, 16, seed=15)
    for cache, exps in ((c.k, c.pool.k_exp), (c.v, c.pool.v_exp)):
        e = c.rng.choice([0, 90, 120, 125, 127, 128, 130, 138, 160], cache.exps.shape).astype(np.uint8)
        if cache is c.k:
            e = np.minimum(e, 130)
        cache.exps[:] = e
        exps[0] = torch.from_numpy(e).to(dev)
    c.v.codes[c.v.exps.repeat(16, 2) == 0] = 128
    c.pool.v[0] = torch.from_numpy(c.v.codes).to(dev)
    q = O.bf16_round(c.rng.standard_normal((c.T, 4, 128)).astype(np.float32))
    got = ops.kv_attention(bf16(torch, q, dev), *c.args())
    ops.device_status()
    check_attention(got, *c.oracle(q))


def test_attention_row_limits(env, path):
    """Per-row limits: none visible (zeros), one key, past the end, and beyond the causal limit."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [100, 37], [6, 5], 2, 16, seed=6)
    q = O.bf16_round(c.rng.standard_normal((c.T, 4, 128)).astype(np.float32))
    lim = np.array([-1, 0, 15, 16, 99, 1000, -5, 36, 3, 31, 32], np.int32)
    got = ops.kv_attention(bf16(torch, q, dev), *c.args(), row_limit=torch.from_numpy(lim).to(dev))
    ops.device_status()
    check_attention(got, *c.oracle(q, lim))
    assert (got[0] == 0).all() and (got[6] == 0).all()


def test_attention_strides_scale(env, path):
    """q (H, T, 128) as qkv_post leaves it, and a caller's scale."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [77], [9], 1, 64, seed=8)
    q = O.bf16_round(c.rng.standard_normal((c.T, 2, 128)).astype(np.float32))
    qt = bf16(torch, q.transpose(1, 0, 2).copy(), dev).transpose(0, 1)
    got = ops.kv_attention(qt, *c.args(), scale_log2=0.25 * np.log2(np.e) / np.sqrt(128))
    ops.device_status()
    check_attention(got, *c.oracle(q * np.float32(0.25)))


def test_attention_poisoned_block(env, path):
    """A block that took in a NaN gives NaN to the rows that see it and to no other."""
    torch, ops, L, dev = env
    for which in ("k", "v"):
        c = Case(torch, ops, dev, [64], [40], 1, 16, seed=9)
        q = O.bf16_round(c.rng.standard_normal((40, 2, 128)).astype(np.float32))
        clean, _ = c.oracle(q)
        getattr(c.pool, which + "_exp")[0, int(c.table[0, 2])] = 255     # positions 32 .. 47, seen by rows >= 8
        got = ops.kv_attention(bf16(torch, q, dev), *c.args()).float().cpu().numpy()
        ops.device_status()
        assert np.isnan(got[8:]).all() and np.isfinite(got[:8]).all()
        assert np.abs(got[:8] - clean[:8].reshape(8, -1)).max() < 0.1


def test_bad_pages_and_sequences_are_reported(env, path):
    """A page outside the pool: its keys count as absent. Impossible sequences are left out. Both set the error word."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [100, 40], [2, 1], 2, 16, seed=10)
    q = O.bf16_round(c.rng.standard_normal((c.T, 4, 128)).astype(np.float32))
    table = c.table.copy()
    table[0, 1], table[0, 3] = -1, c.pages
    present = [np.ones(100, bool), np.ones(40, bool)]
    present[0][16:32] = present[0][48:64] = False
    d_table = torch.from_numpy(table).to(dev)
    got = ops.kv_attention(bf16(torch, q, dev), c.pool, 0, d_table, c.d_len, c.d_start)
    with pytest.raises(L.RedlineError, match="range check"):
        ops.device_status()
    check_attention(got, *c.oracle(q, present=present))
    before = c.pool.k.clone()
    kr, _ = ops.kv_read(c.pool, 0, d_table, c.d_len, torch.tensor([16, 0], dtype=torch.int32, device=dev), 16)
    assert (kr[0] == 0).all() and not (kr[1] == 0).all()
    with pytest.raises(L.RedlineError):
        ops.device_status()
    x = torch.ones((c.T, 2, 128), dtype=torch.bfloat16, device=dev)
    bad = table.copy()
    bad[:, :] = c.pages
    ops.kv_append(c.pool, 0, x, x, torch.from_numpy(bad).to(dev), c.d_len, c.d_start)
    with pytest.raises(L.RedlineError):
        ops.device_status()
    assert torch.equal(before, c.pool.k)
    for kv_len, start in (([1000, 40], [0, 2, 3]), ([1, 40], [0, 2, 3]), ([100, 40], [0, 2, 9]), ([-5, 40], [0, 2, 3]),
                          ([100, 40], [3, 2, 3]), ([100, 40], [-1, 2, 3])):
        lens, st = (torch.tensor(a, dtype=torch.int32, device=dev) for a in (kv_len, start))
        out = torch.full((c.T, 512), 7.0, dtype=torch.bfloat16, device=dev)
        ops.kv_attention(bf16(torch, q, dev), c.pool, 0, c.d_table, lens, st, out=out)
        with pytest.raises(L.RedlineError):
            ops.device_status()
        broken = 1 if start[-1] == 9 else 0
        rows = slice(0, 2) if broken == 0 else slice(2, 3)
        assert (out[rows] == 7).all()


@pytest.mark.parametrize("n,layers,hkv,page", [(1, 1, 1, 16), (5, 3, 2, 64), (40, 2, 8, 128), (1500, 2, 1, 16)])
def test_copy_pages(env, n, layers, hkv, page):
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [page], [1], hkv, page, layers=layers, spare=2 * n + 3, seed=n)
    perm = c.rng.permutation(c.pages)
    src, dst = perm[:n].tolist(), perm[n:2 * n].tolist()
    src[-1] = src[0]                                                  # one page copied to two others
    want = [t.clone() for t in (c.pool.k, c.pool.v, c.pool.k_exp, c.pool.v_exp)]
    for t in want:
        t[:, dst] = t[:, src]
    ops.kv_copy_pages(c.pool, src, dst)
    ops.device_status()
    for got, w in zip((c.pool.k, c.pool.v, c.pool.k_exp, c.pool.v_exp), want):
        assert torch.equal(got, w)


def test_append_and_attend_in_a_graph(env, path):
    """A captured decode step follows the device-side lengths when it is replayed."""
    torch, ops, L, dev = env
    H, hkv = 4, 2
    c = Case(torch, ops, dev, [30, 50], [1, 1], hkv, 16, seed=12, wide=2)
    kn, vn = (torch.empty((2, hkv, 128), dtype=torch.bfloat16, device=dev) for _ in range(2))
    q, out = torch.empty((2, H, 128), dtype=torch.bfloat16, device=dev), None

    def step():
        ops.kv_append(c.pool, 0, kn, vn, c.d_table, c.d_len, c.d_start)
        return ops.kv_attention(q, c.pool, 0, c.d_table, c.d_len, c.d_start)

    data = [[O.bf16_round(c.rng.standard_normal((2, h, 128)).astype(np.float32)) for h in (hkv, hkv, H)] for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t, a in zip((kn, vn, q), data[0]):
            t.copy_(bf16(torch, a, dev))
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, d in enumerate(data):
        kv = [30 + (i % 2), 50 + (i % 2)]
        c.kv = kv
        c.d_len.copy_(torch.tensor(kv, dtype=torch.int32))
        for t, a in zip((kn, vn, q), d):
            t.copy_(bf16(torch, a, dev))
        graph.replay()
        for b in range(2):
            c.k.append(c.table[b], kv[b], d[0][b:b + 1])
            c.v.append(c.table[b], kv[b], d[1][b:b + 1])
        ops.device_status()
        same_pool(c)
        check_attention(out, *c.oracle(d[2]))


def test_both_bindings(env, monkeypatch):
    """The compiled binding and the ctypes one write, read, attend and refuse alike, whatever strides and optional
    arguments they are given."""
    torch, ops, L, dev = env
    assert ops._fast is not None, "the extension is built with the library"
    results = []
    for binding in (ops._fast, None):
        monkeypatch.setattr(ops, "_fast", binding)
        c = Case(torch, ops, dev, [90, 33, 40], [20, 0, 3], 2, 16, seed=21)
        x = O.bf16_round(c.rng.standard_normal((c.T, 2, 128)).astype(np.float32))
        q = O.bf16_round(c.rng.standard_normal((c.T, 4, 128)).astype(np.float32))
        k, qt = bf16(torch, x, dev), bf16(torch, q, dev)
        kt = k.transpose(0, 1).contiguous().transpose(0, 1)
        ops.kv_append(c.pool, 0, kt, k, *c.args()[2:])
        ops.kv_append(c.pool, 0, kt.float(), k.float(), *c.args()[2:])
        got = [c.pool.k, c.pool.v, c.pool.k_exp, *ops.kv_read(c.pool, 0, c.d_table, c.d_len, c.d_len - 30, 35)]
        lim = torch.arange(c.T, dtype=torch.int32, device=dev)
        out = torch.zeros((c.T, 1024), dtype=torch.bfloat16, device=dev)
        got += [ops.kv_attention(qt, *c.args()), ops.kv_attention(qt, *c.args(), row_limit=lim, scale_log2=0.1),
                ops.kv_attention(qt[:, ::2], c.pool, 0, *c.args()[2:]), ops.kv_attention(qt, *c.args(), out=out[:, 512:]), out]
        w = ops.Weight4.from_float(torch.arange(64 * 48, device=dev).reshape(64, 48).float().cos(), 32)
        b = torch.ones(48, dtype=torch.bfloat16, device=dev)
        xs = k.reshape(-1, 64)[:5].contiguous()
        got += [ops.linear_w4(xs, w), ops.linear_w4(xs, w, bias=b), ops.linear_w4(xs, w, out_dtype=torch.float32),
                ops.linear_w4(xs, w, out=torch.empty((5, 48), device=dev))]
        for bad in (lambda: ops.kv_attention(qt.float(), *c.args()), lambda: ops.kv_append(c.pool, 0, kt[:, :1], k[:, :1], *c.args()[2:]),
                    lambda: ops.kv_attention(qt, c.pool, 1, *c.args()[2:]), lambda: ops.kv_attention(qt, c.pool, -1, *c.args()[2:]),
                    lambda: ops.kv_read(c.pool, 0, c.d_table, c.d_len.long(), c.d_len, 3), lambda: ops.linear_w4(xs.t(), w),
                    lambda: ops.linear_w4(xs.cpu(), w), lambda: ops.kv_attention(qt.cpu(), *c.args()),
                    lambda: ops.linear_w4(xs, w, bias=b[:40])):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(L.RedlineError, match="heads"):
            ops.kv_attention(qt[:, :3], *c.args())
        with pytest.raises(L.RedlineError, match="rows"):
            ops.linear_w4(torch.zeros((65, 64), dtype=torch.bfloat16, device=dev), w)
        ops.device_status()
        results.append([t.clone() for t in got])
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_pages_behind_four_gigabytes(env, path):
    """Writes, reads, copies and attention at byte offsets that pass 32 bits (codes of K and of V: 4.8 GB each)."""
    torch, ops, L, dev = env
    pages, hkv, page = 36500, 8, 128
    pool = ops.KVPool.empty(1, pages, hkv, page)
    rng = np.random.default_rng(31)
    kv = 300
    table = np.array([[pages - 1, 3, pages - 7]], np.int32)
    d_table, d_len = torch.from_numpy(table).to(dev), torch.tensor([kv], dtype=torch.int32, device=dev)
    start = torch.tensor([0, kv], dtype=torch.int32, device=dev)
    x = [O.bf16_round(rng.standard_normal((kv, hkv, 128)).astype(np.float32)) for _ in range(2)]
    ops.kv_append(pool, 0, *(bf16(torch, a, dev) for a in x), d_table, d_len, start)
    kr, vr = ops.kv_read(pool, 0, d_table, d_len, torch.zeros(1, dtype=torch.int32, device=dev), kv)
    # the same sequence in a small pool
    small = ops.KVPool.empty(1, 4, hkv, page)
    t2 = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    ops.kv_append(small, 0, *(bf16(torch, a, dev) for a in x), t2, d_len, start)
    ks, vs = ops.kv_read(small, 0, t2, d_len, torch.zeros(1, dtype=torch.int32, device=dev), kv)
    assert torch.equal(kr, ks) and torch.equal(vr, vs)
    q = bf16(torch, rng.standard_normal((5, 16, 128)).astype(np.float32), dev)
    rows = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    want = ops.kv_attention(q, small, 0, t2, d_len, rows)
    assert torch.equal(ops.kv_attention(q, pool, 0, d_table, d_len, rows), want)
    ops.kv_copy_pages(pool, [pages - 1, 3, pages - 7], [11, pages - 20, 12])
    t3 = torch.tensor([[11, pages - 20, 12]], dtype=torch.int32, device=dev)
    assert torch.equal(ops.kv_attention(q, pool, 0, t3, d_len, rows), want)
    ops.device_status()


def test_the_kernel_goes_by_shape(env):
    """A decode step takes the split kernel, in clusters where the context is short, and a long chunk the prompt kernel; they
    agree within two weights' rounding and the output's."""
    torch, ops, L, dev = env
    for kv, new, H, hkv, which in (([500, 300], [1, 1], 8, 2, 3), ([6200, 300], [1, 1], 8, 2, 1),
                                   ([900, 700], [900, 700], 32, 8, 2)):
        c = Case(torch, ops, dev, kv, new, hkv, 64, seed=41)
        q = bf16(torch, c.rng.standard_normal((c.T, H, 128)).astype(np.float32), dev)
        got = []
        for path in (0, 1, 2, 3):
            before = ops.set_kv_attention_path(path)
            got.append(ops.kv_attention(q, *c.args()))
            ops.set_kv_attention_path(before)
        ops.device_status()
        assert torch.equal(got[0], got[which])
        a, b = got[1].float(), got[2].float()
        top = b.abs().reshape(c.T, H, 128).amax(-1, keepdim=True).expand(-1, -1, 128).reshape_as(b)
        assert ((a - b).abs() <= 2.0 ** -7 * top).all()


def test_steps_with_many_sequences(env):
    """1024 sequences of up to 40 tokens, the most a call takes; one more is refused."""
    torch, ops, L, dev = env
    kv = [1 + i % 40 for i in range(1024)]
    c = Case(torch, ops, dev, kv, [1] * 1024, 1, 16, seed=51)
    q = O.bf16_round(c.rng.standard_normal((c.T, 2, 128)).astype(np.float32))
    got = ops.kv_attention(bf16(torch, q, dev), *c.args())
    ops.device_status()
    check_attention(got, *c.oracle(q))
    t = torch.zeros((1025, 1), dtype=torch.int32, device=dev)
    with pytest.raises(L.RedlineError, match="1025 sequences"):
        ops.kv_attention(bf16(torch, q, dev), c.pool, 0, t, t[:, 0].contiguous(), torch.zeros(1026, dtype=torch.int32, device=dev))
