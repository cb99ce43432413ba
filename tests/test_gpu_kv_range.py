"""GPU parity of the attention over the 8-bit paged cache (rl_kv_attention) at the ends of its numeric range: values whose
scales lie far apart, values near the largest float, long tails of small weights.

|o - ref| <= the bound of oracle/cache_oracle.py, which is relative to the largest value that the ROW sees, plus half a bf16
step, 2^-8 |ref|, of the output's rounding. A key that the mask hides from a row must not reach the row in any form."""

import numpy as np
import pytest

from oracle import bfp16_oracle as O
from test_gpu_kv_cache import Case, bf16, check_attention

pytestmark = pytest.mark.gpu

FORMS = {"split": 1, "prompt": 2, "cluster": 3}


@pytest.fixture(scope="module")
def env():
    import torch
    from redline_tiny_b200 import _lib, ops
    assert torch.cuda.is_available()
    return torch, ops, _lib, torch.device("cuda:0")


def attend(ops, form, *args, **kw):
    before = ops.set_kv_attention_path(FORMS[form])
    try:
        return ops.kv_attention(*args, **kw)
    finally:
        ops.set_kv_attention_path(before)


def value_exponents(c, torch, dev, exps):
    """Give the blocks of sequence b's values the exponents exps(b, first position of the block)."""
    for b in range(len(c.kv)):
        for pos in range(0, c.kv[b], 16):
            c.v.exps[c.table[b, pos // c.page], :, pos % c.page // 16] = exps(b, pos)
    c.pool.v_exp[c.layer] = torch.from_numpy(c.v.exps).to(dev)


def limits(c, rng, at):
    """Row limits: nothing, one key, and keys up to and beyond position `at`."""
    lim = rng.integers(-1, max(c.kv), c.T)
    lim[::3] = rng.integers(0, at, len(lim[::3]))
    lim[1::7] = -1
    return lim.astype(np.int32)


def hidden_values(env, form, spread, masks, kv, new, H, hkv, page):
    """From position 192 on, values 2^spread times the others: the rows that see none of them keep their own scale."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, kv, new, hkv, page, seed=spread + H)
    low = 120 - spread // 2
    value_exponents(c, torch, dev, lambda b, pos: low + spread if pos >= 192 else low)
    q = O.bf16_round(c.rng.standard_normal((c.T, H, 128)).astype(np.float32))
    lim = limits(c, c.rng, 192) if masks == "row_limit" else None
    got = attend(ops, form, bf16(torch, q, dev), *c.args(), row_limit=None if lim is None else torch.from_numpy(lim).to(dev))
    ops.device_status()
    ref, tol = c.oracle(q, lim)
    sees = np.concatenate([a - n + np.arange(n) for a, n in zip(kv, new)]) if lim is None else lim
    below = ref[(sees >= 0) & (sees < 192)]
    assert len(below) and np.abs(below).max() > 0
    check_attention(got, ref, tol)


HIDDEN = [([300], [300], 2, 1, 16), ([700, 250], [600, 130], 4, 2, 64)]


@pytest.mark.parametrize("kv,new,H,hkv,page", HIDDEN)
@pytest.mark.parametrize("masks", ["causal", "row_limit"])
@pytest.mark.parametrize("form", ["split", "cluster"])
def test_hidden_values_far_above(env, form, masks, kv, new, H, hkv, page):
    hidden_values(env, form, 180, masks, kv, new, H, hkv, page)


@pytest.mark.parametrize("kv,new,H,hkv,page", HIDDEN)
@pytest.mark.parametrize("masks", ["causal", "row_limit"])
@pytest.mark.parametrize("spread", [4, 24, 25, 29, 30, 31, 40, 100, 180])
@pytest.mark.parametrize("form", ["split", "prompt", "cluster"])
def test_hidden_values(env, form, spread, masks, kv, new, H, hkv, page):
    hidden_values(env, form, spread, masks, kv, new, H, hkv, page)


@pytest.mark.parametrize("form", ["split", "prompt", "cluster"])
def test_hidden_values_beside_absent_and_poisoned_blocks(env, form):
    """Values far apart, a page outside the pool among the low and one among the high ones, a block with a NaN behind; q and
    the output with strides of their own."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [330, 40], [300, 40], 2, 16, seed=13)
    value_exponents(c, torch, dev, lambda b, pos: 150 if pos >= 192 else 110)
    table = c.table.copy()
    table[0, 3], table[0, 13] = -1, c.pages
    present = [np.ones(330, bool), np.ones(40, bool)]
    present[0][48:64] = present[0][208:224] = False
    c.pool.v_exp[0, int(table[0, 17])] = 255                           # positions 272 .. 287
    q = O.bf16_round(c.rng.standard_normal((c.T, 4, 128)).astype(np.float32))
    out = torch.full((c.T, 523), 7.0, dtype=torch.bfloat16, device=dev)
    attend(ops, form, bf16(torch, q.transpose(1, 0, 2).copy(), dev).transpose(0, 1), c.pool, 0, torch.from_numpy(table).to(dev),
           c.d_len, c.d_start, out=out[:, 1:513])
    with pytest.raises(L.RedlineError, match="range check"):
        ops.device_status()
    assert (out[:, 0] == 7).all() and (out[:, 513:] == 7).all()
    ref, tol = c.oracle(q, present=present)
    sees = np.arange(c.T) + 30 >= 272
    sees[300:] = False
    got = out[:, 1:513].float().cpu().numpy().reshape(ref.shape)
    assert np.isnan(got[sees]).all()
    check_attention(torch.from_numpy(got[~sees]), ref[~sees], tol[~sees])


@pytest.mark.parametrize("kv,new,H", [([3000], [1], 4), ([2000, 900], [40, 300], 2)])
@pytest.mark.parametrize("form", ["split", "prompt", "cluster"])
def test_values_near_the_largest(env, form, kv, new, H):
    """Values up to 2^127 over thousands of keys: the sum of weights does not overflow the sum of values."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, kv, new, 1, 64, seed=3)
    value_exponents(c, torch, dev, lambda b, pos: 254 - pos // 16 % 3)
    q = O.bf16_round((c.rng.standard_normal((c.T, H, 128)) * 0.1).astype(np.float32))
    got = attend(ops, form, bf16(torch, q, dev), *c.args())
    ops.device_status()
    check_attention(got, *c.oracle(q))


@pytest.mark.parametrize("weight", [-22.3, -24.9, -25.0, -26.5])
@pytest.mark.parametrize("form", ["split", "prompt", "cluster"])
def test_a_long_tail_of_small_weights(env, form, weight):
    """One key holds nearly all of the softmax, 131071 others 2^weight of it each: their values count."""
    torch, ops, L, dev = env
    n = 131072
    c = Case(torch, ops, dev, [n], [1], 1, 64, seed=7)
    sink = c.table[0, 0]
    for cache, codes, exps in ((c.k, c.pool.k, c.pool.k_exp), (c.v, c.pool.v, c.pool.v_exp)):
        cache.exps[:] = 133                                          # values are codes - 128
        cache.codes[:] = 128 if cache is c.k else 128 + 100
        if cache is c.k:
            cache.codes[sink, 0, 0, :64] = 129                       # the first key's score
        else:
            cache.codes[sink, 0, 0] = 128                            # and its value, zero
        codes[0] = torch.from_numpy(cache.codes).to(dev)
        exps[0] = torch.from_numpy(cache.exps).to(dev)
    q = np.zeros((1, 2, 128), np.float32)
    q[:, :, :64] = O.bf16_round(np.full(64, -weight * np.log(2) * np.sqrt(128) / 64, np.float32))
    got = attend(ops, form, bf16(torch, q, dev), *c.args())
    ops.device_status()
    check_attention(got, *c.oracle(q))


# (the second and third have work for several blocks a warp, whose scales then meet)
@pytest.mark.parametrize("kv,new,H", [([300, 90], [12, 3], 2), ([2000], [700], 4), ([2600] * 30, [1] * 30, 2)])
@pytest.mark.parametrize("form", ["split", "prompt", "cluster"])
def test_absent_pages_bring_no_scale_with_them(env, form, kv, new, H):
    """A page outside the pool among a sequence's: what the kernels read in its place, large values or a NaN, counts for nothing."""
    torch, ops, L, dev = env
    for there in (140, 255):
        c = Case(torch, ops, dev, kv, new, 1, 16, seed=19)
        free = int(c.free[0])
        order = [free] + [p for p in range(c.pages) if p != free]            # page 0 belongs to no sequence
        for t in (c.pool.k, c.pool.v, c.pool.k_exp, c.pool.v_exp):
            t[:] = t[:, order].clone()
        for cache in (c.k, c.v):
            cache.codes, cache.exps = cache.codes[order], cache.exps[order]
        back = np.argsort(order)
        c.table = np.where(c.table >= 0, back[c.table], -1).astype(np.int32)
        c.pool.k_exp[0, 0], c.pool.v_exp[0, 0] = 255 if there == 255 else 127, there
        table, present = c.table.copy(), [np.ones(a, bool) for a in kv]
        for b, a in enumerate(kv):
            for p in range(1, a // 16, 3):
                table[b, p] = -1 if p % 2 else c.pages + 7
                present[b][16 * p:16 * p + 16] = False
        q = O.bf16_round((c.rng.standard_normal((c.T, H, 128)) * 0.1).astype(np.float32))
        got = attend(ops, form, bf16(torch, q, dev), c.pool, 0, torch.from_numpy(table).to(dev), c.d_len, c.d_start)
        with pytest.raises(L.RedlineError, match="range check"):
            ops.device_status()
        check_attention(got, *c.oracle(q, present=present))
