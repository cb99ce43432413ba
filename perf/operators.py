"""The operators that generate tokens, as cases to be timed and compared: writing new keys and values into the 8-bit
paged cache, attention over that cache, copying its pages, and products of a few rows with 4-bit weights.

`run` computes a case in elementary torch operations (own = False) or through redline_tiny_b200.ops (own = True).
Sizes are those of the text decoder's default configuration (hidden 4096, 32 query heads, 8 K/V heads, FFN 12288,
head dim 128), of the smaller decoder layers that the tests use, and generic ones."""

import math

import torch

own = False

HEAD = 128
BLOCK = 16          # tokens that share one exponent (per K/V head)
DEV = "cuda"
SCALE_LOG2 = math.log2(math.e) / math.sqrt(HEAD)


def listed():
    return [
        # one sequence's newest token: the latency of a single decode step's cache write
        dict(name="append_token", op="append", batch=1, kv=778, new=1, kv_heads=8, page=64),
        # four prompts of different lengths admitted together, one of them behind a prefix that is cached already
        dict(name="append_prompts", op="append", batch=4, kv=4095, new=3001, kv_heads=8, page=64),
        # a chat turn of one user: short context, one query token
        dict(name="attend_short", op="attend", batch=1, kv=777, new=1, heads=32, kv_heads=8, page=64),
        # one user with a very long document: all of the GPU has to share one sequence
        dict(name="attend_long", op="attend", batch=1, kv=131071, new=1, heads=32, kv_heads=8, page=64),
        # a full decode batch of sequences of very different lengths
        dict(name="attend_batch", op="attend", batch=64, kv=8192, new=1, heads=32, kv_heads=8, page=64),
        # a few drafted tokens per sequence checked at once, small pages, a smaller decoder
        dict(name="attend_drafts", op="attend", batch=16, kv=4097, new=5, heads=8, kv_heads=2, page=16),
        # chunks of prompts attending over what is cached and over themselves
        dict(name="attend_prompts", op="attend", batch=3, kv=8191, new=1021, heads=32, kv_heads=8, page=64),
        # the last page of a forked sequence, copied before its first write, in a decoder of two layers
        dict(name="copy_page", op="copy", pages=64, copies=1, layers=2, kv_heads=8, page=64),
        # a pool compacted: the pages above its live count moved into the holes, in every layer
        dict(name="copy_pool", op="copy", pages=512, copies=203, layers=36, kv_heads=8, page=64),
        # one token through the QKV projection
        dict(name="w4_token", op="w4", rows=1, k=4096, n=6144, group=64, swiglu=False, bias=False),
        # one token through the gate and up projections with their activation
        dict(name="w4_swiglu", op="w4", rows=1, k=4096, n=24576, group=64, swiglu=True, bias=False),
        # a decode batch through the down projection
        dict(name="w4_batch", op="w4", rows=23, k=12288, n=4096, group=128, swiglu=False, bias=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "copy", "w4", "w4"])
    if op == "append":
        batch = _spread(rng, 1, 64)
        kv = _spread(rng, 1, 16000 // batch)
        return dict(op=op, batch=batch, kv=kv, new=rng.choice([1, _spread(rng, 1, kv)]),
                    kv_heads=rng.choice([1, 2, 8]), page=rng.choice([16, 32, 64, 128]))
    if op == "attend":
        batch, kv_heads = _spread(rng, 1, 64), rng.choice([1, 2, 8])
        kv = _spread(rng, 1, 131072 * 2 // batch if batch > 2 else 131072)
        new = rng.choice([1, min(kv, _spread(rng, 1, 8)), min(kv, _spread(rng, 1, max(1, 8000000 // (kv * batch))))])
        return dict(op=op, batch=batch, kv=kv, new=new, heads=kv_heads * rng.choice([1, 2, 4]), kv_heads=kv_heads,
                    page=rng.choice([16, 32, 64, 128]))
    if op == "copy":
        pages = _spread(rng, 8, 512)
        return dict(op=op, pages=pages, copies=rng.randint(1, pages // 3), layers=_spread(rng, 1, 36),
                    kv_heads=rng.choice([1, 2, 8]), page=rng.choice([16, 32, 64]))
    group = rng.choice([32, 64, 128])
    swiglu = rng.random() < 0.3
    return dict(op=op, rows=_spread(rng, 1, 64), k=group * max(1, _spread(rng, 128, 12288) // group),
                n=_spread(rng, 1, 96) * 256 if swiglu else _spread(rng, 64, 12288), group=group, swiglu=swiglu, bias=rng.random() < 0.5)


def _lengths(case):
    """Cached tokens (the new ones included) and new tokens of each sequence: the first is the longest, the others are
    spread evenly; in larger batches the last slot is an ended sequence without new tokens."""
    kv, new = [], []
    for b in range(case["batch"]):
        f = 1.0 if b == 0 else 0.05 + 0.95 * ((b * 0.6180339887498949) % 1.0)
        n = max(1, int(case["new"] * f))
        kv.append(max(n, int(case["kv"] * f)))
        new.append(n)
    if case["batch"] >= 8:
        new[-1] = 0
    return kv, new


def work(case):
    if case["op"] == "copy":
        page = 2 * case["kv_heads"] * (case["page"] * HEAD + case["page"] // BLOCK)
        return {"bytes": 2 * case["copies"] * case["layers"] * page, "flops": 0}
    if case["op"] == "w4":
        m, k, n = case["rows"], case["k"], case["n"]
        out = n // 2 if case["swiglu"] else n
        return {"bytes": k * n // 2 + 2 * n * k // case["group"] + 2 * m * k + 2 * m * out + 2 * n * case["bias"],
                "flops": 2 * m * n * k}
    kv, new = _lengths(case)
    hk = case["kv_heads"]
    if case["op"] == "append":
        # new K and V in (bf16), codes out, and the touched blocks read back as bf16
        blocks = sum((a + BLOCK - 1) // BLOCK - (a - n) // BLOCK for a, n in zip(kv, new) if n)
        t = sum(new)
        return {"bytes": 2 * hk * (HEAD * (2 * t + t + 2 * t) + 2 * blocks), "flops": 0}
    keys = sum(a for a, n in zip(kv, new) if n)
    seen = sum(n * (a - n) + n * (n + 1) // 2 for a, n in zip(kv, new))
    return {"bytes": 2 * hk * (keys * HEAD + (keys + BLOCK - 1) // BLOCK) + 4 * sum(new) * case["heads"] * HEAD,
            "flops": 4 * HEAD * case["heads"] * seen}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _pool(g, layers, pages, hk, page):
    """Cache pages as the writer leaves them: codes u = m + 128 of values near N(0, 1), block exponents to match."""
    def codes():
        m = torch.empty((layers, pages, hk, page, HEAD), dtype=torch.uint8, device=DEV)
        for i in range(layers):
            m[i] = (torch.randn(m.shape[1:], generator=g, device=DEV, dtype=torch.float16) * 30 + 128).clamp_(0, 255).to(torch.uint8)
        return m

    def exps():
        e = torch.randint(126, 130, (layers, pages, hk, page // BLOCK), generator=g, device=DEV)
        return e.to(torch.uint8)

    return codes(), codes(), exps(), exps()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "w4":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"] = torch.randn((m, k), generator=g, device=DEV).to(torch.bfloat16)
        s["codes"] = (torch.randn((k, n), generator=g, device=DEV) * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
        sign = torch.randint(0, 2, (k // case["group"], n), generator=g, device=DEV) * 2 - 1
        s["scales"] = (0.009 * sign * (0.8 + 0.4 * torch.rand(sign.shape, generator=g, device=DEV))).to(torch.bfloat16)
        s["bias"] = (torch.randn(n, generator=g, device=DEV) * 0.01).to(torch.bfloat16) if case["bias"] else None
        if own:
            from redline_tiny_b200 import ops
            s["w"] = ops.Weight4.from_codes(s["codes"], s["scales"], swiglu=case["swiglu"])
        return s
    hk, page = case["kv_heads"], case["page"]
    if case["op"] == "copy":
        s["pool"] = _pool(g, case["layers"], case["pages"], hk, page)
        order = torch.randperm(case["pages"], generator=g, device=DEV)[:2 * case["copies"]].sort().values.tolist()
        s["src"], s["dst"] = order[case["copies"]:], order[:case["copies"]]
        s["src_t"], s["dst_t"] = torch.tensor(s["src"], device=DEV), torch.tensor(s["dst"], device=DEV)
    else:
        kv, new = _lengths(case)
        need = [(a + page - 1) // page for a in kv]
        width = max(need)
        pages = sum(need) + 3
        s["pool"] = _pool(g, 1, pages, hk, page)
        perm = torch.randperm(pages, generator=g, device=DEV).tolist()
        rows, at = [], 0
        for n in need:
            rows.append(perm[at:at + n] + [-1] * (width - n))
            at += n
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device=DEV)
        s["table"], s["kv_len"] = torch.tensor(rows, **i32), torch.tensor(kv, **i32)
        s["q_start"] = torch.tensor(starts, **i32)
        s["kv_max"], s["new_max"] = max(kv), max(new)
        t = starts[-1]
        if case["op"] == "append":
            s["k"] = torch.randn((t, hk, HEAD), generator=g, device=DEV).to(torch.bfloat16)
            s["v"] = (torch.randn((t, hk, HEAD), generator=g, device=DEV) * 1.5).to(torch.bfloat16)
            # what is read back: the blocks that the new tokens touch
            s["first"] = torch.tensor([(a - n) // BLOCK * BLOCK for a, n in zip(kv, new)], **i32)
            s["count"] = max(a - (a - n) // BLOCK * BLOCK for a, n in zip(kv, new))
        else:
            s["q"] = torch.randn((t, case["heads"], HEAD), generator=g, device=DEV).to(torch.bfloat16)
    if own:
        from redline_tiny_b200 import ops
        s["own_pool"] = ops.KVPool(*s["pool"])
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        from redline_tiny_b200 import ops
        if op == "w4":
            f = ops.swiglu_w4 if s["case"]["swiglu"] else ops.linear_w4
            return f(s["x"], s["w"], bias=s["bias"])
        if op == "copy":
            ops.kv_copy_pages(s["own_pool"], s["src"], s["dst"])
            return s["pool"]
        if op == "append":
            ops.kv_append(s["own_pool"], 0, s["k"], s["v"], s["table"], s["kv_len"], s["q_start"])
            return ops.kv_read(s["own_pool"], 0, s["table"], s["kv_len"], s["first"], s["count"])
        return ops.kv_attention(s["q"], s["own_pool"], 0, s["table"], s["kv_len"], s["q_start"])
    if op == "w4":
        return _plain_w4(s)
    if op == "copy":
        k, v, ke, ve = s["pool"]
        k[:, s["dst_t"]] = k[:, s["src_t"]]
        v[:, s["dst_t"]] = v[:, s["src_t"]]
        ke[:, s["dst_t"]] = ke[:, s["src_t"]]
        ve[:, s["dst_t"]] = ve[:, s["src_t"]]
        return s["pool"]
    if op == "append":
        k, v, ke, ve = s["pool"]
        _plain_append(s, s["k"], k[0], ke[0])
        _plain_append(s, s["v"], v[0], ve[0])
        return _plain_read(s, k[0], ke[0]), _plain_read(s, v[0], ve[0])
    return _plain_attention(s)


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------
def _plain_w4(s):
    x, case = s["x"].float(), s["case"]
    k, n = s["codes"].shape
    w = (s["codes"].view(k // case["group"], case["group"], n).float() - 8.0) * s["scales"].float()[:, None, :]
    c = x @ w.view(k, n)
    if s["bias"] is not None:
        c = c + s["bias"].float()
    if case["swiglu"]:
        gate, up = c.view(-1, n // 128, 2, 64).unbind(2)     # [gate 64 | up 64] per 128 columns
        c = (gate / (1.0 + torch.exp(-gate)) * up).reshape(-1, n // 2)
    return c.to(torch.bfloat16)


def _scale(e):
    """2^(E - 133) in 64 bits; a block that holds a NaN or an infinity (E = 255) reads as NaN."""
    f = torch.exp2(e.double() - 133.0)
    return torch.where(e == 255, torch.full_like(f, math.nan), f)


def _plain_attention(s):
    k, v, ke, ve = (t[0] for t in s["pool"])
    hk, page, heads = s["case"]["kv_heads"], s["case"]["page"], s["case"]["heads"]
    grp, nb = heads // hk, s["table"].shape[0]
    idx = s["table"].long().clamp(min=0)
    tokens = idx.shape[1] * page

    def dense(codes, exps):
        f = _scale(exps[idx]).float()[..., None, None]                       # (b, pages, hk, blocks, 1, 1)
        c = (codes[idx].float() - 128.0).view(*f.shape[:4], BLOCK, HEAD) * f
        return c.view(nb, -1, hk, page, HEAD).permute(0, 2, 1, 3, 4).reshape(nb, hk, tokens, HEAD)

    starts, lens = s["q_start"].long(), s["kv_len"].long()
    n = starts[1:] - starts[:-1]
    j = torch.arange(s["new_max"], device=DEV)
    row = (starts[:-1, None] + j).clamp(max=max(s["q"].shape[0] - 1, 0))
    q = s["q"][row].float().view(nb, -1, hk, grp, HEAD).permute(0, 2, 3, 1, 4).reshape(nb, hk, -1, HEAD)
    sc = (q @ dense(k, ke).transpose(2, 3)) * SCALE_LOG2
    limit = lens[:, None] - n[:, None] + j                                  # last visible key of each query
    hide = torch.arange(tokens, device=DEV)[None, None, :] > limit[:, :, None]
    sc = sc.view(nb, hk, grp, -1, tokens).masked_fill_(hide[:, None, None], -math.inf)
    sc -= sc.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp2(sc)
    o = p.view(nb, hk, -1, tokens) @ dense(v, ve)
    o = o / p.sum(-1, dtype=torch.float32).clamp(min=1e-30).view(nb, hk, -1, 1)
    o = o.view(nb, hk, grp, -1, HEAD).permute(0, 3, 1, 2, 4).reshape(nb, -1, heads * HEAD)
    return o[j < n[:, None]].to(torch.bfloat16)


def _touched(s, codes):
    """The blocks [first, first + count) of each sequence: positions, page and place in the page, which hold older
    tokens, which new ones, and the row of each new token."""
    nb, page = s["table"].shape[0], codes.shape[2]
    lens, starts = s["kv_len"].long(), s["q_start"].long()
    n = starts[1:] - starts[:-1]
    blocks = (s["count"] + BLOCK - 1) // BLOCK
    pos = s["first"].long()[:, None] + torch.arange(blocks * BLOCK, device=DEV)
    old = pos < (lens - n)[:, None]
    new = (pos >= (lens - n)[:, None]) & (pos < lens[:, None])
    pg = s["table"].long().gather(1, (pos // page).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    row = (starts[:-1, None] + pos - (lens - n)[:, None]).clamp(0, starts.max() - 1)
    return nb, blocks, pos, pg, pos % page, old, new, row


def _plain_append(s, x, codes, exps):
    """Blocks with new tokens take the larger of their exponent and the new tokens' own; older codes are shifted."""
    nb, blocks, pos, pg, at, old, new, row = _touched(s, codes)
    hk = x.shape[1]
    xr = x[row].float()                                                     # (b, tokens, hk, 128)
    field = (xr.view(torch.int32) >> 23 & 255) * new[:, :, None, None]
    need = field.view(nb, blocks, BLOCK, hk, HEAD).amax((2, 4))             # (b, blocks, hk)
    has_old = old.view(nb, blocks, BLOCK).any(2)[:, :, None]
    head_blk = pg.view(nb, blocks, BLOCK)[:, :, 0], at.view(nb, blocks, BLOCK)[:, :, 0] // BLOCK
    e_old = exps[head_blk[0], :, head_blk[1]].long()                        # (b, blocks, hk)
    e = torch.where(has_old, torch.maximum(e_old, need), need)
    each = lambda t: t[:, :, None].expand(-1, -1, BLOCK, -1).reshape(nb, -1, hk)  # noqa: E731
    m_old = codes[pg, :, at].double() - 128.0
    m_old = torch.round(m_old * torch.exp2((each(e_old) - each(e)).double().clamp(max=0))[..., None])
    m_new = torch.round(xr.double() * torch.exp2(133.0 - each(e).double())[..., None]).clamp(-128, 127)
    m = torch.where(new[:, :, None, None], m_new, m_old)
    write = (old | new) & new.view(nb, blocks, BLOCK).any(2).repeat_interleave(BLOCK, 1)
    codes[pg[write], :, at[write]] = (m[write] + 128.0).to(torch.uint8)
    wb = new.view(nb, blocks, BLOCK).any(2)
    exps[head_blk[0][wb], :, head_blk[1][wb]] = e[wb].to(torch.uint8)


def _plain_read(s, codes, exps):
    """bf16 (batch, count, hk, 128): positions first .. first + count - 1 of each sequence, zeros at and after its end."""
    page, hk = codes.shape[2], codes.shape[1]
    pos = s["first"].long()[:, None] + torch.arange(s["count"], device=DEV)
    live = pos < s["kv_len"].long()[:, None]
    pg = s["table"].long().gather(1, (pos // page).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    f = _scale(exps[pg, :, pos % page // BLOCK]).float()
    x = (codes[pg, :, pos % page].float() - 128.0) * f[..., None]
    return torch.where(live[:, :, None, None], x, torch.zeros_like(x)).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "copy":
        return None
    with_own = own
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = with_own
    if case["op"] == "w4":
        g = case["group"]
        c = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device=DEV)
        for i in range(case["k"] // g):
            part = s["x"][:, i * g:(i + 1) * g].double() @ (s["codes"][i * g:(i + 1) * g].double() - 8)
            c += part * s["scales"][i].double()
        if s["bias"] is not None:
            c += s["bias"].double()
        if case["swiglu"]:
            z = c.reshape(case["rows"], -1, 128)
            c = (torch.sigmoid(z[..., :64]) * z[..., :64] * z[..., 64:]).flatten(1)
        return c
    if case["op"] == "append":
        return tuple(_exact_append(s, x, c[0], e[0]) for x, c, e in
                     ((s["k"], s["pool"][0], s["pool"][2]), (s["v"], s["pool"][1], s["pool"][3])))
    k, v, ke, ve = (t[0] for t in s["pool"])
    kv, new = _lengths(case)
    grp = case["heads"] // case["kv_heads"]
    out, at = [], 0
    for b, (a, n) in enumerate(zip(kv, new)):
        if n == 0:
            continue
        kd, vd = (_sequence(s["table"][b], a, c, e) for c, e in ((k, ke), (v, ve)))
        q = s["q"][at:at + n].double()
        at += n
        last = a - n + torch.arange(n, device=DEV)
        hide = torch.arange(a, device=DEV)[None, :] > last[:, None]
        o = torch.empty((n, case["heads"], HEAD), dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            z = (q[:, h] @ kd[:, h // grp].T / math.sqrt(HEAD)).masked_fill(hide, -math.inf)
            o[:, h] = torch.softmax(z, -1) @ vd[:, h // grp]
        out.append(o.view(n, -1))
    return torch.cat(out)


def _sequence(table, length, codes, exps):
    """(length, hk, 128) values of one sequence."""
    page = codes.shape[2]
    rows = table[:(length + page - 1) // page].long()
    c = codes[rows].double() - 128
    c = c * torch.exp2(exps[rows].double() - 133).repeat_interleave(BLOCK, 2)[..., None]
    return c.permute(0, 2, 1, 3).reshape(-1, codes.shape[1], HEAD)[:length]


def _exact_append(s, x, codes, exps):
    kv, new = _lengths(s["case"])
    out = torch.zeros((len(kv), s["count"], x.shape[1], HEAD), dtype=torch.float64, device=DEV)
    at = 0
    for b, (a, n) in enumerate(zip(kv, new)):
        if n == 0:
            first = a // BLOCK * BLOCK
            out[b, :a - first] = _sequence(s["table"][b], a, codes, exps)[first:]
            continue
        first = (a - n) // BLOCK * BLOCK
        have = _sequence(s["table"][b], a, codes, exps)[first:a - n]          # older tokens of the first block
        fresh = x[at:at + n].double()
        at += n
        for i in range(0, a - first, BLOCK):
            z = fresh[max(0, first + i - (a - n)):first + i + BLOCK - (a - n)]
            h = have if i == 0 else have[:0]
            top = torch.frexp(z.abs().amax((0, 2)))[1].double() + 126          # exponent field of the largest new value
            if len(h):
                pg, bl = int(s["table"][b, (first + i) // codes.shape[2]]), (first + i) % codes.shape[2] // BLOCK
                top = torch.maximum(top, exps[pg, :, bl].double())
            step = torch.exp2(top - 133)[None, :, None]
            m = torch.cat([torch.round(h / step), torch.clamp(torch.round(z / step), -128, 127)])
            out[b, i:i + len(m)] = m * step
    return out
