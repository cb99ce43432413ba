"""The bookkeeping of cache.PagedKV and cache.Batch on the CPU: the device calls are replaced by a model of the pages'
contents (a page is a list of tokens), so that every sequence can be read back after any run of new, fork, extend,
truncate, free, compact and resize."""

import random

import pytest

torch = pytest.importorskip("torch")

from redline_tiny_b200 import cache, ops  # noqa: E402

PAGE = 16


class FakePool:
    def __init__(self, layers, pages, kv_heads, page, device):
        self.layers, self.kv_heads, self.page = layers, kv_heads, page
        self.k = self.v = self.k_exp = self.v_exp = torch.zeros((layers, pages), dtype=torch.uint8)
        self.tokens = [[None] * page for _ in range(pages)]


@pytest.fixture
def fake(monkeypatch):
    def copy(pool, src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for a, b in zip(src, dst):
            pool.tokens[b] = list(pool.tokens[a])

    def write(t, entries):
        for i, v in entries.items():
            t.view(-1)[i] = v
    monkeypatch.setattr(ops.KVPool, "empty", classmethod(lambda cls, *a: FakePool(*a)))
    monkeypatch.setattr(ops, "kv_copy_pages", copy)
    monkeypatch.setattr(ops, "kv_set", write)


def append(kv, batch, rows):
    """What kv_append does: row j of n goes to position kv_len - n + j of its sequence's table."""
    table, lens, start = (t.tolist() for t in batch.args)
    assert start[-1] == len(rows)
    for b in range(len(batch.seqs)):
        n = start[b + 1] - start[b]
        for j in range(n):
            pos = lens[b] - n + j
            kv.pool.tokens[table[b][pos // PAGE]][pos % PAGE] = rows[start[b] + j]


def read(kv, seq):
    return [kv.pool.tokens[kv.pages(seq)[i // PAGE]][i % PAGE] for i in range(kv.length(seq))]


def check(kv, model):
    refs = [0] * len(kv.refs)
    for s, tokens in model.items():
        assert kv.length(s) == len(tokens) and len(kv.pages(s)) == -(-len(tokens) // PAGE)
        assert read(kv, s) == tokens
        for p in kv.pages(s):
            refs[p] += 1
    assert refs == kv.refs and kv.free_pages == refs.count(0) and sorted(kv._free) == [p for p, r in enumerate(refs) if not r]


@pytest.mark.parametrize("seed", range(12))
def test_random_runs(fake, seed):
    rng = random.Random(seed)
    kv = cache.PagedKV(2, 40, 1, PAGE, "cpu")
    model, stamp = {}, 0
    for _ in range(300):
        act = rng.choice(["new", "fork", "extend", "extend", "extend", "truncate", "free", "compact", "resize"])
        if act == "new" and len(model) < 8:
            model[kv.new()] = []
        elif act == "fork" and model and len(model) < 8:
            s = rng.choice(list(model))
            model[kv.fork(s)] = list(model[s])
        elif act == "extend" and model:
            seqs = rng.sample(list(model), rng.randint(1, len(model)))
            counts = [rng.choice([0, 1, 1, 1, rng.randint(0, 40)]) for _ in seqs]
            batch = kv.batch(seqs, max_pages=64)
            before = kv.refs[:], {s: kv.pages(s) for s in model}, kv.free_pages
            try:
                batch.extend(counts)
            except cache.OutOfPages:
                assert before == (kv.refs[:], {s: kv.pages(s) for s in model}, kv.free_pages)
                continue
            rows = list(range(stamp, stamp + sum(counts)))
            stamp += len(rows)
            append(kv, batch, rows)
            for s, n in zip(seqs, counts):
                model[s] += rows[:n]
                rows = rows[n:]
        elif act == "truncate" and model:
            s = rng.choice(list(model))
            n = rng.randint(0, len(model[s]))
            kv.truncate(s, n)
            del model[s][n:]
        elif act == "free" and model:
            s = rng.choice(list(model))
            kv.free(s)
            del model[s]
        elif act == "compact":
            live = sum(1 for r in kv.refs if r)
            kv.compact()
            assert all(p < live for s in model for p in kv.pages(s))
        elif act == "resize":
            live = sum(1 for r in kv.refs if r)
            tokens = kv.pool.tokens
            pages = rng.randint(max(live, 1), 60)
            shrink = pages < len(kv.refs)
            kv.resize(pages)
            # (the fake pool's contents move with the arrays)
            kv.pool.tokens = (tokens + [[None] * PAGE for _ in range(pages)])[:pages] if not shrink else tokens[:pages]
        check(kv, model)


def test_a_step_of_forks_copies_the_shared_page_once_too_few(fake):
    """The last holder of a shared page writes into it; the others get copies."""
    kv = cache.PagedKV(1, 8, 1, PAGE, "cpu")
    a = kv.new()
    batch = kv.batch([a])
    batch.extend([PAGE + 3])
    append(kv, batch, list(range(PAGE + 3)))
    b, c = kv.fork(a), kv.fork(a)
    assert kv.free_pages == 6 and kv.refs[kv.pages(a)[1]] == 3
    step = kv.batch([a, b, c])
    step.extend([1, 1, 1])
    append(kv, step, [100, 101, 102])
    assert kv.free_pages == 4 and len({kv.pages(s)[1] for s in (a, b, c)}) == 3
    assert [read(kv, s)[-1] for s in (a, b, c)] == [100, 101, 102]
    assert all(read(kv, s)[:-1] == list(range(PAGE + 3)) for s in (a, b, c))


def test_batches_keep_their_addresses(fake):
    kv = cache.PagedKV(1, 8, 1, PAGE, "cpu")
    s = [kv.new(), kv.new()]
    batch = kv.batch(s, max_pages=3)
    ptrs = [t.data_ptr() for t in batch.args]
    for n in ([5, 1], [0, 1], [12, 30]):
        batch.extend(n)
        assert [t.data_ptr() for t in batch.args] == ptrs
        assert batch.q_start.tolist() == [0, n[0], sum(n)]
    assert batch.kv_len.tolist() == [17, 32] and batch.table.shape == (2, 3)


def test_refusals(fake):
    kv = cache.PagedKV(1, 4, 1, PAGE, "cpu")
    a, b = kv.new(), kv.new()
    with pytest.raises(ValueError, match="twice"):
        kv.batch([a, a])
    with pytest.raises(ValueError, match="no sequence"):
        kv.batch([99])
    batch = kv.batch([a, b], max_pages=2)
    with pytest.raises(ValueError, match="counts"):
        batch.extend([1])
    with pytest.raises(ValueError, match="pages a sequence"):
        batch.extend([2 * PAGE + 1, 0])
    with pytest.raises(ValueError, match="new tokens"):
        batch.extend([-1, 0])
    batch.extend([2 * PAGE, PAGE])
    with pytest.raises(cache.OutOfPages):
        kv.batch([kv.new()]).extend([PAGE + 1])
    with pytest.raises(ValueError, match="tokens"):
        kv.truncate(a, 3 * PAGE)
    kv.free(a)
    for call in (lambda: kv.free(a), lambda: kv.fork(a), lambda: kv.truncate(a, 0)):
        with pytest.raises(ValueError, match="no sequence"):
            call()
    with pytest.raises(ValueError, match="no sequence"):
        batch.extend([1, 1])
    with pytest.raises(cache.OutOfPages, match="in use"):
        kv.resize(0)


def test_a_compacted_cache_asks_for_an_extend(fake):
    """Page tables written before pages moved are not handed out."""
    kv = cache.PagedKV(1, 8, 1, PAGE, "cpu")
    a, b = kv.new(), kv.new()
    batch = kv.batch([a, b])
    batch.extend([PAGE, 2 * PAGE])
    assert batch.rows == 3 * PAGE
    only = kv.batch([b])
    only.extend([1])
    kv.free(a)
    assert kv.compact() == 1
    with pytest.raises(RuntimeError, match="moved"):
        only.args
    only.extend([0])
    assert only.table[0, :3].tolist() == list(kv.pages(b)) and sorted(kv.pages(b)) == [0, 1, 2]
    assert only.rows == 0 and kv.compact() == 0
    only.args
