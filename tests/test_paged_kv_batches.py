"""cache.Batch on the CPU where the books move under it: page tables that went stale are not handed out, and a step that
fails leaves the books as they were."""

import pytest

torch = pytest.importorskip("torch")

from redline_tiny_b200 import cache, ops  # noqa: E402
from test_paged_kv import PAGE, append, fake, read  # noqa: E402, F401


def cached(tokens, pages=12):
    """A cache with one sequence of `tokens` tokens and the batch that wrote it."""
    kv = cache.PagedKV(1, pages, 1, PAGE, "cpu")
    a = kv.new()
    batch = kv.batch([a])
    batch.extend([tokens])
    append(kv, batch, list(range(tokens)))
    return kv, a, batch


def refused(batch):
    with pytest.raises(RuntimeError, match="moved since this batch's last extend"):
        batch.args


def test_tables_after_a_copy_on_write_elsewhere(fake):  # noqa: F811
    """Two batches hold a sequence whose tail is shared: when one of them takes a private tail, the other may not write into
    the tail that now belongs to the fork."""
    kv, a, batch = cached(PAGE + 3)
    fork = kv.fork(a)
    batch.args                                        # a fork moves nothing
    other = kv.batch([a])
    other.extend([1])
    append(kv, other, [100])
    assert kv.pages(a)[1] != kv.pages(fork)[1]
    refused(batch)
    batch.extend([1])
    append(kv, batch, [101])
    assert read(kv, a) == list(range(PAGE + 3)) + [100, 101] and read(kv, fork) == list(range(PAGE + 3))
    refused(other)


def test_tables_after_truncate_and_free(fake):  # noqa: F811
    """Pages that were given up belong to whoever takes them next."""
    kv, a, batch = cached(2 * PAGE)
    b = kv.new()
    step = kv.batch([a, b])
    step.extend([0, 5])
    append(kv, step, list(range(5)))
    kv.truncate(a, 2 * PAGE)                          # no change
    batch.args, step.args
    kv.truncate(a, 3)
    refused(batch)
    refused(step)
    step.extend([0, 0])
    step.args
    batch.extend([2])
    append(kv, batch, [50, 51])
    refused(step)
    kv.free(a)
    refused(batch)
    taken = kv.new()
    kv.batch([taken]).extend([3 * PAGE])
    refused(batch)
    assert read(kv, b) == list(range(5))


def test_other_sequences_do_not_matter(fake):  # noqa: F811
    kv, a, batch = cached(PAGE)
    b = kv.new()
    other = kv.batch([b])
    other.extend([PAGE + 1])
    kv.truncate(b, 1)
    c = kv.fork(a)
    kv.free(c)
    kv.free(b)
    table, lens, _ = batch.args
    assert table[0, 0] == kv.pages(a)[0] and lens.tolist() == [PAGE]
    assert kv.compact() == 0
    batch.args


@pytest.mark.parametrize("call", ["kv_copy_pages", "kv_set"])
def test_a_step_whose_device_calls_fail(fake, monkeypatch, call):  # noqa: F811
    """No page is taken and no tail moved; the same step then succeeds, with tables that are right from end to end."""
    kv, a, batch = cached(PAGE + 3)
    fork = kv.fork(a)
    step = kv.batch([fork, a])
    step.extend([0, 0])
    state = lambda: (kv.refs[:], sorted(kv._free), {s: (kv.pages(s), kv.length(s)) for s in (a, fork)})  # noqa: E731
    before = state()
    real = getattr(ops, call)

    def partly(*args):
        if call == "kv_set":
            real(args[0], dict(list(args[1].items())[:2]))       # some entries are written before the failure
        raise RuntimeError("no device")
    monkeypatch.setattr(ops, call, partly)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no device"):
            step.extend([PAGE, 1])
        assert state() == before
    monkeypatch.setattr(ops, call, real)
    batch.args                                                   # the books did not move
    if call == "kv_set":
        refused(step)
    step.extend([PAGE, 1])
    append(kv, step, list(range(200, 200 + PAGE + 1)))
    assert read(kv, fork) == list(range(PAGE + 3)) + list(range(200, 200 + PAGE))
    assert read(kv, a) == list(range(PAGE + 3)) + [200 + PAGE]
    table, lens, starts = (t.tolist() for t in step.args)
    for row, s in zip(table, (fork, a)):
        assert row[:len(kv.pages(s))] == list(kv.pages(s))
    assert lens == [kv.length(fork), kv.length(a)] and starts == [0, PAGE, PAGE + 1] and step.rows == PAGE + 1


def test_batches_that_no_kernel_takes(fake):  # noqa: F811
    """More sequences, or tables for more tokens, than a kernel takes: refused when the batch is made, before any extend."""
    kv = cache.PagedKV(1, 4, 1, PAGE, "cpu")
    seqs = [kv.new() for _ in range(1025)]
    with pytest.raises(ValueError, match="1025 sequences"):
        kv.batch(seqs)
    assert len(kv.batch(seqs[1:], max_pages=1).seqs) == 1024
    for pages in (-1, (1 << 26) + 1):
        with pytest.raises(ValueError, match="pages a sequence"):
            kv.batch(seqs[:1], max_pages=pages)
    assert kv.batch(seqs[:1]).width == 4
