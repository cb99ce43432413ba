"""What the writer of the paged cache does with row ranges and lengths that no sequence can have."""

import pytest

from test_gpu_kv_cache import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from redline_tiny_b200 import _lib, ops
    assert torch.cuda.is_available()
    return torch, ops, _lib, torch.device("cuda:0")


def test_row_ranges_that_fall_are_reported_by_the_writer(env):
    """A sequence whose rows end before they begin is reported by kv_append as it is by kv_attention; so is one that writes
    nothing but has an impossible length."""
    torch, ops, L, dev = env
    c = Case(torch, ops, dev, [40, 30, 50], [2, 3, 1], 2, 16)
    x = torch.ones((c.T, 2, 128), dtype=torch.bfloat16, device=dev)
    for kv_len, start in (([40, 30, 50], [0, 5, 3, 6]), ([40, 30, 50], [3, 2, 4, 6]), ([40, -1, 50], [0, 2, 2, 3]),
                          ([40, 30, 5000], [0, 2, 5, 5])):
        lens, st = (torch.tensor(a, dtype=torch.int32, device=dev) for a in (kv_len, start))
        ops.kv_append(c.pool, 0, x, x, c.d_table, lens, st)
        with pytest.raises(L.RedlineError, match="range check"):
            ops.device_status()
    ops.kv_append(c.pool, 0, x, x, c.d_table, c.d_len, c.d_start)
    ops.device_status()
