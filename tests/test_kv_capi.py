"""CPU-side refusals of the cache and 4-bit entry points: bad arguments give a status and a message before any device
is touched (no kernel is launched here)."""

import ctypes

import pytest

from redline_tiny_b200 import _lib as L


@pytest.fixture(scope="module")
def lib():
    from redline_tiny_b200 import build
    build.build()
    return L.lib()


BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(BUF) + 255) // 256 * 256      # an aligned host address; never read


def refused(lib, name, args, status, text):
    assert getattr(lib, name)(*args) == status
    assert text in lib.rl_last_error()


def append_args(**k):
    a = dict(k=P, st=128, sh=128, sd=1, dtype=L.RL_BF16, T=1, pool=P, ke=P, pages=4, hkv=1, page=16, table=P, ld=2,
             kv_len=P, q_start=P, B=1)
    a.update(k)
    return (a["k"], a["st"], a["sh"], a["sd"], P, 128, 128, 1, a["dtype"], a["T"], a["pool"], P, a["ke"], P, a["pages"],
            a["hkv"], a["page"], a["table"], a["ld"], a["kv_len"], a["q_start"], a["B"], None)


@pytest.mark.parametrize("change,status,text", [
    (dict(pool=None), -1, b"NULL pool"), (dict(page=48), -1, b"page size"), (dict(pages=0), -1, b"pages"),
    (dict(hkv=0), -1, b"kv_heads"), (dict(pool=P + 1), -2, b"aligned"), (dict(table=None), -1, b"table"),
    (dict(B=1025), -1, b"sequences"), (dict(ld=0), -1, b"table"), (dict(T=-1), -1, b"rows"), (dict(dtype=7), -1, b"dtype"),
    (dict(k=None), -1, b"NULL"), (dict(k=P + 1), -2, b"aligned"), (dict(table=P + 2), -2, b"int32"),
])
def test_append(lib, change, status, text):
    refused(lib, "rl_kv_append", append_args(**change), status, text)


def attention_args(**k):
    a = dict(q=P, q_st=128, q_sh=128, T=1, heads=2, hkv=1, page=16, ld=2, B=1, o=P, ldo=256, ws=P, nbytes=1 << 40)
    a.update(k)
    return (a["q"], a["q_st"], a["q_sh"], a["T"], a["heads"], P, P, P, P, 4, a["hkv"], a["page"], P, a["ld"], P, P, a["B"],
            None, 1.0, a["o"], a["ldo"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("change,status,text", [
    (dict(heads=3, hkv=2), -1, b"heads"), (dict(heads=0), -1, b"heads"), (dict(q=None), -1, b"NULL"),
    (dict(q=P + 2), -2, b"aligned"), (dict(q_st=132), -2, b"strides"), (dict(ldo=255), -1, b"ldo"),
    (dict(ws=None), -1, b"workspace"), (dict(nbytes=16), -1, b"workspace"), (dict(ws=P + 4), -2, b"workspace"),
    (dict(ld=1 << 24, page=256), -1, b"tokens"),
])
def test_attention(lib, change, status, text):
    refused(lib, "rl_kv_attention", attention_args(**change), status, text)


def test_read(lib):
    def args(count=4, start=P, out=P):
        return (P, P, P, P, 4, 1, 16, P, 2, P, start, 1, count, out, P, None)
    refused(lib, "rl_kv_read", args(count=-1), -1, b"count")
    refused(lib, "rl_kv_read", args(start=None), -1, b"NULL")
    refused(lib, "rl_kv_read", args(out=P + 8), -2, b"aligned")


@pytest.mark.parametrize("src,dst,i", [([4], [0], 0), ([0], [-1], 0), ([0, 1], [2, 2], 1), ([0, 2], [2, 3], 1),
                                       ([1, 2], [3, 2], 1)])
def test_copy_pages(lib, src, dst, i):
    """Pages outside the pool, two copies into one page, a page that one copy reads and another writes."""
    n = len(src)
    a, b = (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst)
    refused(lib, "rl_kv_copy_pages", (P, P, P, P, 1, 4, 1, 16, a, b, n, None), -1, f"copy {i} ".encode())


def test_copy_pages_counts(lib):
    a = (ctypes.c_int32 * 1)(0)
    refused(lib, "rl_kv_copy_pages", (P, P, P, P, 1, 4, 1, 16, a, a, 5, None), -1, b"copies")
    refused(lib, "rl_kv_copy_pages", (P, P, P, P, 0, 4, 1, 16, a, a, 1, None), -1, b"layers")
    assert lib.rl_kv_copy_pages(P, P, P, P, 1, 4, 1, 16, None, None, 0, None) == 0


@pytest.mark.parametrize("M,K,group,N,epi,text", [
    (65, 64, 32, 16, 0, b"rows"), (1, 48, 32, 16, 0, b"multiple"), (1, 64, 16, 16, 0, b"groups"),
    (1, 64, 32, 0, 0, b"N = 0"), (1, 64, 32, 192, 2, b"128"), (1, 64, 32, 16, 1, b"bias"), (1, 64, 32, 16, 9, b"epilogue"),
])
def test_linear_w4(lib, M, K, group, N, epi, text):
    refused(lib, "rl_linear_w4", (P, M, K, P, P, N, group, None, epi, P, 1, None), -1, text)


def test_w4_sizes(lib):
    cb, sb = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.rl_w4_bytes(160, 33, 32, 0, ctypes.byref(cb), ctypes.byref(sb)) == 0
    assert (cb.value, sb.value) == (3 * 2 * 1024, 3 * 8 * 16 * 2)     # N padded to 48, K to 256
    refused(lib, "rl_w4_bytes", (160, 33, 64, 0, ctypes.byref(cb), ctypes.byref(sb)), -1, b"multiple")
    refused(lib, "rl_linear_w4", (P + 2, 1, 64, P, P, 16, 32, None, 0, P, 1, None), -2, b"aligned")


def test_host_tensors_are_refused():
    """The Python layer turns down tensors in host memory before their addresses reach a kernel, whichever argument they
    are, and tells a wrong type or shape from them."""
    torch = pytest.importorskip("torch")
    from redline_tiny_b200 import ops
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8

    class OnDevice:   # a tensor that claims to lie on a device
        def __init__(self, *shape, dtype=bf):
            self.t = torch.zeros(shape, dtype=dtype)

        def get_device(self):
            return 0

        def __getattr__(self, name):
            return getattr(self.t, name)

    codes, exps = torch.full((1, 4, 2, 16, 128), 128, dtype=u8), torch.zeros((1, 4, 2, 1), dtype=u8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVPool(codes, codes, exps, exps)
    pool = ops.KVPool.__new__(ops.KVPool)
    pool.k, pool.layers, pool.pages, pool.kv_heads, pool.page, pool._ptrs = codes, 1, 4, 2, 16, [(0, 0, 0, 0)]
    table, lens, start = torch.zeros((1, 2), dtype=i32), torch.ones(1, dtype=i32), torch.zeros(2, dtype=i32)
    kv, q = torch.zeros((1, 2, 128), dtype=bf), torch.zeros((1, 4, 128), dtype=bf)
    w = ops.Weight4(torch.zeros(1024, dtype=u8), torch.zeros(64, dtype=u8), 32, 16, 32)
    calls = [lambda: ops.kv_append(pool, 0, kv, kv, table, lens, start), lambda: ops.kv_read(pool, 0, table, lens, lens, 1),
             lambda: ops.kv_attention(q, pool, 0, table, lens, start), lambda: ops.kv_copy_pages(pool, [0], [1]),
             lambda: ops.kv_set(table, {0: 1}), lambda: ops.linear_w4(torch.zeros((1, 32), dtype=bf), w),
             lambda: ops.quantize_w4(torch.zeros((32, 16)), 32),
             lambda: ops.Weight4.from_codes(torch.zeros((32, 16), dtype=u8), torch.zeros((1, 16), dtype=bf))]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()
    # one host tensor among device tensors, in each place
    if torch.cuda.is_available():
        return
    try:
        torch._C._cuda_getDevice()
    except Exception:
        real, torch._C._cuda_getDevice = torch._C._cuda_getDevice, lambda: 0
    else:
        real = None
    try:
        good = [OnDevice(1, 2, 128), OnDevice(1, 2, 128), OnDevice(1, 2, dtype=i32), OnDevice(1, dtype=i32), OnDevice(2, dtype=i32)]
        pool.k = OnDevice(1, 4, 2, 16, 128, dtype=u8)
        for i in range(5):
            args = list(good)
            args[i] = good[i].t
            with pytest.raises(ValueError, match="CUDA"):
                ops.kv_append(pool, 0, *args)
        with pytest.raises(ValueError, match="current device"):
            class Elsewhere(OnDevice):
                def get_device(self):
                    return 1
            ops.kv_append(pool, 0, Elsewhere(1, 2, 128), *good[1:])
    finally:
        if real is not None:
            torch._C._cuda_getDevice = real
