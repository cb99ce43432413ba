"""Row-major PyTorch-facing API of the bfp16 hot path (torch CUDA tensors in, torch CUDA tensors out).

torch provides device memory and streams only; every computation is a CUDA kernel of libredline_b200.so, called
through its C ABI on the current torch stream.

  quantize_bfp16   npu_layouts.to_bfp16 (+ a_layout)             redline/npu_layouts.py:62-88, 18-23
  dequantize_bfp16 npu_layouts.from_bfp16 (+ a_unlayout)          redline/npu_layouts.py:90-94, 56-60
  pack_b           pack_weights.pack_b                            redline/pack_weights.py:72-79
  PackedWeight     a packed B operand resident on the GPU (native tile order)
  linear_bfp16     gemm() / matmul_vectorized_bfp16 (+ bias)      redline/forward.py:194-197
  swiglu_up        matmul_swiglu_bfp16 (up GEMM + SwiGLU flush)   kernels/atb3/mm_bfp_swiglu.cc:88-168

Continuing sequences token by token (no counterpart in the reference):

  KVPool, kv_append, kv_read, kv_copy_pages, kv_set, kv_attention   the 8-bit paged cache (cache.PagedKV keeps its pages)
  Weight4, linear_w4, swiglu_w4                             products of up to 64 rows with 4-bit weights
"""

import array
import ctypes
import functools
import math

import torch

from . import _lib as L

try:   # the hot calls in one step each (csrc/rl_torch.cpp); None: through ctypes, with the same checks and results
    from . import _rl_torch as _fast
except ImportError:
    _fast = None


def _stream():
    return ctypes_ptr(torch.cuda.current_stream().cuda_stream)


def ctypes_ptr(v):
    return None if v is None else int(v)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_cuda(*ts):
    for t in ts:
        if t is not None:
            if not t.is_cuda:
                raise ValueError("redline_tiny_b200 ops take CUDA tensors (no CPU path)")
            if not t.is_contiguous():
                raise ValueError("tensor must be contiguous")


def _dtype_code(t):
    if t.dtype == torch.float32:
        return L.RL_F32
    if t.dtype == torch.bfloat16:
        return L.RL_BF16
    raise ValueError(f"unsupported dtype {t.dtype}")


_LAYOUTS = {"rowmajor": L.RL_ROWMAJOR, "a_layout": L.RL_A_LAYOUT, "c_atb": L.RL_C_ATB}


def permute_bf16(x, M, K, src="rowmajor", dst="c_atb", out=None):
    """bf16 (M, K) values from one stream order to another (flat tensors for the NPU orders)."""
    _check_cuda(x, out)
    if out is None:
        out = torch.empty(M * K, dtype=torch.bfloat16, device=x.device)
    L.call("rl_permute_bf16", _ptr(x), _LAYOUTS[src], _ptr(out), _LAYOUTS[dst], M, K, _stream())
    return out


def quantize_bfp16(x, layout="rowmajor", want_bytes=True, want_decoded=True):
    """x (M, K) fp32/bf16 -> (bfp16 bytes uint8 [M*K/8*9] in `layout` order or None,
    decoded bf16 (M, K) row-major or None)."""
    _check_cuda(x)
    M, K = x.shape
    q = torch.empty(M * K // 8 * 9, dtype=torch.uint8, device=x.device) if want_bytes else None
    dq = torch.empty((M, K), dtype=torch.bfloat16, device=x.device) if want_decoded else None
    L.call("rl_quantize_bfp16", _ptr(x), _dtype_code(x), M, K, _LAYOUTS[layout], _ptr(q), _ptr(dq), _stream())
    return q, dq


def dequantize_bfp16(q, M, K, layout="rowmajor", dtype=torch.float32):
    _check_cuda(q)
    out = torch.empty((M, K), dtype=dtype, device=q.device)
    L.call("rl_dequantize_bfp16", _ptr(q), _LAYOUTS[layout], M, K, _ptr(out), _dtype_code(out), _stream())
    return out


def pack_b(B):
    """B (K, N) fp32/bf16 -> the reference's packed stream to_bfp16(b_layout(B, 64, 128)) as uint8."""
    _check_cuda(B)
    K, N = B.shape
    out = torch.empty(K * N // 8 * 9, dtype=torch.uint8, device=B.device)
    L.call("rl_pack_b", _ptr(B), _dtype_code(B), K, N, _ptr(out), _stream())
    return out


class PackedWeight:
    """A B operand (K, N) resident on the GPU in the native tile order (1.125 bytes per weight).

    swiglu=True marks an up matrix with [gate 64 | proj 64] per 128 columns (pack_weights.interleave_up); its
    rows are arranged for the fused SwiGLU epilogue."""

    def __init__(self, native, K, N, swiglu=False):
        self.native, self.K, self.N, self.swiglu = native, int(K), int(N), bool(swiglu)

    @classmethod
    def from_pack_b(cls, packed, K, N, swiglu=False):
        """The reference's packed bytes (bNN_*.bin contents, as a CUDA uint8 tensor) -> native tiles."""
        _check_cuda(packed)
        if packed.numel() != K * N // 8 * 9:
            raise ValueError(f"packed stream has {packed.numel()} bytes, expected {K * N // 8 * 9}")
        native = torch.empty_like(packed)
        L.call("rl_weights_from_pack_b", _ptr(packed), K, N, int(swiglu), _ptr(native), _stream())
        return cls(native, K, N, swiglu)

    @classmethod
    def from_float(cls, B, swiglu=False):
        """Float B (K, N) on the GPU -> native tiles (quantised on the device)."""
        _check_cuda(B)
        K, N = B.shape
        native = torch.empty(K * N // 8 * 9, dtype=torch.uint8, device=B.device)
        L.call("rl_pack_weights", _ptr(B), _dtype_code(B), K, N, int(swiglu), _ptr(native), _stream())
        return cls(native, K, N, swiglu)

    def shard(self, rank, world):
        """Columns [n0, n0 + N / world) of this weight as a view of its own bytes (no copy): the N-split standalone
        GEMM's operand on GPU `rank`. Returns (PackedWeight, n0)."""
        n0, cols, off, count = weights_shard(self.K, self.N, rank, world)
        return PackedWeight(self.native.narrow(0, off, count), self.K, cols, self.swiglu), n0


def weights_shard(K, N, rank, world):
    """(n0, n_cols, byte_offset, byte_count) of column shard `rank` of `world` of a packed B (K, N): the same bytes
    in the reference's pack_b stream and in the native tiles (rl_weights_shard)."""
    v = [ctypes.c_int64() for _ in range(4)]
    L.call("rl_weights_shard", int(K), int(N), int(rank), int(world), *[ctypes.byref(x) for x in v])
    return tuple(x.value for x in v)


def gemm_workspace(M, K, N, device, workspace=None, epilogue=L.RL_EPI_NONE):
    """A device workspace for the GEMM's split-K schedule (rl_linear_bfp16_workspace bytes; None when the shape does
    not split). A given workspace that is large enough is reused."""
    need = L.lib().rl_linear_bfp16_workspace(int(M), int(K), int(N), int(epilogue))
    if need == 0:
        return None
    if workspace is not None and workspace.numel() >= need:
        return workspace
    return torch.empty(need, dtype=torch.uint8, device=device)


def linear_bfp16(x_dq, w, bias=None, out=None, out_dtype=torch.bfloat16, workspace=None):
    """C = x_dq @ B (+ bias), x_dq = bf16 (M, K) holding bfp16 values (quantize_bfp16's decoded output). Shapes with
    too few tiles to fill the GPU and a long K run split-K through a workspace (`workspace`, else one from torch's
    allocator)."""
    _check_cuda(x_dq, w.native, bias, out, workspace)
    if x_dq.dtype != torch.bfloat16:
        raise ValueError("x must be bf16 holding bfp16-exact values (quantize_bfp16 decoded output)")
    M, K = x_dq.shape
    if K != w.K:
        raise ValueError(f"K mismatch: x has {K}, weight has {w.K}")
    if out is None:
        out = torch.empty((M, w.N), dtype=out_dtype, device=x_dq.device)
    epi = L.RL_EPI_BIAS if bias is not None else L.RL_EPI_NONE
    ws = gemm_workspace(M, K, w.N, x_dq.device, workspace, epi)
    L.call("rl_linear_bfp16_ws", _ptr(x_dq), M, K, _ptr(w.native), w.N, _ptr(bias), epi, _ptr(out),
           _dtype_code(out), _ptr(ws), 0 if ws is None else ws.numel(), _stream())
    return out


def swiglu_up(x_dq, w_up, bias=None, out=None):
    """H = silu(x @ Bgate) * (x @ Bproj), rounded to bfp16 blocks of 8 along F and returned as bf16 (M, F): the
    down projection's A operand. w_up must be packed with swiglu=True."""
    _check_cuda(x_dq, w_up.native, bias, out)
    if not w_up.swiglu:
        raise ValueError("swiglu_up needs a PackedWeight packed with swiglu=True")
    M, K = x_dq.shape
    if out is None:
        out = torch.empty((M, w_up.N // 2), dtype=torch.bfloat16, device=x_dq.device)
    L.call("rl_linear_bfp16", _ptr(x_dq), M, K, _ptr(w_up.native), w_up.N, _ptr(bias), L.RL_EPI_SWIGLU,
           _ptr(out), L.RL_BF16, _stream())
    return out


def swiglu_mlp(x, w_up, w_down, out=None, out_dtype=torch.bfloat16, x_quantized=False, workspace=None):
    """out = (silu(x @ Bgate) * (x @ Bproj)) @ Bdown with bfp16 operands (H rounded to bfp16, as the reference's
    fused flush does). x (M, K) bf16/fp32 raw activations (or bf16 bfp16-exact values with x_quantized=True)."""
    _check_cuda(x, w_up.native, w_down.native, out)
    if not w_up.swiglu:
        raise ValueError("w_up must be packed with swiglu=True")
    M, K = x.shape
    F = w_up.N // 2
    if w_down.K != F or w_up.K != K:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, up ({w_up.K}, {w_up.N}), down ({w_down.K}, {w_down.N})")
    if out is None:
        out = torch.empty((M, w_down.N), dtype=out_dtype, device=x.device)
    need = L.lib().rl_swiglu_mlp_workspace(M, K, F, int(x_quantized))
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    L.call("rl_swiglu_mlp", _ptr(x), _dtype_code(x), int(x_quantized), M, K, _ptr(w_up.native), w_up.N,
           _ptr(w_down.native), w_down.N, _ptr(out), _dtype_code(out), _ptr(workspace), workspace.numel(), _stream())
    return out


def ln_mod(x, branch, params, row_split=0, want_x=True, want_y_bytes=False, rms=False):
    """x' = bf16(x + g * branch); y = LayerNorm(x') * sc (rms=True: RMSNorm, vlm_run.rms_ref) rounded to bfp16
    (run_ln.ln_ref). params: bf16 (2, 2, D) = two rows [g | sc] (run_ln.ln_params); rows < row_split use row 1.
    Returns (x' bf16 or None, y decoded bf16, y bfp16 bytes or None)."""
    _check_cuda(x, branch, params)
    M, D = x.shape
    xo = torch.empty_like(x) if want_x else None
    y = torch.empty_like(x)
    yq = torch.empty(M * D // 8 * 9, dtype=torch.uint8, device=x.device) if want_y_bytes else None
    bdt = L.RL_BF16 if branch is None else _dtype_code(branch)
    L.call("rl_rms_mod" if rms else "rl_ln_mod", _ptr(x), _ptr(branch), bdt, _ptr(params), M, D, int(row_split),
           _ptr(xo), _ptr(y), _ptr(yq), _stream())
    return xo, y, yq


def qkv_post(qkv, rope_cs, w_q, w_k, heads, ldv=None, kv_heads=None):
    """QKV GEMM output (M, (H + 2 Hkv) * 128) -> q (H, M, 128), k (Hkv, M, 128) after RMSNorm * w and RoPE;
    vt (Hkv, 128, ldv) = V^T. kv_heads defaults to heads (no grouping)."""
    _check_cuda(qkv, rope_cs, w_q, w_k)
    M = qkv.shape[0]
    hkv = heads if kv_heads is None else int(kv_heads)
    ldv = ldv or (M + 127) // 128 * 128
    q = torch.empty((heads, M, 128), dtype=torch.bfloat16, device=qkv.device)
    k = torch.empty((hkv, M, 128), dtype=torch.bfloat16, device=qkv.device)
    vt = torch.empty((hkv, 128, ldv), dtype=torch.bfloat16, device=qkv.device)
    L.call("rl_qkv_post_gqa", _ptr(qkv), _ptr(rope_cs), _ptr(w_q), _ptr(w_k), M, heads, hkv, _ptr(q), _ptr(k),
           _ptr(vt), ldv, _stream())
    return q, k, vt


def qkv_linear(x_dq, w, rope_cs, w_q, w_k, heads, ldv=None, kv_heads=None):
    """linear_bfp16(x_dq, w) followed by qkv_post in one GEMM launch (the norm and RoPE run in the GEMM's epilogue):
    w = the packed (K, (H + 2 Hkv) * 128) QKV weight. Outputs as qkv_post."""
    _check_cuda(x_dq, w.native, rope_cs, w_q, w_k)
    M, K = x_dq.shape
    hkv = heads if kv_heads is None else int(kv_heads)
    if w.N != (heads + 2 * hkv) * 128:
        raise ValueError(f"qkv_linear: weight has {w.N} columns, heads need {(heads + 2 * hkv) * 128}")
    ldv = ldv or (M + 127) // 128 * 128
    q = torch.empty((heads, M, 128), dtype=torch.bfloat16, device=x_dq.device)
    k = torch.empty((hkv, M, 128), dtype=torch.bfloat16, device=x_dq.device)
    vt = torch.empty((hkv, 128, ldv), dtype=torch.bfloat16, device=x_dq.device)
    L.call("rl_qkv_linear", _ptr(x_dq), M, K, _ptr(w.native), heads, hkv, _ptr(rope_cs), _ptr(w_q), _ptr(w_k),
           _ptr(q), _ptr(k), _ptr(vt), ldv, _stream())
    return q, k, vt


def attention(q, k, vt, nkv=None, row_limit=None, scale_log2=None, out=None, ldo=None, out_dtype=torch.bfloat16):
    """Flash attention per head: q (H, Nq, 128), k (Hkv, Nk, 128), vt (Hkv, 128, ldv) bf16 -> o (Nq, ldo) with
    head h at columns 128h..; bf16 rounded to bfp16 along the head dim (the out-projection's A operand), or with
    out_dtype=torch.float32 the unrounded fp32 O / l. With Hkv < H query head h reads K/V head h / (H / Hkv)
    (grouped-query attention). scale_log2 defaults to log2(e)/sqrt(128)."""
    _check_cuda(q, k, vt, row_limit, out)
    H, Nq, _ = q.shape
    Nk = k.shape[1]
    ldv = vt.shape[2]
    nkv = Nk if nkv is None else int(nkv)
    scale_log2 = math.log2(math.e) / math.sqrt(128) if scale_log2 is None else float(scale_log2)
    ldo = ldo or H * 128
    if out is None:
        out = torch.empty((Nq, ldo), dtype=out_dtype, device=q.device)
    if row_limit is not None and row_limit.dtype != torch.int32:
        raise ValueError("row_limit must be int32")
    fn = "rl_attention_gqa_f32" if out.dtype == torch.float32 else "rl_attention_gqa"
    L.call(fn, _ptr(q), _ptr(k), _ptr(vt), ldv, H, k.shape[0], Nq, Nk, nkv, _ptr(row_limit), scale_log2, _ptr(out),
           ldo, _stream())
    return out


def conv_k(cin, taps):
    """The conv GEMM's K: taps^2 taps of Cin channels, each rounded up to a multiple of 64 (zero rows)."""
    return taps * taps * ((cin + 63) // 64 * 64)


def conv_weight(w, bias=None, cout_pad=128):
    """Conv weight (Cout, Cin, k, k), k = 3 or 1, on the GPU -> (PackedWeight of B = [(dy, dx, ci)][co], bf16 bias or
    None, taps). Each tap's Cin rows are zero-padded to a multiple of 64 (K = conv_k(Cin, k)), Cout to a multiple of
    `cout_pad` (the GEMM's N tile)."""
    _check_cuda(w, bias)
    cout, cin, k, _ = w.shape
    n = (cout + cout_pad - 1) // cout_pad * cout_pad
    kt = conv_k(cin, 1)
    B = torch.zeros((k * k, kt, n), dtype=torch.float32, device=w.device)
    B[:, :cin, :cout] = w.float().permute(2, 3, 1, 0).reshape(k * k, cin, cout)
    B = B.reshape(k * k * kt, n)
    b = None
    if bias is not None:
        b = torch.zeros(n, dtype=torch.bfloat16, device=w.device)
        b[:cout] = bias.to(torch.bfloat16)
    return PackedWeight.from_float(B), b, k


def conv2d(x_dq, w, bias, taps, out=None):
    """VAE conv: x_dq (H, W, Cin) bf16 holding bfp16 values -> (H, W, N) bf16 (N = the padded Cout)."""
    _check_cuda(x_dq, w.native, bias, out)
    H, Wd, C = x_dq.shape
    if w.K != conv_k(C, taps):
        raise ValueError(f"conv weight has K = {w.K}, a {taps}x{taps} conv over {C} channels needs {conv_k(C, taps)}")
    if out is None:
        out = torch.empty((H, Wd, w.N), dtype=torch.bfloat16, device=x_dq.device)
    nbytes = L.lib().rl_conv2d_workspace(H, Wd, C, taps)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x_dq.device)
    L.call("rl_conv2d_bfp16", _ptr(x_dq), H, Wd, C, _ptr(w.native), w.N, taps, _ptr(bias), _ptr(out), _ptr(ws),
           ws.numel(), _stream())
    return out


def _here(*ts):
    """The current device's index, after checking that the tensors (None allowed) lie on it."""
    dev = None
    for t in ts:
        if t is None:
            continue
        d = t.get_device()
        if d != dev:
            if d < 0:
                raise ValueError("redline_tiny_b200 ops take CUDA tensors (no CPU path)")
            dev = torch._C._cuda_getDevice()
            if d != dev:
                raise ValueError(f"tensor on cuda:{d}, but the current device is cuda:{dev}")
    return dev


def _stream_of(dev):
    """The current stream of device `dev` as an integer (torch.cuda.current_stream builds an object first, ~2 us)."""
    return torch._C._cuda_getCurrentRawStream(dev)


def _check_int32(name, t, *shape):
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 of shape {shape}, not {t.dtype} {tuple(t.shape)}")


KV_BLOCK = 16   # tokens of one K/V head that share an exponent
KV_SEQUENCES, KV_TOKENS = 1024, 1 << 30   # the most that a call takes, and that a sequence's page table spans


class KVPool:
    """The pages of an 8-bit cache: k, v uint8 (layers, pages, kv_heads, page, 128) and k_exp, v_exp uint8
    (layers, pages, kv_heads, page / 16). A block of 16 tokens of one head shares one exponent:
    value = (k - 128) * 2^(k_exp - 133); exponent 255 reads as NaN."""

    _fast = ()   # per layer: what _rl_torch takes for it

    def __init__(self, k, v, k_exp, v_exp):
        _here(k, v, k_exp, v_exp)
        if k.dim() != 5 or k.shape[4] != 128 or k.shape[3] not in (16, 32, 64, 128, 256):
            raise ValueError("cache codes must be (layers, pages, kv_heads, page, 128), page = 16, 32, 64, 128 or 256")
        exps = (*k.shape[:3], k.shape[3] // KV_BLOCK)
        for t, shape in ((k, k.shape), (v, k.shape), (k_exp, exps), (v_exp, exps)):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.shape != shape:
                raise ValueError(f"cache tensors must be contiguous uint8; expected {tuple(shape)}, got {tuple(t.shape)}")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.layers, self.pages, self.kv_heads, self.page = k.shape[:4]
        self._ptrs = [tuple(t[i].data_ptr() for t in (k, v, k_exp, v_exp)) for i in range(self.layers)]
        self._fast = [(*self._args(i), k.get_device()) for i in range(self.layers)]

    @classmethod
    def empty(cls, layers, pages, kv_heads, page=64, device="cuda"):
        codes = (layers, pages, kv_heads, page, 128)
        exps = (layers, pages, kv_heads, page // KV_BLOCK)
        return cls(*[torch.full(s, f, dtype=torch.uint8, device=device) for s, f in
                     ((codes, 128), (codes, 128), (exps, 0), (exps, 0))])

    def _args(self, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of a cache with {self.layers}")
        return (*self._ptrs[layer], self.pages, self.kv_heads, self.page)


def _batch(table, kv_len, starts, extra):
    """Sequences and page table width of a batch's int32 arrays."""
    if table.dim() != 2 or table.shape[1] == 0:
        raise ValueError("table must be int32 (sequences, pages)")
    B, width = table.shape
    i32 = torch.int32
    if not (table.dtype is i32 and kv_len.dtype is i32 and starts.dtype is i32 and table.is_contiguous()
            and kv_len.is_contiguous() and starts.is_contiguous() and kv_len.shape == (B,)
            and starts.shape == (B + extra,)):
        _check_int32("table", table, B, width)
        _check_int32("kv_len", kv_len, B)
        _check_int32("q_start" if extra else "start", starts, B + extra)
    return B, width


def kv_append(pool, layer, k, v, table, kv_len, q_start):
    """Write the keys and values of new tokens, k, v (T, kv_heads, 128) bf16 or fp32 of any strides, into a layer of the
    cache. table int32 (B, pages), kv_len int32 (B) with the new tokens counted, q_start int32 (B + 1): the new tokens
    of sequence b are rows q_start[b] .. q_start[b + 1] - 1 and take its last positions. A block's exponent grows to
    hold them, and older codes of the block are shifted. The pages written must belong to one sequence each."""
    if _fast is not None and 0 <= layer < len(pool._fast):
        st = _fast.kv_append(pool._fast[layer], k, v, table, kv_len, q_start)
        if st is not None:
            return L.check("rl_kv_append", st)
    dev = _here(pool.k, k, v, table, kv_len, q_start)
    B, width = _batch(table, kv_len, q_start, 1)
    T = k.shape[0]
    if k.shape != (T, pool.kv_heads, 128) or k.shape != v.shape or k.dtype is not v.dtype:
        raise ValueError(f"k and v must be (rows, {pool.kv_heads}, 128) of one dtype")
    L.call("rl_kv_append", k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), _dtype_code(k), T, *pool._args(layer),
           table.data_ptr(), width, kv_len.data_ptr(), q_start.data_ptr(), B, _stream_of(dev))


def kv_read(pool, layer, table, kv_len, start, count):
    """Positions start[b] .. start[b] + count - 1 of each sequence of a layer as (k, v) bf16 (B, count, kv_heads, 128),
    exactly; zeros at and after kv_len[b]."""
    if _fast is not None and 0 <= layer < len(pool._fast):
        out = _fast.kv_read(pool._fast[layer], table, kv_len, start, count)
        if out is not None:
            return out if type(out) is tuple else L.check("rl_kv_read", out)
    dev = _here(pool.k, table, kv_len, start)
    B, width = _batch(table, kv_len, start, 0)
    kv = torch.empty((2, B, count, pool.kv_heads, 128), dtype=torch.bfloat16, device=pool.k.device)
    k, v = kv.unbind(0)
    L.call("rl_kv_read", *pool._args(layer), table.data_ptr(), width, kv_len.data_ptr(), start.data_ptr(), B, count,
           k.data_ptr(), v.data_ptr(), _stream_of(dev))
    return k, v


def kv_copy_pages(pool, src, dst):
    """Copy page src[i] to page dst[i] in every layer (src, dst: sequences of ints on the host). The copies run at once:
    a page that is written is neither read nor written by another copy of the call."""
    dev = _here(pool.k)
    a, b = array.array("i", src), array.array("i", dst)
    if len(a) != len(b):
        raise ValueError(f"{len(a)} source pages for {len(b)} destinations")
    L.call("rl_kv_copy_pages", *pool._ptrs[0], pool.layers, pool.pages, pool.kv_heads, pool.page, a.buffer_info()[0],
           b.buffer_info()[0], len(a), _stream_of(dev))


def kv_set(t, entries):
    """t.view(-1)[i] = value for the items of `entries` (a dict on the host) of a contiguous int32 tensor, in stream
    order, without a copy from host memory."""
    dev = _here(t)
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise ValueError("kv_set takes a contiguous int32 tensor")
    at, value = array.array("i", entries.keys()), array.array("i", entries.values())
    L.call("rl_kv_set", t.data_ptr(), t.numel(), at.buffer_info()[0], value.buffer_info()[0], len(at), _stream_of(dev))


@functools.lru_cache(maxsize=4096)
def _kv_attention_workspace(dev, T, B, heads, kv_heads):
    return max(L.lib().rl_kv_attention_workspace(T, B, heads, kv_heads), 16)


def kv_attention(q, pool, layer, table, kv_len, q_start, row_limit=None, scale_log2=None, out=None):
    """Attention of new tokens q (T, heads, 128) bf16 (any row and head strides that are multiples of 8) over a layer of
    the cache, which holds their own keys already (kv_append). Row j of sequence b's n new rows sees positions
    <= kv_len[b] - n + j, or <= min(row_limit[row], kv_len[b] - 1) with row_limit int32 (T); a row that sees no key gives
    zeros; a row of no sequence is left as it was in `out`, and without `out` holds whatever its memory held. Returns bf16
    (T, heads * 128); `out` must not overlap q. Contexts of up to 6144 tokens are fastest with a table no wider than that (the
    kernel is chosen by shapes alone). scale_log2 defaults to log2(e)/sqrt(128)."""
    scale = _SCALE_LOG2 if scale_log2 is None else float(scale_log2)
    if _fast is not None and 0 <= layer < len(pool._fast):
        o = _fast.kv_attention(q, pool._fast[layer], table, kv_len, q_start, row_limit, scale, out)
        if o is not None:
            return o if type(o) is not int else L.check("rl_kv_attention", o)
    dev = _here(q, pool.k, table, kv_len, q_start, row_limit, out)
    B, width = _batch(table, kv_len, q_start, 1)
    if q.dim() != 3 or q.dtype is not torch.bfloat16:
        raise ValueError("q must be bf16 (rows, heads, 128)")
    T, H, D = q.shape
    st, sh, sd = q.stride()
    if D != 128 or sd != 1:
        raise ValueError("q must be (rows, heads, 128) with contiguous head vectors")
    if row_limit is not None:
        _check_int32("row_limit", row_limit, T)
    if out is None:
        out = q.new_empty((T, H * 128))
    elif out.dtype is not torch.bfloat16 or out.shape != (T, H * 128) or out.stride(1) != 1:
        raise ValueError(f"out must be bf16 ({T}, {H * 128}) with contiguous rows")
    if T == 1:
        st = 0   # a single row's stride says nothing
    if H == 1:
        sh = 0
    ldo = H * 128 if T == 1 else out.stride(0)
    ws = pool.k.new_empty(_kv_attention_workspace(dev, T, B, H, pool.kv_heads))
    L.call("rl_kv_attention", q.data_ptr(), st, sh, T, H, *pool._args(layer), table.data_ptr(), width,
           kv_len.data_ptr(), q_start.data_ptr(), B, None if row_limit is None else row_limit.data_ptr(),
           scale, out.data_ptr(), ldo, ws.data_ptr(), ws.numel(),
           _stream_of(dev))
    return out


_SCALE_LOG2 = math.log2(math.e) / math.sqrt(128)


class Weight4:
    """A B operand (K, N) in 4 bits with a bf16 scale per `group` values of a column, resident on the GPU in the native
    order: value (u - 8) * s. swiglu=True marks an up matrix with [gate 64 | proj 64] per 128 columns, as PackedWeight."""

    def __init__(self, codes, scales, K, N, group, swiglu=False):
        self.codes, self.scales = codes, scales
        self.K, self.N, self.group, self.swiglu = int(K), int(N), int(group), bool(swiglu)
        self._ptrs = codes.data_ptr(), scales.data_ptr()
        self._fast = (*self._ptrs, self.K, self.N, self.group, codes.get_device())

    @classmethod
    def from_codes(cls, codes, scales, swiglu=False):
        """codes uint8 (K, N), one value 0 .. 15 per byte, and scales bf16 (K / group, N) -> native order."""
        dev = _here(codes, scales)
        _check_cuda(codes, scales)
        K, N = codes.shape
        if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16 or scales.shape[1] != N or \
                scales.shape[0] == 0 or K % scales.shape[0]:
            raise ValueError("codes must be uint8 (K, N) and scales bf16 (K / group, N)")
        group = K // scales.shape[0]
        nb = [ctypes.c_size_t(), ctypes.c_size_t()]
        L.call("rl_w4_bytes", K, N, group, int(swiglu), *[ctypes.byref(b) for b in nb])
        w, s = (torch.empty(b.value, dtype=torch.uint8, device=codes.device) for b in nb)
        L.call("rl_w4_pack", _ptr(codes), _ptr(scales), K, N, group, int(swiglu), _ptr(w), _ptr(s), _stream_of(dev))
        return cls(w, s, K, N, group, swiglu)

    @classmethod
    def from_float(cls, B, group=64, swiglu=False):
        """Float B (K, N) on the GPU, rounded to 4 bits there."""
        return cls.from_codes(*quantize_w4(B, group), swiglu=swiglu)


def quantize_w4(B, group=64):
    """B (K, N) fp32/bf16 -> (codes uint8 (K, N), scales bf16 (K / group, N)): s = bf16(e / -8) with e the group's value
    of largest magnitude, u = clip(rint(w / s) + 8, 0, 15)."""
    dev = _here(B)
    _check_cuda(B)
    K, N = B.shape
    codes = torch.empty((K, N), dtype=torch.uint8, device=B.device)
    scales = torch.empty((K // max(int(group), 1), N), dtype=torch.bfloat16, device=B.device)
    L.call("rl_w4_quantize", _ptr(B), _dtype_code(B), K, N, int(group), _ptr(codes), _ptr(scales), _stream_of(dev))
    return codes, scales


def _w4(x, w, bias, epi, out, cols, out_dtype):
    if _fast is not None and out is None and (out_dtype is torch.bfloat16 or out_dtype is torch.float32):
        o = _fast.linear_w4(x, w._fast, bias, epi, cols, out_dtype is torch.float32)
        if o is not None:
            return o if type(o) is not int else L.check("rl_linear_w4", o)
    dev = _here(x, w.codes, bias, out)
    M = x.shape[0]
    if x.shape != (M, w.K) or x.dtype is not torch.bfloat16:
        raise ValueError(f"x must be bf16 (rows, {w.K}), not {x.dtype} {tuple(x.shape)}")
    if not x.is_contiguous() or (bias is not None and not bias.is_contiguous()) or (out is not None and not out.is_contiguous()):
        raise ValueError("tensor must be contiguous")
    if bias is not None and (bias.dtype is not torch.bfloat16 or bias.shape != (w.N,)):
        raise ValueError(f"bias must be bf16 ({w.N},)")
    if out is None:
        out = x.new_empty((M, cols), dtype=out_dtype)
    elif out.shape != (M, cols):
        raise ValueError(f"out must be {(M, cols)}")
    L.call("rl_linear_w4", x.data_ptr(), M, w.K, *w._ptrs, w.N, w.group, None if bias is None else bias.data_ptr(), epi,
           out.data_ptr(), _dtype_code(out), _stream_of(dev))
    return out


def linear_w4(x, w, bias=None, out=None, out_dtype=torch.bfloat16):
    """C = x @ B (+ bias) for up to 64 rows x (M, K) bf16 (any bf16 values) and a Weight4: the products of a decode step
    (linear_bfp16 takes more rows). `out` must not overlap x."""
    if w.swiglu:
        raise ValueError("linear_w4 takes a Weight4 packed without swiglu (swiglu_w4 takes the others)")
    return _w4(x, w, bias, L.RL_EPI_NONE if bias is None else L.RL_EPI_BIAS, out, w.N, out_dtype)


def swiglu_w4(x, w_up, bias=None, out=None, out_dtype=torch.bfloat16):
    """H = silu(x @ Bgate) * (x @ Bproj) for up to 64 rows, bf16 (M, N / 2) rounded once (not to bfp16 blocks: linear_w4
    takes any bf16 values). w_up must be packed with swiglu=True."""
    if not w_up.swiglu:
        raise ValueError("swiglu_w4 needs a Weight4 packed with swiglu=True")
    return _w4(x, w_up, bias, L.RL_EPI_SWIGLU, out, w_up.N // 2, out_dtype)


def set_gemm_variant(v):
    return L.lib().rl_set_gemm_variant(int(v))


def set_attention_variant(v):
    """0 = two query tiles per CTA (default), 1 = one query tile per CTA; returns the previous choice."""
    return L.lib().rl_set_attention_variant(int(v))


def set_kv_attention_path(v):
    """0 = by shape (default), 1 = the kernel that splits keys over the GPU, 2 = the tcgen05 prompt kernel, 3 = the
    first in clusters, one launch; returns the previous choice."""
    return L.lib().rl_set_kv_attention_path(int(v))


def device_status():
    return L.device_status()
