"""GPU parity of the 4-bit weights (rl_w4_quantize, rl_w4_pack, rl_linear_w4) against oracle/cache_oracle.py.

Codes and scales are held bit for bit. Products: |c - ref| <= the oracle's fp32 sum bound (+ half a step, 2^-8 |ref|, of
a bf16 output); SwiGLU carries both sums' bounds through silu (|silu'| <= 1.1) and adds 2^-18 for the exponential and
the division."""

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


def bf16(torch, a, dev):
    return torch.from_numpy(O.bf16_bits(np.asarray(a, np.float32)).view(np.int16)).to(dev).view(torch.bfloat16)


def make(rng, M, K, N, G):
    x = O.bf16_round((rng.standard_normal((M, K)) * 3).astype(np.float32))
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = O.bf16_round((rng.standard_normal((K // G, N)) * 0.02).astype(np.float32))
    bias = O.bf16_round(rng.standard_normal(N).astype(np.float32))
    return x, codes, scales, bias


def close(got, ref, tol):
    got = got.float().cpu().numpy().astype(np.float64)
    assert got.shape == ref.shape and np.isfinite(got).all()
    off = np.abs(got - ref) - tol
    assert off.max() <= 0, f"largest excess {off.max():.3e}"


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("K,N,G", [(32, 1, 32), (128, 16, 128), (96, 33, 32), (320, 100, 64), (2176, 257, 64),
                                   (1152, 515, 128), (4128, 48, 32)])
def test_linear(env, M, K, N, G):
    torch, ops, L, dev = env
    rng = np.random.default_rng(M * 1000 + K + N)
    x, codes, scales, bias = make(rng, M, K, N, G)
    w = ops.Weight4.from_codes(torch.from_numpy(codes).to(dev), bf16(torch, scales, dev))
    assert (w.K, w.N, w.group) == (K, N, G)
    xt, bt = bf16(torch, x, dev), bf16(torch, bias, dev)
    ref, tol = C.linear_w4(x, codes, scales)
    c32 = ops.linear_w4(xt, w, out_dtype=torch.float32)
    c16 = ops.linear_w4(xt, w, bias=bt)
    ops.device_status()
    close(c32, ref, tol)
    close(c16, ref + bias, tol + 2.0 ** -23 * np.abs(ref) + 2.0 ** -8 * np.abs(ref + bias) + 2.0 ** -8 * tol)
    assert torch.equal(c32, ops.linear_w4(xt, w, out_dtype=torch.float32))


@pytest.mark.parametrize("M,K,F,G", [(1, 128, 64, 32), (3, 512, 192, 64), (12, 1184, 320, 32), (40, 256, 128, 128)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_swiglu(env, M, K, F, G, with_bias):
    torch, ops, L, dev = env
    rng = np.random.default_rng(M + K + F)
    x, codes, scales, bias = make(rng, M, K, 2 * F, G)
    w = ops.Weight4.from_codes(torch.from_numpy(codes).to(dev), bf16(torch, scales, dev), swiglu=True)
    got = ops.swiglu_w4(bf16(torch, x, dev), w, bias=bf16(torch, bias, dev) if with_bias else None)
    ops.device_status()
    ref, tol = C.linear_w4(x, codes, scales)
    if with_bias:
        ref = ref + bias
        tol = tol + 2.0 ** -23 * np.abs(ref)
    z, e = ref.reshape(M, -1, 2, 64), tol.reshape(M, -1, 2, 64)
    g, u, eg, eu = z[:, :, 0], z[:, :, 1], e[:, :, 0], e[:, :, 1]
    with np.errstate(over="ignore"):
        silu = g / (1 + np.exp(-g))
    h = (silu * u).reshape(M, F)
    eh = (1.1 * eg * (np.abs(u) + eu) + np.abs(silu) * eu).reshape(M, F) + 2.0 ** -18 * np.abs(h)
    close(got, h, eh + 2.0 ** -8 * (np.abs(h) + eh))


@pytest.mark.parametrize("K,N,G", [(64, 5, 32), (384, 130, 64), (256, 300, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize(env, K, N, G, dtype):
    torch, ops, L, dev = env
    rng = np.random.default_rng(K + N)
    B = (rng.standard_normal((K, N)) * 0.02).astype(np.float32)
    B[:, 0] = 0
    B[:G, 1] = np.tile(np.array([0.5, -0.5], np.float32), G // 2)     # equal magnitudes: the first one counts
    if dtype == "bf16":
        B = O.bf16_round(B)
    t = torch.from_numpy(B).to(dev)
    codes, scales = ops.quantize_w4(t.to(torch.bfloat16) if dtype == "bf16" else t, G)
    want, s = C.quantize_w4(B, G)
    assert np.array_equal(scales.float().cpu().numpy(), s) and np.array_equal(codes.cpu().numpy(), want)
    x = O.bf16_round(rng.standard_normal((4, K)).astype(np.float32))
    ref, tol = C.linear_w4(x, want, s)
    got = ops.linear_w4(bf16(torch, x, dev), ops.Weight4.from_float(t, G), out_dtype=torch.float32)
    ops.device_status()
    close(got, ref, tol)


def test_non_finite(env):
    """An infinity or a NaN in a row of x reaches that row only; a NaN weight group reaches its column only."""
    torch, ops, L, dev = env
    rng = np.random.default_rng(1)
    x, codes, scales, _ = make(rng, 5, 256, 40, 64)
    codes[:] = np.where(codes == 8, 9, codes)
    x[2, 100] = np.inf
    x[3, 7] = np.nan
    scales[1, 11] = np.nan
    w = ops.Weight4.from_codes(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev).to(torch.bfloat16))
    got = ops.linear_w4(torch.from_numpy(x).to(dev).to(torch.bfloat16), w).float().cpu().numpy()
    ops.device_status()
    bad = ~np.isfinite(got)
    want = np.zeros((5, 40), bool)
    want[2:4] = True
    want[:, 11] = True
    assert np.array_equal(bad, want)
    B = torch.full((64, 2), 0.1, device=dev)
    B[3, 0] = float("inf")
    _, s = ops.quantize_w4(B, 64)
    assert torch.isnan(s[0, 0]) and torch.isfinite(s[0, 1])


def test_refusals(env):
    torch, ops, L, dev = env
    codes = torch.full((64, 32), 8, dtype=torch.uint8, device=dev)
    scales = torch.ones((1, 32), dtype=torch.bfloat16, device=dev)
    w = ops.Weight4.from_codes(codes, scales)
    x = torch.zeros((65, 64), dtype=torch.bfloat16, device=dev)
    with pytest.raises(L.RedlineError, match="rows"):
        ops.linear_w4(x, w)
    for bad in (x[:4].float(), x[:4, :32].contiguous(), x[:4].cpu()):
        with pytest.raises(ValueError):
            ops.linear_w4(bad, w)
    with pytest.raises(ValueError):
        ops.swiglu_w4(x[:1], w)
    with pytest.raises(ValueError):
        ops.linear_w4(x[:1], w, bias=torch.zeros(31, dtype=torch.bfloat16, device=dev))
    with pytest.raises(L.RedlineError, match="group"):
        ops.Weight4.from_codes(codes, torch.ones((4, 32), dtype=torch.bfloat16, device=dev))
    with pytest.raises(L.RedlineError, match="128"):
        ops.Weight4.from_codes(codes, scales, swiglu=True)
    assert ops.linear_w4(x[:0], w).shape == (0, 32)
