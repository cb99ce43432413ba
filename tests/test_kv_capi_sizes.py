"""CPU-side refusals of cache calls that would need more CTAs than a launch has (no kernel is launched)."""

from test_kv_capi import append_args, lib, refused  # noqa: F401


def test_append(lib):  # noqa: F811
    refused(lib, "rl_kv_append", append_args(T=1 << 24, hkv=2048), -1, b"rows of 2048 heads")
