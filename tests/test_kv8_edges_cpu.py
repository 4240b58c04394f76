"""Edges of the paged KV cache in 8 bits that need no GPU."""

from __future__ import annotations

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def part_count(tmp_path_factory):
    """kv8_part_count of the kernels' own source, built for the host."""
    folder = tmp_path_factory.mktemp("parts")
    (folder / "parts.cpp").write_text('#include "kv8_parts.cuh"\nextern "C" int count(int a, int b, int c, int d) '
                                      "{ return t2c::kv8_part_count(a, b, c, d); }\n")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", str(REPO / "torch2vk_b200" / "csrc"), str(folder / "parts.cpp"),
                    "-o", str(folder / "parts.so")], check=True)
    return ctypes.CDLL(str(folder / "parts.so")).count


def test_join_takes_the_records_of_a_run(part_count):
    """Runs of equal tile counts over units of any lengths: what the CTAs record is always taken, with its count."""
    rng = random.Random(5)
    for _ in range(300):
        units = [rng.randint(1, 40) for _ in range(rng.randint(1, 60))]
        total, tiles = sum(units), max(units)
        ctas = min(rng.choice([1, 2, 7, 60, 592]), len(units) * tiles)
        used, starts = min(ctas, total), []
        for c in range(used):
            starts.append(c * (total // used) + min(c, total % used))
        at = 0
        for n in units:
            first = max(c for c in range(used) if starts[c] <= at)
            last = max(c for c in range(used) if starts[c] <= at + n - 1)
            assert part_count(first, last, ctas, min(ctas, tiles)) == last - first + 1
            at += n


def test_join_makes_no_index_of_a_record_that_was_not_written(part_count):
    """Whatever an unwritten record holds, the parts that are read lie in the workspace and fit the factors."""
    rng = random.Random(6)
    edges = [-(1 << 31), -2, -1, 0, 1, 7, 8, 591, 592, (1 << 31) - 1, 0x7F7F7F7F, 0x7FC00000]
    for ctas, most in ((1, 1), (8, 3), (592, 592), (592, 40), (8192, 8192)):
        for first in edges:
            for last in edges + [rng.randrange(-(1 << 31), 1 << 31) for _ in range(20)]:
                n = part_count(first, last, ctas, most)
                assert n == (last - first + 1 if 0 <= first <= last < ctas and last - first < most else 0)


def test_workspace_sizes_are_kept_per_device(monkeypatch):
    """A workspace's size goes by the device's SMs: what was asked on one device is no answer for another."""
    from types import SimpleNamespace

    from torch2vk_b200 import kernels

    now = {"device": 0}
    floats = {0: 1000, 1: 2000}
    monkeypatch.setattr(kernels.torch.cuda, "current_device", lambda: now["device"])
    monkeypatch.setattr(kernels._lib, "lib", lambda: SimpleNamespace(raw=lambda name: lambda *args: floats[now["device"]]))
    pages = SimpleNamespace(n_kv=8, head_dim=128, page_size=64)
    table = SimpleNamespace(shape=(4, 100))
    kernels._q8_workspace_floats.cache_clear()
    try:
        for device in (0, 1, 0, 1):
            now["device"] = device
            assert kernels.attn_decode_q8_workspace(pages, table, batch=4, n_heads=32) == floats[device]
            assert kernels.attn_prefill_q8_workspace(pages, table, batch=4, tokens=5, n_heads=32) == floats[device]
    finally:
        kernels._q8_workspace_floats.cache_clear()


def test_stream_handle_without_torch_internals(monkeypatch):
    """A torch without the raw-handle function: its current stream is asked instead."""
    from types import SimpleNamespace

    from torch2vk_b200 import _lib

    monkeypatch.setattr(_lib.torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=77))
    monkeypatch.setattr(_lib, "_raw_stream", None)
    assert _lib.stream_ptr() == 77
    assert _lib.stream_ptr(SimpleNamespace(cuda_stream=5)) == 5
