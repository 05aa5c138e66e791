"""Sizes at the ends of their range: the workspace queries and argument rules of
the operators for a batch of requests return, whatever they are asked."""

from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

from leanstack_amd import _lib

REPO = Path(__file__).resolve().parent.parent
MOST = 2**31 - 1


@pytest.mark.parametrize("b,t,n_q,n_kv,prefix,rows", [
    (1 << 20, 1 << 20, 32, 8, 1000, 100),   # 2^35 tiles of query rows: 0 in 32 bits
    (1 << 23, 1 << 19, 4, 1, 1 << 20, 0), (MOST, MOST, MOST, MOST, MOST, MOST), (MOST, 1, 1, 1, 1000, 1000),
    (1, MOST, 8, 8, 0, 1000), (1, 1, 32, 8, MOST, 0), (1, 1, 32, 8, 0, MOST), (1, 1, 32, 8, 1 << 23, 1 << 23),
])
def test_attention_workspace_of_sizes_it_does_not_serve(b, t, n_q, n_kv, prefix, rows):
    assert _lib.load().lsk_prefix_attention_workspace_bytes(b, t, n_q, n_kv, prefix, rows) == 0


@pytest.mark.parametrize("m,n,k,rank_tiles,count,epilogue", [
    (MOST, MOST, MOST, 8, MOST, 0), (300, 1 << 22, 32, 1, 1, 0), (300, 32, 1 << 22, 1, 1, 0), (300, 40, 32, 1, 1, 0),
    (300, 48, 32, 1, 1, 1), (MOST, 16, 32, 1, 1, 0), (300, 16, 32, 1, 1, 7),
])
def test_adapter_workspace_of_sizes_it_does_not_serve(m, n, k, rank_tiles, count, epilogue):
    assert _lib.load().lsk_lora_workspace_bytes(m, n, k, rank_tiles, count, epilogue) == 0


@pytest.mark.parametrize("scale", [3e38, -3.4e38])
def test_attention_scales_that_overflow_in_base_2(scale):
    """scale * log2(e) has to be finite, or equal scores of zero would give NaN."""
    at = 0x10000  # aligned, never dereferenced
    status = _lib.load().lsk_prefix_attention_bf16(at, 1024, 128, 1024, 1, 1, 8, 2, 128, at, at, 128 * 64, 128, 64, at, at, 2 * 128 * 8,
                                                   128 * 8, 128, 8, at, scale, at, None, 0, None)
    assert status == _lib.ERR_INVALID and "scale" in _lib.last_error()


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_size_rules_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "batch_rules_driver"
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=undefined", f"-I{REPO / 'include'}", f"-I{REPO / 'leanstack_amd' / 'csrc'}",
           str(REPO / "leanstack_amd" / "csrc" / "host_rules.cpp"), str(REPO / "tests" / "asan" / "batch_rules_driver.cpp"),
           "-o", str(exe)]
    build = subprocess.run(cmd, capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    env = dict(os.environ, ASAN_OPTIONS="halt_on_error=1:detect_leaks=1", UBSAN_OPTIONS="halt_on_error=1")
    run = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr
