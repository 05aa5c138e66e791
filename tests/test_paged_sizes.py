"""Sizes at the ends of their range, and workspaces: the argument rules of the paged
cache and of sampled tokens return, whatever they are asked."""

from __future__ import annotations

import os
import shutil
import subprocess
from ctypes import byref
from pathlib import Path

import pytest

from leanstack_amd import _lib

REPO = Path(__file__).resolve().parent.parent
MOST = 2**31 - 1
FAKE = 0x10000  # aligned, never dereferenced


@pytest.mark.parametrize("b,t,n_q,n_kv,capacity", [
    (MOST, MOST, MOST, MOST, MOST), (1 << 20, 1 << 20, 32, 8, 4096), (MOST, 1, 1, 1, 4096), (1, MOST, 8, 8, 4096),
    (0, 1, 8, 8, 4096), (1, 0, 8, 8, 4096), (1, 1, 8, 0, 4096), (1, 1, 7, 8, 4096), (1, 1, 12, 8, 4096), (1, 1, 8, 8, 0),
    (1, 1, 8, 8, -16), (1, 1, 8, 8, 4095), (1, 1, 8, 8, MOST), (1, 1, 8, 8, (1 << 30) + 16), (1 << 16, 64, 8, 8, 1 << 30),
    (4, 1, 32, 8, 1536), (16, 5, 32, 8, 2048), (63, 16, 32, 8, 2048),   # (served by one launch without a workspace)
])
def test_no_workspace(b, t, n_q, n_kv, capacity):
    assert _lib.load().lsk_paged_attention_workspace_bytes(b, t, n_q, n_kv, capacity) == 0


@pytest.mark.parametrize("b,t,n_q,n_kv,capacity", [
    (1, 1, 32, 8, 1552), (16, 5, 32, 8, 2064), (64, 1, 32, 8, 64), (64, 1, 32, 8, 1 << 16), (24, 5, 32, 8, 4096), (2, 1500, 32, 8, 2048), (1, 1, 8, 8, 1 << 30),
    (1, 17, 32, 8, 64), (4096, 1, 32, 8, 8192), (1, 1, 4096, 4096, 2048),
])
@pytest.mark.parametrize("bad", ["none", "small", "misaligned"])
def test_workspace_is_checked(b, t, n_q, n_kv, capacity, bad):
    lib = _lib.load()
    need = lib.lsk_paged_attention_workspace_bytes(b, t, n_q, n_kv, capacity)
    # (parts of a wave or a workgroup: more would be more than they are worth)
    assert 0 < need < 1 << 30
    pool = _lib.PagedPool(FAKE, FAKE, FAKE, FAKE, 1, n_kv, 16, capacity // 16, FAKE, capacity // 16)
    at, size = {"none": (None, need), "small": (FAKE, need - 1), "misaligned": (FAKE + 8, need + 64)}[bad]
    status = lib.lsk_paged_attention_bf16(byref(pool), FAKE, n_q * t * 128, t * 128, 128, b, t, n_q, 128, FAKE, None, 0.1, FAKE, at,
                                          size, None)
    assert status == _lib.ERR_WORKSPACE and str(need) in _lib.last_error()


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_size_rules_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "paged_rules_driver"
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=undefined", f"-I{REPO / 'include'}", f"-I{REPO / 'leanstack_amd' / 'csrc'}",
           str(REPO / "leanstack_amd" / "csrc" / "host_rules.cpp"), str(REPO / "tests" / "asan" / "paged_rules_driver.cpp"),
           "-o", str(exe)]
    build = subprocess.run(cmd, capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    env = dict(os.environ, ASAN_OPTIONS="halt_on_error=1:detect_leaks=1", UBSAN_OPTIONS="halt_on_error=1")
    run = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr
