"""The per-stream workspaces among host threads (tests/sanitize/workspace_turns.cpp):
a buffer that one thread has and has not yet launched on is neither released nor
evicted by another.  Built for the CPU with AddressSanitizer on a stand-in for the
HIP runtime; no GPU is used."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from test_sanitize import CSRC, HOST_SOURCES, ROOT, SAN, _run


@pytest.fixture(scope="module")
def turns(tmp_path_factory):
    gxx = shutil.which("g++")
    hip_lib = Path("/opt/rocm/lib")
    if not gxx or not (hip_lib / "libamdhip64.so").exists():
        pytest.skip("needs g++ and the ROCm runtime library")
    out = tmp_path_factory.mktemp("turns") / "workspace_turns"
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-D__HIP_PLATFORM_AMD__",
           "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{CSRC}",
           str(SAN / "workspace_turns.cpp"), str(SAN / "launch_stubs.cpp"),
           *[str(CSRC / s) for s in HOST_SOURCES],
           f"-L{hip_lib}", "-lamdhip64", f"-Wl,-rpath,{hip_lib}", "-lpthread", "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, f"build failed:\n{r.stderr[-4000:]}"
    return out


@pytest.mark.parametrize("what", ["release", "evict", "threads"])
def test_a_buffer_in_hand_stays(turns, what):
    assert "ok" in _run(turns, what, timeout=60)
