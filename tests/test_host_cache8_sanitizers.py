"""The 8-bit caches', the shared prefix's and the residual norm's host code under AddressSanitizer and UndefinedBehaviorSanitizer.

Their sources are compiled with the sanitizers on the host compilation only
(`-Xarch_host`), linked into a shared library and driven by
tests/host_cache8_driver.cpp: every size field at its extremes, in calls that
return before a launch (no kernel runs).  Runs on the CPU.
"""

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "latent_amd" / "csrc"
HIPCC = os.environ.get("HIPCC") or shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
CLANGXX = str(Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin" / "clang++")
SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
       "-Xarch_host", "-fno-sanitize-recover=undefined", "-Xarch_host", "-fno-omit-frame-pointer"]
# Device code is compiled (the host side refers to its code object) but never loaded.
COMMON = ["-O1", "-g", "-std=c++17", "--offload-arch=gfx950", "-Xarch_device", "-O3", "-Xarch_device", "-g0",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-fPIC", "-Wno-unused-command-line-argument"]


def test_8_bit_entry_points_are_clean_under_asan_and_ubsan(tmp_path):
    if not Path(HIPCC).exists() or not Path(CLANGXX).exists():
        pytest.skip("hipcc / clang++ not found")
    names = ("kvcache", "decode", "decode8", "prompt", "prompt8", "shared", "norm")
    cmds = [[HIPCC, *COMMON, *SAN, "-c", str(CSRC / f"{n}.hip"), "-o", str(tmp_path / f"{n}.o")] for n in names]
    with ThreadPoolExecutor(max_workers=len(cmds)) as pool:
        for r in pool.map(lambda c: subprocess.run(c, capture_output=True, text=True), cmds):
            assert r.returncode == 0, r.stderr[-3000:]
    lib = tmp_path / "libcache8_san.so"
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *SAN, *[str(tmp_path / f"{n}.o") for n in names],
                        "-o", str(lib)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    exe = tmp_path / "host_cache8_driver"
    r = subprocess.run([CLANGXX, "-O1", "-g", "-std=c++17", *SAN, "-I", str(ROOT / "include"),
                        str(ROOT / "tests" / "host_cache8_driver.cpp"), str(lib), f"-Wl,-rpath,{tmp_path}", "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ)
    env["ASAN_OPTIONS"] = "detect_leaks=0:halt_on_error=1:abort_on_error=0:verify_asan_link_order=0"
    env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1"
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    log = r.stdout + r.stderr
    assert "AddressSanitizer" not in log and "runtime error" not in log, log[-4000:]
    assert r.returncode == 0 and "host 8-bit cache checks: 0 failed" in r.stdout, log[-4000:]
