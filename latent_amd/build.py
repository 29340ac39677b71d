"""Build liblatent_hip.so (gfx950) and the attention calls' binding, _attend.so, in-tree.

    python latent_amd/build.py

(Run as a script: importing the package would load the library being rebuilt.)

The library links only against the HIP runtime; no torch headers.  When the
Python binding loads it after `import torch`, the dynamic linker binds it to
the HIP runtime torch already loaded (same SONAME), so torch's streams and
device pointers are valid in it.  _attend.so (bind_attend.cpp, host code) is a
Python extension over torch's C++ interface, for the calls of a decode step whose
arguments take longer to look at from Python than the GPU needs for them.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import Optional

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
SOURCES = ["chain32.hip", "codec.hip", "decode.hip", "decode8.hip", "expert.hip", "kvcache.hip", "moe.hip", "noalloc.hip", "norm.hip",
           "prefill.hip", "prompt.hip", "prompt8.hip", "route.hip", "rows.hip", "shared.hip", "stream.hip"]
LIB = PKG / "liblatent_hip.so"
BINDING = PKG / "_attend.so"
ARCH = os.environ.get("LATENT_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    f"--offload-arch={ARCH}",
    "-fPIC",
    # Keep the compiler from forming packed-FP32 (v_pk_*_f32) instructions.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-munsafe-fp-atomics",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC)")


def binding_command(out: Path) -> Optional[list]:
    """None without torch: there is nothing to bind to."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    torch = Path(spec.submodule_search_locations[0])
    rocm = Path(hipcc()).resolve().parent.parent / "include"
    include = [torch / "include", rocm, sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            *[f"-I{i}" for i in include], str(CSRC / "bind_attend.cpp"), "-o", str(out), f"-L{torch / 'lib'}",
            "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip"]


def build(verbose: bool = False) -> Path:
    """Compile every source and link the shared library and the binding; always rebuilds.

    The library needs hipcc alone and is in place before an error of the binding's (torch's headers, g++) is raised;
    a binding that cannot be built leaves none, and without it everything but the attention calls works.
    """
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    cc = hipcc()
    cmds, objs = [], []
    for src in SOURCES:
        obj = objdir / (Path(src).stem + ".o")
        cmds.append([cc, *HIPCC_FLAGS, "-c", str(CSRC / src), "-o", str(obj)])
        objs.append(str(obj))
    tmp_binding = BINDING.with_suffix(".so.tmp")
    binding = binding_command(tmp_binding)

    def run(cmd):
        try:
            return subprocess.run(cmd, capture_output=True, text=True)
        except OSError as e:  # no such program
            return subprocess.CompletedProcess(cmd, 127, "", f"{cmd[0]}: {e}\n")

    # One compiler process per source, at most `jobs` at a time.
    jobs = max(1, min(len(cmds) + 1, int(os.environ.get("MAX_JOBS", os.cpu_count() or 1))))
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        for cmd in cmds + [binding or []]:
            if verbose and cmd:
                print(" ".join(cmd), flush=True)
        bound = pool.submit(run, binding) if binding else None
        for result in pool.map(run, cmds):
            sys.stderr.write(result.stderr)
            if result.returncode != 0:
                raise subprocess.CalledProcessError(result.returncode, result.args, result.stdout, result.stderr)
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    if bound is not None and bound.result().returncode == 0:
        sys.stderr.write(bound.result().stderr)
        os.replace(tmp_binding, BINDING)
        return LIB
    BINDING.unlink(missing_ok=True)  # an older one may not fit the library
    if bound is not None:
        raise RuntimeError(f"{LIB.name} is built, the binding {BINDING.name} is not:\n{bound.result().stderr}")
    print(f"torch not found: {BINDING.name}, the binding of the attention calls, is not built", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv)
    print(path)
