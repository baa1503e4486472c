"""Build the native parts in-tree.

    python -m minispeed_amd.build [--verbose]

* ``libminispeed_boundary.so``: the HIP kernels for gfx950 behind a plain C
  ABI (no torch headers), compiled with hipcc;
* ``_walk.so``: a small host-only Python extension (g++, torch and pybind11
  headers) that collects the device addresses of parameter gradients and
  storages for the segment tables;
* ``libminispeed_ops.so``: the language-model operators' HIP kernels behind a C
  ABI of their own (``include/minispeed_ops.h``), and ``_ops.so``, the Python
  extension that checks their tensors and launches them.

All are written next to this file so that they travel with the source tree.
(bench.py's streaming probes are built by ``bench_probes/build.py``.)
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from typing import List

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
SOURCES = [os.path.join(PKG_DIR, "csrc", "boundary.hip")]
INCLUDE = os.path.join(REPO_DIR, "include")
OUTPUT = os.path.join(PKG_DIR, "libminispeed_boundary.so")
ARCH = "gfx950"
OPS_SOURCES = [os.path.join(PKG_DIR, "csrc", f"{name}.hip")
               for name in ("embedding", "logprobs", "act8", "linear", "norm", "posbias")]
OPS_OUTPUT = os.path.join(PKG_DIR, "libminispeed_ops.so")

# -ffp-contract=off: every a*b+c the kernels do not write as fmaf stays two
#   roundings, matching the op-by-op rounding of the torch sequence they
#   replace.
# -packed-fp32-ops: keep the compiler from emitting packed fp32 VALU ops.
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (expected /opt/rocm/bin/hipcc)")


def command(output: str = OUTPUT) -> List[str]:
    return [hipcc(), *HIP_FLAGS, f"-I{INCLUDE}", *SOURCES, "-o", output]


def ops_command(output: str = OPS_OUTPUT) -> List[str]:
    return [hipcc(), *HIP_FLAGS, "-parallel-jobs=6", f"-I{INCLUDE}", *OPS_SOURCES, "-o", output]


def _compile_hip(cmd: List[str], tmp: str, output: str, verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the packed-fp32 feature; that warning is
    # expected and harmless.
    noise = ("packed-fp32-ops", "--hip-link")
    log = "\n".join(
        line for line in (proc.stdout + proc.stderr).splitlines()
        if line.strip() and not any(n in line for n in noise)
    )
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{log}")
    if verbose and log:
        print(log)
    os.replace(tmp, output)
    return output


def build(verbose: bool = False) -> str:
    """Compile the boundary library (always, even when an older build exists)."""
    tmp = OUTPUT + ".tmp"
    return _compile_hip(command(tmp), tmp, OUTPUT, verbose)


def build_ops(verbose: bool = False) -> str:
    """Compile the operators' library (always)."""
    tmp = OPS_OUTPUT + ".tmp"
    return _compile_hip(ops_command(tmp), tmp, OPS_OUTPUT, verbose)


WALK_SOURCE = os.path.join(PKG_DIR, "csrc", "walk.cpp")
WALK_OUTPUT = os.path.join(PKG_DIR, "_walk.so")


OPS_BIND_SOURCE = os.path.join(PKG_DIR, "csrc", "ops_bind.cpp")
OPS_BIND_OUTPUT = os.path.join(PKG_DIR, "_ops.so")


def _extension_command(source: str, output: str, *more: str) -> List[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    incs = [sysconfig.get_paths()["include"], *cpp_extension.include_paths()]
    libdir = cpp_extension.library_paths()[0]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *[f"-I{d}" for d in incs], source,
            "-o", output, f"-L{libdir}", "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", *more]


def walk_command(output: str = WALK_OUTPUT) -> List[str]:
    return _extension_command(WALK_SOURCE, output)


def ops_bind_command(output: str = OPS_BIND_OUTPUT) -> List[str]:
    rocm = os.path.dirname(os.path.dirname(hipcc()))
    return _extension_command(
        OPS_BIND_SOURCE, output, "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM", f"-I{rocm}/include",
        f"-I{INCLUDE}", "-lc10_hip", f"-L{PKG_DIR}", "-lminispeed_ops", "-Wl,-rpath,$ORIGIN")


def _compile_extension(cmd: List[str], tmp: str, output: str, verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stdout}{proc.stderr}")
    os.replace(tmp, output)
    return output


def build_walk(verbose: bool = False) -> str:
    """Compile ``_walk.so`` (always)."""
    tmp = WALK_OUTPUT + ".tmp"
    return _compile_extension(walk_command(tmp), tmp, WALK_OUTPUT, verbose)


def build_ops_bind(verbose: bool = False) -> str:
    """Compile ``_ops.so`` (always), against the ``libminispeed_ops.so`` next to it."""
    tmp = OPS_BIND_OUTPUT + ".tmp"
    return _compile_extension(ops_bind_command(tmp), tmp, OPS_BIND_OUTPUT, verbose)


def build_all(verbose: bool = False) -> List[str]:
    """Everything, the independent parts at the same time."""
    with ThreadPoolExecutor(3) as pool:
        jobs = [pool.submit(build, verbose), pool.submit(build_walk, verbose),
                pool.submit(lambda: [build_ops(verbose), build_ops_bind(verbose)])]
        boundary, walk, ops = [job.result() for job in jobs]
    return [boundary, walk, *ops]


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args(argv)
    for path in build_all(verbose=args.verbose):
        print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
