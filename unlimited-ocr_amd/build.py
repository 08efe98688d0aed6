"""Build libsrswa.so (the gfx950 HIP kernels + C ABI) in-tree with hipcc, and
_host.so (the native host path of the 8-bit cache and page pool calls) with g++.

Usage: ``python unlimited-ocr_amd/build.py [-j N] [-v]``.  Every ``csrc/*.hip``
file is compiled to an object in parallel and linked into
``srswa/libsrswa.so`` next to the Python package that loads it.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
OUT = os.path.join(HERE, "srswa", "libsrswa.so")
HOST_OUT = os.path.join(HERE, "srswa", "_host.so")
ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    # no packed-fp32 instructions anywhere in the device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


# Files whose results must follow a fixed rounding order (each product and sum
# rounded on its own): hipcc fuses a*b + c into an FMA by default and its
# backend does so even under `#pragma clang fp contract(off)`.
NO_CONTRACT = {"rope2d.hip", "router.hip", "route_serve.hip"}


# Kernels whose matrix-instruction accumulators stay in the vector registers:
# left to itself the compiler keeps them in the accumulation registers and copies
# them over and back in every pass of a loop that also rescales them.
MFMA_VGPRS = {"cache8_decode.hip", "cache8_prefill.hip"}


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required to build libsrswa.so)")


def _compile(src: str, obj: str, verbose: bool) -> str:
    extra = ["-ffp-contract=off"] if os.path.basename(src) in NO_CONTRACT else []
    if os.path.basename(src) in MFMA_VGPRS:
        extra += ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
    cmd = [hipcc(), *HIPCC_FLAGS, *extra, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    msg = "\n".join(line for line in (res.stdout + res.stderr).splitlines()
                    if "packed-fp32-ops" not in line and line.strip())
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {os.path.basename(src)}:\n{msg}")
    return msg


def _host_object(obj: str, verbose: bool) -> None:
    import torch
    from torch.utils.cpp_extension import include_paths

    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           f"-I{sysconfig.get_paths()['include']}", "-isystem", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
           *(x for p in include_paths() for x in ("-isystem", p)), "-c", os.path.join(CSRC, "host.cpp"), "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on host.cpp:\n{res.stdout}{res.stderr}")


def _host_link(obj: str) -> None:
    """_host.so next to the library it calls; torch's libraries are the ones ``import torch`` has loaded."""
    import torch

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = HOST_OUT + ".tmp"
    res = subprocess.run(["g++", "-shared", "-fPIC", "-o", tmp, obj, OUT, f"-L{lib}", "-ltorch_python", "-ltorch_cpu",
                          "-ltorch", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"], capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of _host.so failed:\n{res.stdout}{res.stderr}")
    os.replace(tmp, HOST_OUT)


def build(jobs: int | None = None, verbose: bool = False) -> str:
    """Compile all kernels and link ``srswa/libsrswa.so``, then ``srswa/_host.so``;
    returns the library's path."""
    srcs = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))
    if not srcs:
        raise RuntimeError("no HIP sources under csrc/")
    jobs = jobs or min(len(srcs), max(1, (os.cpu_count() or 4)))
    with tempfile.TemporaryDirectory(prefix="srswa_build_") as tmp:
        objs = [os.path.join(tmp, os.path.basename(s)[:-4] + ".o") for s in srcs]
        with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
            futs = [ex.submit(_compile, s, o, verbose) for s, o in zip(srcs, objs)]
            host_obj = os.path.join(tmp, "host.o")
            host = ex.submit(_host_object, host_obj, verbose)
            for f in futs:
                warn = f.result()
                if warn and verbose:
                    print(warn, flush=True)
            host.result()
        tmp_out = OUT + ".tmp"
        # --no-undefined: a kernel whose host stub was not emitted fails here, not at load time
        cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-Wl,--no-undefined", "-Wl,-soname,libsrswa.so", "-o", tmp_out, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}{res.stderr}")
        os.replace(tmp_out, OUT)
        _host_link(host_obj)
    return OUT


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("-j", "--jobs", type=int, default=None)
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args(argv)
    path = build(args.jobs, args.verbose)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
