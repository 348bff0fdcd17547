"""Builds libaria_q4.so in-tree with nvcc for sm_100a (B200).

    python -m aria_b200.build          # incremental
    python -m aria_b200.build --force

The library is a plain C-ABI shared object (include/aria_q4.h) with the CUDA
runtime linked statically, so any host language can dlopen it; Python reaches it
through ctypes (aria_b200/_lib.py).  Objects go to aria_b200/_build/.  nvcc and its host
compiler are all that it needs.  Where torch is installed with its headers, the serving
operators get a second, shorter way from Python, the module aria_b200._fastcall
(csrc/fastcall.cpp), built for this Python and this torch.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libaria_q4.so")
FASTCALL = os.path.join(PKG, "_fastcall" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
SOURCES = ["q4_pack.cu", "q4_gemv.cu", "q4_decode.cu", "q4_gemm_tc.cu", "q4_layer.cu", "attn_prefill.cu",
           "attn_paged.cu", "prompt_weights.cu", "cache_evict.cu", "logits.cu", "p2p_allreduce.cu", "q4_capi.cu",
           "paged_capi.cu"]
HEADERS = ["q4_common.cuh", "q4_tcgen05.cuh", "q4_status.cuh", "q4_paged.cuh", "q4_logits.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else (shutil.which("nvcc") or "nvcc")


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def build_fastcall(force: bool = False) -> str | None:
    """The C++ binding of the serving operators (host code only; torch's headers and the
    libraries that `import torch` loads), or None where torch or its headers are absent."""
    from ._lib import fastcall_key
    key, src = fastcall_key(), os.path.join(CSRC, "fastcall.cpp")
    key_file = os.path.join(OBJ, "fastcall.key")
    if key is None:
        return None
    built = open(key_file).read() if os.path.exists(key_file) else ""
    if not force and built == key and not _newer(FASTCALL, [src, os.path.join(ROOT, "include", "aria_q4.h")]):
        return FASTCALL
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    # torch's headers name CUDA types even where no CUDA call is made
    inc = [*include_paths(), sysconfig.get_paths()["include"],
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    if torch.version.cuda is None or not any(os.path.exists(os.path.join(d, "ATen", "ATen.h")) for d in inc) or not any(
            os.path.exists(os.path.join(d, "Python.h")) for d in inc):
        return None
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f'-DFASTCALL_KEY="{key}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *[f"-I{d}" for d in inc], src,
           "-o", FASTCALL, *[f"-L{d}" for d in library_paths()], "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10",
           "-lc10_cuda"]
    env = {k: v for k, v in os.environ.items() if k not in ("CC", "CXX")}
    r = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on fastcall.cpp:\n{r.stdout}\n{r.stderr}")
    with open(key_file, "w") as f:
        f.write(key)
    return FASTCALL


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "aria_q4.h")]
    objs = []
    env = dict(os.environ)
    env.pop("CC", None)
    env.pop("CXX", None)
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        if not os.path.exists(s):
            continue
        o = os.path.join(OBJ, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _newer(o, [s] + headers):
            cmd = [nvcc(), *NVCC_FLAGS, "-ccbin", "g++", "-c", s, "-o", o]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            r = subprocess.run(cmd, capture_output=True, text=True, env=env)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
            if verbose:
                sys.stderr.write(r.stderr)
    if force or _newer(LIB, objs):
        cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-ccbin", "g++",
               "-o", LIB, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True, env=env)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if build_fastcall(force) is None:
        sys.stderr.write("aria_b200: no torch headers here: without aria_b200._fastcall the serving operators' calls "
                         "take a few microseconds longer\n")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
