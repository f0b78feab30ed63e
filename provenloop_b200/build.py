"""Build libtsgpu.so (the CUDA engine behind the C ABI in include/tsgpu.h).

Compiles every CUDA source for sm_100a only, in-tree, with plain nvcc, and
where torch is installed the checks of the torch entry points beside it
(_torch_ops.so, host code, for that torch and Python):

    python -m provenloop_b200.build           # or __graft_entry__.build()

Host code is compiled with -ffp-contract=off so the f64 FFT tables built on
the host round exactly like the reference's (glibc cos/sin, no FMA).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtsgpu.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")  # torch tensors to argument blocks (csrc/torch_ops.cpp)
SOURCES = ["kernels.cu", "k_ntt.cu", "k_encode.cu", "k_encrypt.cu", "k_decrypt.cu", "tsgpu.cu", "noalloc.cu",
           "k_lowrank.cu", "k_project.cu", "k_rules.cu", "decode_ops.cu", "k_loss.cu", "k_clip.cu", "train_ops.cu"]
HEADERS = ["common.cuh", "ntt.cuh", "fft.cuh", "kernels.cuh", "launch.cuh", "lowrank.cuh",
           "sm100.cuh", "entry.cuh", "train.cuh"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def flags(verbose_ptxas: bool = False):
    f = [
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-O3", "-lineinfo", "-std=c++17",
        "-Xcompiler", "-fPIC,-ffp-contract=off,-fno-fast-math",
        "-I", os.path.join(ROOT, "include"),
    ]
    if verbose_ptxas:
        f += ["-Xptxas", "-v"]
    return f


def have_torch() -> bool:
    return importlib.util.find_spec("torch") is not None


def torch_tag() -> str:
    """What a build of _torch_ops.so is for; the module carries it as text."""
    return f"torch {importlib.metadata.version('torch')}, {sys.implementation.cache_tag}"


def torch_ops_command(out: str):
    import sysconfig

    import torch
    base = os.path.dirname(torch.__file__)
    inc, libs = os.path.join(base, "include"), os.path.join(base, "lib")
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    # the C++ library by its shared object: a compiler that finds only the static
    # one would give the module a second copy beside torch's, and an exception
    # that passes between them ends the process
    return [shutil.which("g++") or os.environ.get("CXX", "c++"), "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DTSGPU_BUILT_FOR="{torch_tag()}"', "-I", inc,
            "-I", os.path.join(inc, "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"],
            "-I", os.path.join(cuda, "include"), os.path.join(CSRC, "torch_ops.cpp"), "-o", out, "-L", libs, "-ltorch_python", "-ltorch",
            "-ltorch_cpu", "-lc10", "-lc10_cuda", "-nostdlib++", "-l:libstdc++.so.6"]


def _older(path: str, sources) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    deps = [os.path.join(CSRC, s) for s in sources] + [os.path.join(ROOT, "include", "tsgpu.h")]
    return any(os.path.getmtime(p) > t for p in deps if os.path.exists(p))


def torch_ops_fits() -> bool:
    """Whether _torch_ops.so was built for this torch and this Python."""
    with open(TORCH_OPS, "rb") as f:
        return torch_tag().encode() in f.read()


def torch_ops_stale() -> bool:
    return have_torch() and (_older(TORCH_OPS, ["torch_ops.cpp"]) or not torch_ops_fits())


def needs_build() -> bool:
    return _older(LIB, SOURCES + HEADERS) or torch_ops_stale()


def _finish(name: str, process, verbose: bool) -> None:
    out, err = process.communicate()
    if process.returncode != 0:
        raise RuntimeError(f"compiling {name} failed:\n{out}\n{err}")
    if verbose:
        sys.stdout.write(out + err)


def build(force: bool = False, verbose: bool = False) -> str:
    """The library, which needs nvcc only, and with torch installed the torch
    module, which needs its headers and g++: the library is there even if the
    module cannot be built."""
    pipes = dict(stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    ops = None
    if have_torch() and (force or torch_ops_stale()):
        try:
            ops = subprocess.Popen(torch_ops_command(TORCH_OPS + ".tmp"), **pipes)
        except Exception as e:  # a torch that does not import, no compiler: told once the library is there
            ops = e
    if force or _older(LIB, SOURCES + HEADERS):
        nvcc = nvcc_path()
        objs = []
        procs = []
        # the sources compile in parallel, each kernel whole within its file (not
        # --split-compile: its partitioning of a kernel file measured 10-20 %
        # slower, run-to-run unstable code for the fused decrypt kernel)
        for s in SOURCES:
            obj = os.path.join(CSRC, s.replace(".cu", ".o"))
            cmd = [nvcc, "-c", os.path.join(CSRC, s), "-o", obj] + flags(verbose)
            procs.append((s, subprocess.Popen(cmd, **pipes)))
            objs.append(obj)
        for s, p in procs:
            _finish(s, p, verbose)
        tmp = LIB + ".tmp"
        cmd = [nvcc, "-shared", "-o", tmp] + objs + ["-gencode", "arch=compute_100a,code=sm_100a", "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
        for o in objs:
            os.remove(o)
    if isinstance(ops, Exception):
        raise RuntimeError("torch_ops.cpp could not be compiled") from ops
    if ops is not None:
        _finish("torch_ops.cpp", ops, verbose)
        os.replace(TORCH_OPS + ".tmp", TORCH_OPS)
    elif not have_torch():
        print("torch is not installed: _torch_ops.so (provenloop_b200.adapters, .logits and .losses) was not built", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
