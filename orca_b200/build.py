"""Builds liborca_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and _rows.so (calls of it on tensors) with g++."""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liborca_b200.so")
ROWS = os.path.join(HERE, "_rows.so")      # a Python module: csrc/torch_rows.cpp
SOURCES = ["sampler.cu", "attention.cu", "gemm.cu", "state.cu", "pipeline.cu", "planner.cu", "planner_mrd.cu", "planner_lists.cu", "planner_rand.cu", "csr_build.cu", "tc_gemm.cu", "context.cu", "metrics.cu", "group.cu", "chain.cu", "attn_query.cu", "attn_out.cu", "gru_rows.cu", "score_rows.cu", "packed.cu", "lookup.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]


def _older(target, sources):
    return not os.path.exists(target) or any(os.path.getmtime(d) > os.path.getmtime(target) for d in sources)


def _sources(of_module):
    """What the module is made of (of_module), or the library."""
    mine = [f for f in os.listdir(CSRC) if f.endswith(".cpp") == of_module]
    return [os.path.join(CSRC, f) for f in mine] + [os.path.join(os.path.dirname(HERE), "include", "orca_b200.h")]


def rows_made_for():
    """What the module derives from beside its source, as it stands in a module that was built: PyTorch, Python and the library's
    interface (its nodes are PyTorch's classes, whose layout another version may change)."""
    import torch
    from . import _lib
    return f"orca_b200._rows of PyTorch {torch.__version__}, Python {sysconfig.get_config_var('SOABI')}, interface {_lib.VERSION}"


def rows_fit():
    """Whether the module is there and was built for what runs here."""
    if not os.path.exists(ROWS):
        return False
    with open(ROWS, "rb") as f:
        return rows_made_for().encode() + b"\0" in f.read()


def _rows_command():
    import torch
    at = os.path.dirname(torch.__file__)
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    include = [os.path.join(at, "include"), os.path.join(at, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include")]
    # (torch's libraries are found by their names, for they are loaded already; this one's beside it)
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DORCA_ROWS_MADE_FOR="{rows_made_for()}"', *[x for i in include for x in ("-isystem", i)],
            os.path.join(CSRC, "torch_rows.cpp"), "-o", ROWS, "-L" + os.path.join(at, "lib"),
            *["-l" + n for n in ("torch_python", "torch", "torch_cpu", "torch_cuda", "c10", "c10_cuda")],
            "-L" + HERE, "-l:liborca_b200.so", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds what is out of date and returns the library.  The module is a step of its own behind it, for which g++ and PyTorch's headers are
    needed: without them the library is whole, and who uses the module is told (orca_b200._lib.rows)."""
    if force or _older(LIB, _sources(False)):
        _build_library(verbose)
    try:
        if force or _older(ROWS, _sources(True)) or not rows_fit():
            _build_rows()
    except Exception as e:
        if os.path.exists(ROWS):
            os.remove(ROWS)      # (of an earlier source)
        sys.stderr.write(f"orca_b200/_rows.so (rows in 4 bits and lookups on PyTorch's tensors) could not be built, the library is: {e}\n")
    return LIB


def _build_rows():
    made = ROWS + ".new"
    r = subprocess.run([made if a == ROWS else a for a in _rows_command()], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed\n{r.stdout}")
    os.replace(made, ROWS)


def _build_library(verbose):
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in SOURCES:
        obj = os.path.join(HERE, "build", src.replace(".cu", ".o"))
        objs.append(obj)
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed = True
            sys.stderr.write(f"--- nvcc failed on {src}\n{out}\n")
        elif verbose or out.strip():
            sys.stderr.write(f"--- {src}\n{out}\n")
    if failed:
        raise RuntimeError("nvcc failed")
    subprocess.check_call([nvcc, "-shared", "-o", LIB, *objs, "-lcudart"])


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
