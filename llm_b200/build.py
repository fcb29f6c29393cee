"""Builds llm_b200/libllmb200.so with nvcc for sm_100a, and _native.abi3.so, the Python calls of its operators (in-tree, so
that they travel with the repository). The latter needs a C compiler ($CC or gcc) and the headers of Python 3.12 or later;
without them it is left out, with a note: the library and the rest of the package do not need it, KV8Cache and
logits_control raise ImportError.

    python -m llm_b200.build          # incremental
    python -m llm_b200.build --force  # rebuild everything
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libllmb200.so")
CALL = os.path.join(HERE, "_native.abi3.so")
SOURCES = ["gguf.cpp", "kernels.cu", "gemm.cu", "decode.cu", "engine.cu", "noalloc.cu", "ops.cpp", "kv8.cu", "kv8_chunk.cu", "logits.cu"]
HEADERS = ["gguf.hpp", "device.hpp", "kernels.hpp", "ops.hpp", "ptx.hpp", "kv8.hpp", "kv8_chunk.hpp", os.path.join("..", "..", "include", "llm_b200.h")]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden", "-I", os.path.join(ROOT, "include")]
# The persistent decode kernel's launch bounds still set its register budget; with this flag ptxas allocates
# 252 registers instead of 254, and config 1 decodes 0.6 % faster on a B200 (measured, same box).
SOURCE_FLAGS = {"decode.cu": ["-maxrregcount=224"]}


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "nvcc"


def _no_calls() -> str:
    """Why the Python calls of the operators cannot be built here ("": they can)."""
    cc = os.environ.get("CC", "gcc").split()
    if not cc or not shutil.which(cc[0]):
        return f"no C compiler {' '.join(cc)!r}"
    if sys.version_info < (3, 12):
        return "Python 3.12 or later is needed"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "no Python.h"
    return ""


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    hdr_mtime = max([os.path.getmtime(os.path.join(CSRC, h)) for h in HEADERS] + [os.path.getmtime(__file__)])
    objs, newest = [], 0.0
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_mtime):
            cmd = [_nvcc(), *ARCH, *FLAGS, *SOURCE_FLAGS.get(src, []), "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            subprocess.run(cmd, check=True)
        newest = max(newest, os.path.getmtime(o))
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        tmp = LIB + ".tmp"
        subprocess.run([_nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-lcudart_static", "-lrt", "-ldl", "-lpthread"],
                       check=True)
        os.replace(tmp, LIB)
    src = os.path.join(CSRC, "call.c")
    header = os.path.join(ROOT, "include", "llm_b200.h")
    why = _no_calls()
    if why:
        print(f"llm_b200: built without the Python calls of the operators: {why}", file=sys.stderr)
    elif force or not os.path.exists(CALL) or os.path.getmtime(CALL) < max(os.path.getmtime(f) for f in (src, header, __file__)):
        tmp = CALL + ".tmp"
        subprocess.run([*os.environ.get("CC", "gcc").split(), "-O2", "-std=c11", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                        "-I", sysconfig.get_paths()["include"], src, "-o", tmp, "-L", HERE, "-l:libllmb200.so",
                        "-Wl,-rpath,$ORIGIN"], check=True)
        os.replace(tmp, CALL)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
