"""Builds libsllm_b200.so (the CUDA engine + C ABI) in-tree with nvcc for sm_100a."""
from __future__ import annotations

import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libsllm_b200.so")
OBJ = os.path.join(HERE, "build")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-diag-suppress", "550"]


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))) + [
        os.path.join(os.path.dirname(HERE), "include", "sllm.h")]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(s) > t for s in sources())


def _object_is_new(obj: str) -> bool:
    """Whether an object is newer than all it was compiled from (its .d file lists them)."""
    try:
        t = os.path.getmtime(obj)
        with open(obj[:-2] + ".d") as f:
            deps = f.read().split(":", 1)[1].replace("\\\n", " ").split()
        return all(os.path.getmtime(d) <= t for d in deps)
    except (OSError, IndexError):
        return False


def build(force: bool = False, verbose: bool = False) -> str:
    if force or needs_build():
        nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
        env = dict(os.environ)
        env.pop("CC", None)
        env.pop("CXX", None)
        os.makedirs(OBJ, exist_ok=True)
        todo, objs = [], []
        for s in sources():
            if not s.endswith(".cu"):
                continue
            obj = os.path.join(OBJ, os.path.basename(s)[:-3] + ".o")
            objs.append(obj)
            if force or not _object_is_new(obj):
                todo.append([nvcc, *(["-Xptxas=-v"] if verbose else []), *NVCC_FLAGS, "-MD", "-MF", obj[:-2] + ".d", "-c", "-o", obj, s])
        with ThreadPoolExecutor(max(1, len(todo))) as pool:
            for _ in pool.map(lambda cmd: subprocess.run(cmd, check=True, env=env), todo):
                pass
        subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", LIB, *objs], check=True, env=env)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
