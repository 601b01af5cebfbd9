"""Builds `libiqb200.so` in-tree with nvcc for sm_100a (no torch headers, no pybind)."""

from __future__ import annotations

import os
import shutil
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libiqb200.so")
OBJ = os.path.join(HERE, "build")
# source -> the headers it includes (beside the C ABI's)
SOURCES = {
    "kernels.cu": ("common.cuh", "stream_core.cuh", "direct.cuh", "direct_gate.cuh"),
    "attention.cu": ("common.cuh", "paged.cuh"),
    "kv_cache.cu": ("common.cuh", "paged.cuh"),
}
NVCC_FLAGS = (
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
)


def _nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found: cannot build libiqb200.so")
    return path


def _newer(target: str, deps) -> bool:
    """Whether `target` is missing or older than one of `deps`."""
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    return any(os.path.getmtime(d) > built for d in deps)


def _deps(source: str):
    return [os.path.join(CSRC, f) for f in (source, *SOURCES[source])] + \
        [os.path.join(HERE, os.pardir, "include", "iqb200.h")]


def stale() -> bool:
    return any(_newer(LIB, _deps(s)) for s in SOURCES)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if it is missing or older than its sources; returns its path.
    The sources are compiled side by side, and only those older than what they include
    (all of them with `force`)."""
    if not force and not stale():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()
    new = f".{os.getpid()}.new"                  # another process may be building too
    objects, running = [], []
    for source in SOURCES:
        obj = os.path.join(OBJ, source.replace(".cu", ".o"))
        objects.append(obj)
        if not force and not _newer(obj, _deps(source)):
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-c", "-o", obj + new, os.path.join(CSRC, source)]
        if verbose:
            cmd[1:1] = ["-Xptxas", "-v"]
        # (into a file: a pipe that fills up would hold its compiler until it is read)
        out = tempfile.TemporaryFile("w+", errors="replace")
        running.append((obj, out, subprocess.Popen(cmd, stdout=out, stderr=subprocess.STDOUT)))
    failed = []
    for obj, out, proc in running:
        proc.wait()
        out.seek(0)
        text = out.read()
        out.close()
        if proc.returncode != 0:
            failed.append(text)
            continue
        os.replace(obj + new, obj)
        if verbose:
            print(text)
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    # link beside the target and rename: a reader never sees a half-written library
    staged = LIB + new
    proc = subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", staged, *objects],
                          capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed:\n{proc.stdout}\n{proc.stderr}")
    os.replace(staged, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
