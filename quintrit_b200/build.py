"""Builds libquintrit_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU)."""
from __future__ import annotations

import fcntl
import hashlib
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libquintrit_b200.so")
SOURCES = ["csrc/capi.cu", "csrc/paged.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


STAMP = LIB + ".srchash"  # hash of the sources the library was built from (file times do not survive every copy of the tree)


def _source_files():
    srcs = [os.path.join(HERE, "csrc", f) for f in sorted(os.listdir(os.path.join(HERE, "csrc"))) if f.endswith((".cu", ".cuh", ".hpp", ".h"))]
    inc = os.path.join(os.path.dirname(HERE), "include")
    return srcs + [os.path.join(inc, f) for f in sorted(os.listdir(inc)) if f.endswith(".h")]


def _source_hash(files=None) -> str:
    h = hashlib.sha256()
    for path in _source_files() if files is None else files:
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(NVCC_FLAGS + os.environ.get("QUINTRIT_B200_NVCC_EXTRA", "").split()).encode())
    return h.hexdigest()


def needs_build() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(STAMP):
        return True
    try:
        return open(STAMP).read().strip() != _source_hash()
    except OSError:
        return True


def _included(path: str, seen=None):
    """A source and the files of this repository that it includes, in order."""
    seen = [] if seen is None else seen
    if path not in seen and os.path.exists(path):
        seen.append(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), flags=re.M):
                _included(os.path.normpath(os.path.join(os.path.dirname(path), name)), seen)
    return seen


def _compile(source: str, force: bool, verbose: bool, extra) -> tuple:
    """One source to its object, unless the object at hand was made from the same text; returns (object, what the compiler printed)."""
    path = os.path.join(HERE, source)
    obj = path + ".o"
    stamp, want = obj + ".srchash", _source_hash(_included(path))
    if not force and os.path.exists(obj) and os.path.exists(stamp) and open(stamp).read().strip() == want:
        return obj, ""
    if os.path.exists(stamp):  # (an object that a compilation left half written, or that was written and not stamped, is nobody's)
        os.remove(stamp)
    flags = [f for f in NVCC_FLAGS if f != "-shared"]
    cmd = [_nvcc(), *(["-Xptxas", "-v"] if verbose else []), *flags, *extra, "-c", "-o", obj, path]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    with open(stamp, "w") as f:
        f.write(want)
    return obj, r.stderr


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library if its sources changed. Safe to call from several processes at once (one rank per GPU): a file lock lets one of
    them compile into a temporary file that is renamed into place; the others find the library up to date when they get the lock."""
    if not force and not needs_build():
        return LIB
    with open(os.path.join(HERE, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if force or needs_build():
                extra = os.environ.get("QUINTRIT_B200_NVCC_EXTRA", "").split()  # experiment knob, e.g. -DQTB_GEMV_DEPTH=2
                tmp = f"{LIB}.tmp.{os.getpid()}"
                with ThreadPoolExecutor(len(SOURCES)) as pool:
                    done = list(pool.map(lambda src: _compile(src, force, verbose, extra), SOURCES))
                r = subprocess.run([_nvcc(), *NVCC_FLAGS, *extra, "-o", tmp, *[obj for obj, _ in done]], capture_output=True, text=True)
                if r.returncode != 0:
                    if os.path.exists(tmp):
                        os.remove(tmp)
                    raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
                os.replace(tmp, LIB)
                with open(STAMP + ".tmp", "w") as f:
                    f.write(_source_hash())
                os.replace(STAMP + ".tmp", STAMP)
                if verbose:
                    print("".join(said for _, said in done))
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
