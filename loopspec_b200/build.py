"""Build libloopspec_engine.so in-tree for sm_100a with nvcc, and beside it the
CPython module _tensor_facts.so (host code that reads torch tensors; where torch
is installed).

    python -m loopspec_b200.build            # rebuild if any source is newer
    python -m loopspec_b200.build --force
"""

from __future__ import annotations

import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
# translation units compiled in parallel, then linked into one library
SRCS = [os.path.join(HERE, "csrc", name) for name in ("engine.cu", "serving.cu")]
OUT = os.path.join(HERE, "libloopspec_engine.so")
FACTS_SRC = os.path.join(HERE, "csrc", "tensor_facts.cpp")
FACTS_OUT = os.path.join(HERE, "_tensor_facts.so")
OBJ_DIR = os.path.join(HERE, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-diag-suppress", "177"]


def _sources():
    return glob.glob(os.path.join(HERE, "csrc", "*.cu*")) + glob.glob(os.path.join(ROOT, "include", "*.h"))


def _nvcc():
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def build(force: bool = False, verbose: bool = False) -> str:
    facts = build_facts(force)
    try:
        return build_engine(force, verbose)
    finally:
        finish_facts(facts)


def torch_root():
    """Where torch is installed (it is not imported), or None."""
    spec = importlib.util.find_spec("torch")
    return spec and os.path.dirname(spec.origin)


def facts_stamp():
    return os.path.join(OBJ_DIR, "tensor_facts.made_for")


def facts_made_for(root):
    """What the tensor module depends on besides its source: the interpreter and the torch it is compiled against."""
    with open(os.path.join(root, "version.py")) as f:
        return f"{sys.implementation.cache_tag} {root}\n{f.read()}"


def build_facts(force):
    """Start the compiler on the tensor module; None if it is newer than its source and made for this Python and
    torch, or without torch, whose tensors it reads: the library by itself needs none."""
    root = torch_root()
    if root is None:
        return None
    made_for = facts_made_for(root)
    if not force and os.path.exists(FACTS_OUT) and os.path.getmtime(FACTS_OUT) >= os.path.getmtime(FACTS_SRC):
        try:
            with open(facts_stamp()) as f:
                if f.read() == made_for:
                    return None
        except OSError:
            pass
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", *(f"-I{path}" for path in includes), "-o", FACTS_OUT + ".tmp",
           FACTS_SRC, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def finish_facts(proc):
    if proc is None:
        return
    text, _ = proc.communicate()
    if proc.returncode != 0:
        raise RuntimeError("g++ failed:\n" + text)
    os.replace(FACTS_OUT + ".tmp", FACTS_OUT)
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(facts_stamp(), "w") as f:
        f.write(facts_made_for(torch_root()))


def build_engine(force: bool, verbose: bool) -> str:
    if not force and os.path.exists(OUT):
        newest = max(os.path.getmtime(p) for p in _sources())
        if os.path.getmtime(OUT) >= newest:
            return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = _nvcc()
    jobs = []
    for src in SRCS:
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        cmd = [nvcc, *NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), "-c", "-o", obj, src]
        jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    errors = []
    for obj, proc in jobs:
        out, err = proc.communicate()
        if proc.returncode != 0:
            errors.append(out + err)
        elif verbose:
            sys.stderr.write(err)
    if errors:
        raise RuntimeError("nvcc failed:\n" + "\n".join(errors))
    tmp = OUT + ".tmp"
    res = subprocess.run([nvcc, *ARCH, "-shared", "-o", tmp, *(o for o, _ in jobs)],
                         capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc link failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
