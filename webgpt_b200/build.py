"""Builds libwebgpt_b200.so (sm_100a only) next to this file with nvcc.

The shared library is the product's only compute path. It links the CUDA runtime statically and nothing
else, so it loads on a machine without a GPU (where every device call then reports an error).
"""
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libwebgpt_b200.so")
SOURCES = ["api.cu", "serving.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "--use_fast_math=false",
    "-Xcompiler", "-fPIC,-fvisibility=hidden,-O3", "-shared", "-cudart", "static",
]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "webgpt_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    if not force and not needs_build():
        return LIB
    flags = [f for f in NVCC_FLAGS if f not in ("--use_fast_math=false", "-shared")]
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]
        jobs = [subprocess.Popen([_nvcc()] + flags + (["-Xptxas", "-v"] if verbose else []) +
                                 ["-c", os.path.join(CSRC, s), "-o", o],
                                 stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
                for s, o in zip(SOURCES, objects)]
        said = [j.communicate()[0] for j in jobs]
        if any(j.returncode for j in jobs):
            sys.stderr.write("".join(said))
            raise RuntimeError("nvcc failed")
        res = subprocess.run([_nvcc()] + NVCC_FLAGS[:2] + ["-shared", "-cudart", "static", "-o", LIB] + objects,
                             capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed")
    if verbose:
        sys.stderr.write("".join(said))
    return LIB


if __name__ == "__main__":
    build(force=True, verbose="-v" in sys.argv)
    print(LIB)
