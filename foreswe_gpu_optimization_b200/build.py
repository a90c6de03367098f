"""Build libgeoattn.so in-tree with nvcc for sm_100a (no torch extension machinery; plain C ABI)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libgeoattn.so")
OBJ = os.path.join(HERE, "_build")
SOURCES = ("geoattn.cu", "xattn.cu")
HEADERS = {"geoattn.cu": ("geoattn_kernels.cuh", "sm100.cuh", "tma_host.h", "host_util.h"),
           "xattn.cu": ("xattn_common.cuh", "xattn_rows.cuh", "xattn_simt.cuh", "xattn_tc.cuh", "xattn_aux.cuh", "philox.cuh",
                        "sm100.cuh", "tma_host.h", "host_util.h")}
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC"]


def nvcc():
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def _deps(src):
    return [os.path.join(CSRC, f) for f in (src,) + HEADERS[src]] + [os.path.join(HERE, "..", "include", "geoattn.h")]


def _newer(target, deps):
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= t for f in deps)


def build(force=False, verbose=False):
    """Compile csrc/*.cu (in parallel, those that changed) and link libgeoattn.so next to this file; returns the path."""
    if not force and _newer(OUT, [d for s in SOURCES for d in _deps(s)]):
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    objs, jobs = [], []
    for src in SOURCES:
        obj = os.path.join(OBJ, src[:-3] + ".o")
        objs.append(obj)
        if not force and _newer(obj, _deps(src)):
            continue
        tmp = "%s.%d" % (obj, os.getpid())
        cmd = [nvcc(), *NVCC_FLAGS, "-c", "-o", tmp, os.path.join(CSRC, src)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        jobs.append((cmd, tmp, obj, subprocess.Popen(cmd, stdout=None if verbose else subprocess.PIPE,
                                                     stderr=None if verbose else subprocess.STDOUT)))
    done = [(cmd, tmp, obj, p, p.communicate()[0]) for cmd, tmp, obj, p in jobs]
    for cmd, tmp, obj, p, out in done:
        if p.returncode:
            raise subprocess.CalledProcessError(p.returncode, cmd, output=out)
        os.replace(tmp, obj)
    tmp = "%s.%d" % (OUT, os.getpid())
    subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", tmp, *objs], check=True, capture_output=not verbose)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(force=True, verbose=True))
