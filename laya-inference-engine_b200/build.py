"""Build liblaya_b200.so in-tree with nvcc for sm_100a.

    python laya-inference-engine_b200/build.py [--force]

Every .cu under csrc/ is compiled to an object in _build/ (in parallel, only
when its sources changed) and linked into laya_b200/liblaya_b200.so.  nvcc
cross-compiles without a GPU.  csrc/torch_ops.cpp becomes laya_b200/_torch_ops.so
(the torch calls of laya_b200/ops.py), linked to that library, when torch is
installed; the engine itself does not need it.
"""
import argparse
import concurrent.futures as cf
import hashlib
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT = HERE / "laya_b200" / "liblaya_b200.so"
TORCH_OUT = HERE / "laya_b200" / "_torch_ops.so"
BUILD = HERE / "_build"
INCLUDE = HERE.parent / "include"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def nvcc():
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = Path(cuda) / "bin" / "nvcc"
    return str(path) if path.exists() else "nvcc"


def _digest(src):
    h = hashlib.sha256()
    h.update(" ".join(NVCC_FLAGS).encode())
    for p in sorted(list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))):
        h.update(p.read_bytes())
    h.update(src.read_bytes())
    return h.hexdigest()[:16]


def _compile(src, force):
    obj = BUILD / f"{src.stem}.o"
    stamp = BUILD / f"{src.stem}.stamp"
    dig = _digest(src)
    if not force and obj.exists() and stamp.exists() and stamp.read_text() == dig:
        return obj
    cmd = [nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stderr}")
    stamp.write_text(dig)
    return obj


def build(force=False, verbose=False):
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force), sources))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(tmp),
           *map(str, objs), "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, OUT)
    if verbose:
        print(f"built {OUT}")
    if _build_torch_ops(force) and verbose:
        print(f"built {TORCH_OUT}")
    return OUT


def _build_torch_ops(force):
    try:
        import torch
    except ImportError:
        return False
    src = CSRC / "torch_ops.cpp"
    root = Path(torch.__file__).resolve().parent
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    flags = ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
             f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", f"-I{cuda}/include",
             f"-I{sysconfig.get_paths()['include']}"]
    # the object by its path: a dependency of the name that lies beside it at run time
    link = ["-shared", f"-L{OUT.parent}", f"-l:{OUT.name}", "-Wl,-rpath,$ORIGIN", f"-L{root}/lib", "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    h = hashlib.sha256(" ".join(flags + link + [torch.__version__]).encode())
    h.update(src.read_bytes())
    h.update((INCLUDE / "laya_b200.h").read_bytes())
    stamp = BUILD / "torch_ops.stamp"
    if not force and TORCH_OUT.exists() and stamp.exists() and stamp.read_text() == h.hexdigest():
        return True
    tmp = TORCH_OUT.with_suffix(".so.tmp")
    r = subprocess.run(["g++", *flags, str(src), "-o", str(tmp), *link], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{r.stderr}")
    os.replace(tmp, TORCH_OUT)
    stamp.write_text(h.hexdigest())
    return True


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    try:
        build(force=args.force, verbose=True)
    except RuntimeError as exc:
        print(exc, file=sys.stderr)
        sys.exit(1)
