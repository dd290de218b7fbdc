"""Build libasca_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU).

    python -m asca_b200.build [--force] [--verbose]

asca_b200/_torch_ops.so, the binding of asca_b200.ops to torch tensors (csrc/torch_ops.cpp), is built beside it with g++
against the torch of this interpreter.

Each .cu under csrc/ is compiled to an object in csrc/build/ (skipped when newer than the
source and the headers), then linked into asca_b200/libasca_b200.so with the static CUDA
runtime, so loading the library needs no CUDA installation beyond the driver.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = CSRC / "build"
SO = PKG / "libasca_b200.so"
TORCH_OPS = PKG / "_torch_ops.so"
INCLUDE = PKG.parent / "include"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-I", str(INCLUDE),
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found; libasca_b200.so cannot be built")
    return exe


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    OBJ.mkdir(exist_ok=True)
    jobs = []
    for src in sources:
        obj = OBJ / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {cmd[-3]}")
    objs = [OBJ / (s.stem + ".o") for s in sources]
    if force or jobs or _stale(SO, objs):
        cmd = [nvcc(), "-shared", "-o", str(SO), *map(str, objs), "-cudart", "static",
               "-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return SO


def build_torch_ops(force: bool = False) -> Path | None:
    """The binding of asca_b200.ops (the library itself has been built), or None where torch is not installed, which nothing else
    needs. Torch's own libraries are in the process when it is loaded; libasca_b200.so is found beside it. It names the torch and the
    interpreter that it was built for, and is built again for others."""
    import importlib.util
    import sysconfig

    src = CSRC / "torch_ops.cpp"
    spec = importlib.util.find_spec("torch")
    if spec is None:
        sys.stderr.write("torch is not installed: asca_b200/_torch_ops.so is not built\n")
        return None
    import torch as installed

    torch = Path(spec.origin).parent
    built_for = f"torch {installed.__version__}, {sysconfig.get_config_var('SOABI')}"
    if not force and not _stale(TORCH_OPS, [src, *sorted(INCLUDE.glob("*.h"))]) and built_for.encode() in TORCH_OPS.read_bytes():
        return TORCH_OPS
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(installed.compiled_with_cxx11_abi())}", f'-DASCA_BUILT_FOR="{built_for}"',
           "-I", sysconfig.get_paths()["include"], "-I", str(torch / "include"), "-I", str(torch / "include/torch/csrc/api/include"),
           "-I", str(cuda / "include"), str(src), "-o", str(TORCH_OPS), "-L", str(PKG), f"-l:{SO.name}", "-L", str(torch / "lib"),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        raise RuntimeError("g++ failed on torch_ops.cpp")
    return TORCH_OPS


if __name__ == "__main__":
    out = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    build_torch_ops(force="--force" in sys.argv)
    print(out)
