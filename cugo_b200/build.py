"""Builds the native library in-tree: cugo_b200/lib/libcugo_b200.so (sm_100a only).

    python -m cugo_b200.build [--force]

The library is torch-free: CUDA sources under cugo_b200/csrc/ compiled by nvcc with
the CUDA runtime linked statically, exporting the C ABI of include/cugo_b200.h.  Beside
it cugo_b200/lib/_cugo_b200_update.so, the policy update's calls on that ABI for Python
(csrc/update_binding.cpp), compiled by the host compiler against torch; where that cannot
be (no torch with CUDA, no g++, no Python headers) the library is built all the same, and
losses.py and optim.py raise when they are called.
"""
from __future__ import annotations

import argparse
import fcntl
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from contextlib import contextmanager
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB = LIB_DIR / "libcugo_b200.so"
BINDING = LIB_DIR / "_cugo_b200_update.so"
BINDING_SOURCE = CSRC / "update_binding.cpp"

SOURCES = ["env_kernels.cu", "drivers.cu", "policy_kernels.cu", "mlp_kernels.cu", "seq_kernels.cu",
           "rollout_kernels.cu", "update_kernels.cu", "loss_kernels.cu", "optim_kernels.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--cudart", "static",
              "-Xcompiler", "-fvisibility=hidden"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the cugo_b200 native library needs the CUDA toolkit")


def _inputs() -> list[Path]:
    files = [CSRC / s for s in SOURCES]
    files += sorted(CSRC.rglob("*.cuh")) + [ROOT / "include" / "cugo_b200.h", Path(__file__)]
    return [f for f in files if f.exists()]


@contextmanager
def _alone():
    """One build at a time: ranks that start together would write the same files.  Who waited
    finds what the first one built."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    folder = os.open(LIB_DIR, os.O_RDONLY)  # the lock's holder: no file of its own
    try:
        fcntl.flock(folder, fcntl.LOCK_EX)
        yield
    finally:
        os.close(folder)


def _newer(target: Path, inputs: list[Path]) -> bool:
    return target.exists() and target.stat().st_mtime >= max(f.stat().st_mtime for f in inputs)


def up_to_date() -> bool:
    return _newer(LIB, _inputs())


def _built_for() -> str:
    """What a binding of this process has to be built against; the binding holds it as text."""
    import sysconfig

    import torch
    return f"cugo_b200 binding for torch {torch.__version__}, {sysconfig.get_config_var('SOABI')};"


def binding_fits() -> bool:
    """Whether there is a binding that was built against this process's torch and Python."""
    return BINDING.exists() and _built_for().encode() in BINDING.read_bytes()


def build_binding(force: bool = False) -> Path:
    """The Python binding of the policy update's calls; links the library beside it."""
    with _alone():
        return _build_binding(force)


def _build_binding(force: bool) -> Path:
    if not force and binding_fits() and _newer(BINDING, [BINDING_SOURCE, ROOT / "include" / "cugo_b200.h",
                                                         Path(__file__)]):
        return BINDING
    import sysconfig

    import torch
    home = Path(torch.__file__).resolve().parent
    includes = [home / "include", home / "include" / "torch" / "csrc" / "api" / "include",
                Path(nvcc()).resolve().parents[1] / "include", Path(sysconfig.get_paths()["include"])]
    out = BINDING.with_suffix(".so.tmp")
    subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                    f'-DCUGO_BUILT_FOR="{_built_for()}"',
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                    *(f"-I{p}" for p in includes), str(BINDING_SOURCE), "-o", str(out),
                    f"-L{home / 'lib'}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10",
                    "-lc10_cuda", f"-L{LIB_DIR}", "-lcugo_b200", "-Wl,-rpath,$ORIGIN"], check=True)
    out.replace(BINDING)
    return BINDING


def _try_binding(force: bool = False) -> None:
    """The binding where it can be built; the library stands without it."""
    try:
        _build_binding(force)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        print(f"cugo_b200: {BINDING.name} (the Python calls of losses.py and optim.py) was not built: {e}",
              file=sys.stderr)


def build(force: bool = False, verbose: bool = False) -> Path:
    with _alone():
        return _build(force, verbose)


def _build(force: bool, verbose: bool) -> Path:
    if not force and up_to_date():
        _try_binding()
        return LIB
    tmp = LIB_DIR / "obj"
    tmp.mkdir(exist_ok=True)

    def compile_one(src: str) -> str:
        obj = tmp / (Path(src).stem + ".o")
        cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-c", str(CSRC / src), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        return str(obj)

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    out = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH_FLAGS, "--cudart", "static", "-shared", *objs, "-o", str(out)]
    subprocess.run(cmd, check=True)
    out.replace(LIB)
    _try_binding(force)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
