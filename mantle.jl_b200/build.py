"""Build libmantle_cuda.so in-tree for sm_100a.

    python mantle.jl_b200/build.py            # incremental
    python mantle.jl_b200/build.py --force    # rebuild everything

Every translation unit is compiled by nvcc with
`-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`, then linked into one
shared library with the CUDA runtime linked statically, so the library does not
depend on which libcudart another package in the process loaded.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
OUT = HERE / "mantle_cuda" / "libmantle_cuda.so"
OBJ = HERE / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(ROOT / "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")) + list(CSRC.glob("kernels/*.cu")))


def headers() -> list[Path]:
    return sorted(list(CSRC.rglob("*.hpp")) + list(CSRC.rglob("*.cuh")) + [ROOT / "include" / "mantle_cuda.h"])


# Flags for single translation units. showcase.cu and mesh_raster.cu: no FMA
# contraction, so their float arithmetic is the sequence of IEEE operations the
# C oracle performs.
PER_FILE = {"showcase.cu": ["-fmad=false"], "mesh_raster.cu": ["-fmad=false"]}


def compile_one(src: Path, force: bool) -> Path:
    obj = OBJ / (src.relative_to(CSRC).as_posix().replace("/", "__") + ".o")
    newest_dep = max([src.stat().st_mtime] + [h.stat().st_mtime for h in headers()])
    if not force and obj.exists() and obj.stat().st_mtime >= newest_dep:
        return obj
    cmd = [nvcc(), *ARCH, *COMMON, *PER_FILE.get(src.name, []), "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd = [nvcc(), *COMMON, "-x", "c++", "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


LAUNCH_SRC = CSRC / "python" / "launch.cpp"
LAUNCH_OUT = HERE / "mantle_cuda" / f"_launch{sysconfig.get_config_var('EXT_SUFFIX')}"  # this Python's alone


def build_launch(force: bool = False) -> None:
    """The Python host's short way to a launch with torch tensors (mantle_cuda/_launch),
    against the torch that is installed, and again when another is. The library does
    without: where this cannot be built, launches take the long way."""
    found = importlib.util.find_spec("torch")
    if found is None or not found.origin:  # no torch, or what is left of one
        return
    home, stamp = Path(found.origin).parent, OBJ / "launch.stamp"
    version = home / "version.py"
    built_for = f"{sys.version}\n{home}\n{version.read_text() if version.exists() else ''}"
    newest_dep = max(f.stat().st_mtime for f in (LAUNCH_SRC, ROOT / "include" / "mantle_cuda.h", Path(__file__)))
    if (not force and LAUNCH_OUT.exists() and LAUNCH_OUT.stat().st_mtime >= newest_dep
            and stamp.exists() and stamp.read_text() == built_for):
        return
    for old in (LAUNCH_OUT, LAUNCH_OUT.with_name("_launch.so"), stamp):  # built for something else: never loaded again
        old.unlink(missing_ok=True)
    try:
        import torch
        from torch.utils.cpp_extension import include_paths

        if not torch.version.cuda:
            return
        cuda = Path(nvcc()).resolve().parent.parent / "include"
        cmd = ["g++", "-O2", "-std=c++20", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               f'-DBUILT_FOR_TORCH="{torch.__version__}"',
               *[f"-I{d}" for d in (*include_paths(), sysconfig.get_paths()["include"], cuda)], str(LAUNCH_SRC), "-o", str(LAUNCH_OUT),
               f"-L{home / 'lib'}", f"-Wl,-rpath,{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        why = f"{' '.join(cmd)}\n{r.stdout}\n{r.stderr}" if r.returncode else ""
    except (ImportError, OSError) as e:  # a torch that does not load, no g++
        why = str(e)
    if why:
        LAUNCH_OUT.unlink(missing_ok=True)
        print(f"mantle_cuda/_launch was not built; launches with torch tensors cost the host more without it: {why}", file=sys.stderr)
        return
    stamp.write_text(built_for)


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: compile_one(s, force), srcs))
    newest = max(o.stat().st_mtime for o in objs)
    if force or not OUT.exists() or OUT.stat().st_mtime < newest:
        # --no-undefined: a symbol missing from the library fails the build, not the first load
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-Xlinker", "--no-undefined", "-o", str(OUT),
               *map(str, objs), "-ldl", "-lpthread", "-lrt"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    build_launch(force)
    if verbose:
        print(OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    try:
        build(force=args.force, verbose=True)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
