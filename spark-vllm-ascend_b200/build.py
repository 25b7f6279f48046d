"""Build the sm_100a CUDA library of the Spark B200 decode path.

    python spark-vllm-ascend_b200/build.py          # -> spark_b200/_lib/libspark_b200.so

The library is a plain C-ABI shared object (include/spark_b200.h); it has no
torch dependency.  nvcc cross-compiles without a GPU.  The sources are compiled side by
side; one whose object is newer than all it includes is not compiled again.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
OUT_DIR = HERE / "spark_b200" / "_lib"
OBJ_DIR = HERE / "_build"
LIB = OUT_DIR / "libspark_b200.so"
SOURCES = [CSRC / "spark_b200.cu", CSRC / "paged.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-I", str(ROOT / "include"), "-I", str(CSRC),
]


def _stale() -> bool:
    if not LIB.exists():
        return True
    mtime = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))
    return any(p.stat().st_mtime > mtime for p in deps)


def _object(src: Path) -> Path:
    return OBJ_DIR / (src.stem + ".o")


def _stale_object(src: Path) -> bool:
    """The object is missing, or older than a file of this tree that its compilation read."""
    obj, dep = _object(src), _object(src).with_suffix(".d")
    if not obj.exists() or not dep.exists():
        return True
    files = dep.read_text().replace("\\\n", " ").split(":", 1)[-1].split()
    mine = [Path(f) for f in files if f.startswith(str(ROOT))]
    return not mine or any(not p.exists() or p.stat().st_mtime > obj.stat().st_mtime for p in mine)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    jobs = []
    for src in SOURCES:
        if not force and not _stale_object(src):
            continue
        obj = _object(src)
        tmp = obj.with_suffix(".o.tmp")
        cmd = [NVCC, *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-MD", "-MF", str(obj.with_suffix(".d")),
               "-c", str(src), "-o", str(tmp)]
        jobs.append((cmd, tmp, obj, subprocess.Popen(cmd)))
    codes = [p.wait() for _, _, _, p in jobs]  # every compilation ends before one is reported
    for (cmd, tmp, obj, _), rc in zip(jobs, codes):
        if rc:
            raise subprocess.CalledProcessError(rc, cmd)
        os.replace(tmp, obj)
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler", "-fPIC", "-shared",
                    *(str(_object(s)) for s in SOURCES), "-o", str(tmp)], check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
