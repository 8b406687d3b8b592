"""Build the sm_100a shared library ``minicpm_b200/_lib/libminicpm_b200.so`` in place.

    python build.py            # from this directory, or call build() from Python

One nvcc invocation per ``csrc/*.cu`` (the kernels are headers they include),
all at once, for ``-gencode arch=compute_100a,code=sm_100a`` only, then one
link with the CUDA runtime static so the library does not depend on which
libcudart the host process loaded first.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
REPO = HERE.parent
OUT = HERE / "minicpm_b200" / "_lib" / "libminicpm_b200.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted((HERE / "csrc").glob("*.cu*")) + sorted((HERE / "csrc").glob("*.h")) + [REPO / "include" / "minicpm_b200.h"]


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    mtime = OUT.stat().st_mtime
    return all(p.stat().st_mtime <= mtime for p in sources() + [Path(__file__)])


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    if not force and up_to_date():
        return OUT
    OUT.parent.mkdir(parents=True, exist_ok=True)
    tmp = OUT.with_suffix(".so.tmp")
    inc = ["-I", str(REPO / "include"), "-I", str(HERE / "csrc")]

    def run(cmd: list[str]) -> str:
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{' '.join(cmd)} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        return res.stdout + res.stderr

    def compile_one(src: Path) -> tuple[Path, str]:
        obj = OUT.parent / (src.stem + ".o")
        if not force and obj.exists() and all(p.stat().st_mtime <= obj.stat().st_mtime for p in headers + [src]):
            return obj, ""
        return obj, run([nvcc(), *NVCC_FLAGS, *(extra or []), *inc, "-c", str(src), "-o", str(obj)])

    headers = [p for p in sources() if p.suffix != ".cu"] + [Path(__file__)]
    units = [p for p in sources() if p.suffix == ".cu"]
    with ThreadPoolExecutor(max_workers=len(units)) as pool:
        done = list(pool.map(compile_one, units))
    log = "".join(text for _, text in done)
    log += run([nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-cudart", "static",
                *(str(obj) for obj, _ in done), "-o", str(tmp)])
    if verbose and log:
        print(log, flush=True)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    extra = [a for a in sys.argv[1:] if a not in ("-f", "--force", "-v")]
    build(force=True, verbose="-v" in sys.argv, extra=extra)
    print(OUT)
