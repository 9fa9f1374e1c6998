"""Build step for the CUDA bridge: nvcc -> rustane_b200/libcudabridge.so (in tree).

The library is compiled for sm_100a only (B200). nvcc cross-compiles without a
GPU, so this runs on any machine with CUDA 12.9.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libcudabridge.so"
OBJ_DIR = PKG / "build"
SOURCES = [CSRC / "bridge.cu", CSRC / "paged.cu"]
HEADERS = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [ROOT / "include" / "cuda_bridge.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def nccl_dirs():
    """(include dir, library file) of the NCCL that ships with torch, if present."""
    try:
        import nvidia.nccl  # namespace package from the nvidia-nccl wheel
        base = Path(list(nvidia.nccl.__path__)[0])
    except Exception:
        return None, None
    inc, lib = base / "include", base / "lib" / "libnccl.so.2"
    return (inc if (inc / "nccl.h").exists() else None), (lib if lib.exists() else None)


def nvcc_path() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    p = Path(cuda) / "bin" / "nvcc"
    return str(p) if p.exists() else "nvcc"


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in SOURCES + HEADERS if p.exists())


def _object_is_current(obj: Path, cmd: str) -> bool:
    """Whether an object is newer than everything its last compile read (nvcc's own list,
    -MD) and was made by the same command."""
    deps, made_by = obj.with_suffix(".d"), obj.with_suffix(".cmd")
    if not (obj.exists() and deps.exists() and made_by.exists()) or made_by.read_text() != cmd:
        return False
    files = deps.read_text().replace("\\\n", " ").split(":", 1)[1].split()
    t = obj.stat().st_mtime
    return all(os.path.exists(f) and os.stat(f).st_mtime <= t for f in files)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    inc, nccl_lib = nccl_dirs()
    if inc is None:
        raise RuntimeError("nccl.h not found (the nvidia-nccl wheel provides it)")
    extra = [f"-I{inc}"]
    if nccl_lib is not None:
        extra.append(f'-DCB_NCCL_DEFAULT_PATH="{nccl_lib}"')
    OBJ_DIR.mkdir(exist_ok=True)
    running = []
    for src in SOURCES:  # the sources compile side by side
        obj = OBJ_DIR / (src.stem + ".o")
        cmd = [nvcc_path(), *NVCC_FLAGS, f"-I{ROOT / 'include'}", f"-I{CSRC}", *extra,
               "-MD", "-MF", str(obj.with_suffix(".d")), "-c", "-o", str(obj), str(src)]
        line = " ".join(cmd)
        if not force and _object_is_current(obj, line):
            continue
        if verbose:
            print(line, file=sys.stderr)
        obj.unlink(missing_ok=True)
        running.append((obj, line, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                                    stderr=subprocess.STDOUT, text=True)))
    failed = []
    for obj, line, p in running:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"nvcc failed ({p.returncode}):\n{out}")
        else:
            obj.with_suffix(".cmd").write_text(line)
    if failed:
        raise RuntimeError("\n".join(failed))
    cmd = [nvcc_path(), *NVCC_FLAGS, "-shared", "-o", str(LIB),
           *(str(OBJ_DIR / (s.stem + ".o")) for s in SOURCES), "-ldl", "-lpthread"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
