"""In-tree nvcc build of libweftmoe_b200.so for sm_100a (no JIT cache, no fallback).

The reference builds its native runtime lazily with nvcc behind `weftmoe/jit.py:183-246`; here
the build is one explicit step whose output sits beside the package so that it is the file the
process loads.  `python -m weftmoe_b200.build` rebuilds; `build()` is idempotent.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
LIBRARY = PACKAGE / "libweftmoe_b200.so"
OBJECTS = PACKAGE / "build"

BINDING_SOURCE = PACKAGE / "binding" / "torch_binding.cpp"
BINDING = PACKAGE / ("_torch_binding" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
          "-Xcompiler", "-fvisibility=hidden", "-Xcompiler", "-Wall"]


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    candidate = Path(cuda_home) / "bin" / "nvcc"
    path = str(candidate) if candidate.is_file() else shutil.which("nvcc")
    if not path:
        raise RuntimeError("nvcc not found: set CUDA_HOME")
    return path


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, inputs: list[Path]) -> bool:
    if not target.is_file():
        return True
    stamp = target.stat().st_mtime_ns
    return any(p.stat().st_mtime_ns > stamp for p in inputs)


def _run(cmd, verbose=False):
    if verbose:
        print(" ".join(map(str, cmd)), flush=True)
    done = subprocess.run(cmd, capture_output=True, text=True)
    if done.returncode:
        raise RuntimeError(f"build failed:\n{' '.join(map(str, cmd))}\n{done.stdout}\n{done.stderr}")
    return done.stderr


def _binding_command(obj):
    """Host compilation of the autograd binding against the installed torch."""
    import torch
    root = Path(torch.__file__).resolve().parent / "include"
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"
    includes = [root, root / "torch/csrc/api/include", sysconfig.get_paths()["include"], cuda]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_torch_binding",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            *(f"-isystem{path}" for path in includes), "-c", str(BINDING_SOURCE), "-o", str(obj)]


def _binding_link(obj):
    import torch
    libraries = Path(torch.__file__).resolve().parent / "lib"
    return ["g++", "-shared", str(obj), "-o", str(BINDING), f"-L{libraries}", "-lc10", "-lc10_cuda", "-ltorch",
            "-ltorch_cpu", "-ltorch_python", f"-L{PACKAGE}", f"-l:{LIBRARY.name}", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile every .cu under csrc/ for sm_100a, link the shared library, and build the autograd binding on it."""
    nvcc = _nvcc()
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + \
        sorted((PACKAGE.parent / "include").glob("*.h"))
    OBJECTS.mkdir(exist_ok=True)
    binding = None
    if force or _stale(BINDING, [BINDING_SOURCE, *headers]):   # host compiler, beside the kernels
        binding = ThreadPoolExecutor(max_workers=1).submit(_run, _binding_command(OBJECTS / "torch_binding.o"), verbose)
    jobs = []
    for src in sources():
        obj = OBJECTS / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [nvcc, *ARCH_FLAGS, *COMMON, "-c", str(src), "-o", str(obj)]
            if ptxas_info:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        return _run(cmd, verbose)

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as pool:
        logs = list(pool.map(run, jobs))
    if ptxas_info:
        print("\n".join(logs))
    objects = [OBJECTS / (src.stem + ".o") for src in sources()]
    if force or jobs or _stale(LIBRARY, objects):
        run([nvcc, *ARCH_FLAGS, "-shared", "-o", str(LIBRARY), *map(str, objects),
             "-cudart", "static", "-Xcompiler", "-fPIC"])
    if binding is not None:
        binding.result()
        run(_binding_link(OBJECTS / "torch_binding.o"))
    return LIBRARY


if __name__ == "__main__":
    out = build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv)
    print(f"built {out}")
