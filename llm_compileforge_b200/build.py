"""Build libsfb.so (the CUDA kernels + C ABI) in-tree for sm_100a.

    python -m llm_compileforge_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU.  Each ``csrc/*.cu`` becomes an object under
``csrc/_obj`` (rebuilt only when it or a header changed) and the objects are
linked, with the static CUDA runtime, into ``llm_compileforge_b200/libsfb.so``.
``csrc/calls.cpp`` becomes the extension module ``_calls`` beside it (host code
against PyTorch's headers: the quick way from Python into the library).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(CSRC, "_obj")
LIB = os.path.join(PKG, "libsfb.so")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def _headers_mtime() -> float:
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    paths += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return max(os.path.getmtime(p) for p in paths)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile and link.  ``SFB_NVCC_FLAGS`` adds compiler flags and ``SFB_LIB_OUT`` writes such a variant to another path
    (objects beside it), leaving the regular library alone."""
    global OBJ, LIB
    extra = os.environ.get("SFB_NVCC_FLAGS", "").split()
    if os.environ.get("SFB_LIB_OUT"):
        LIB = os.path.abspath(os.environ["SFB_LIB_OUT"])
        OBJ = LIB + "_obj"
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))
    hdr = _headers_mtime()
    jobs = []
    for src in sources:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src[:-3] + ".o")
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            cmd = [nvcc, *NVCC_FLAGS, *extra, "-I", INCLUDE, "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd: list[str]) -> None:
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode:
            sys.stderr.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
        if res.returncode:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed for {cmd[-3]}")

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as pool:
        list(pool.map(run, jobs))
    objs = [os.path.join(OBJ, s[:-3] + ".o") for s in sources]
    if jobs or force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        cmd = [nvcc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static"]
        run(cmd)
    if not os.environ.get("SFB_LIB_OUT"):
        build_calls(force, run)
    return LIB


def calls_path() -> str:
    return os.path.join(PKG, "_calls" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_calls(force: bool, run) -> None:
    """The extension module, for the torch that is installed: it is built again when that changes.  Where torch, its or Python's
    headers or a C++ compiler are missing there is none, and the library, which needs none of them, stands by itself."""
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError as e:
        sys.stderr.write(f"no extension module _calls: torch does not import ({e})\n")
        return
    src, out, note = os.path.join(CSRC, "calls.cpp"), calls_path(), os.path.join(OBJ, "_calls.torch")
    built_for = None
    if os.path.exists(out) and os.path.exists(note):
        with open(note) as f:
            built_for = f.read()
    if not force and built_for == torch.__version__ and os.path.getmtime(out) >= max(os.path.getmtime(src), _headers_mtime()):
        return
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    missing = [h for h in ("torch/csrc/autograd/python_variable.h", "Python.h") if not any(os.path.exists(os.path.join(d, h)) for d in include)]
    if missing or not shutil.which("g++"):
        sys.stderr.write(f"no extension module _calls: {f'headers missing ({missing[0]})' if missing else 'no g++'}\n")
        if os.path.exists(out):
            os.remove(out)  # of another torch, or older than its sources
        return
    run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         f'-DSFB_TORCH_VERSION="{torch.__version__}"',
         *(f"-I{d}" for d in include), src, "-o", out, *(f"-L{d}" for d in cpp_extension.library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"])
    with open(note, "w") as f:
        f.write(torch.__version__)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
