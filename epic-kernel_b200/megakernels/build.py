"""Build libek.so and the tensor binding _ekops.so in-tree for sm_100a (nvcc, no JIT cache).

    python -m megakernels.build [--force]

The library is written next to mk_llama.py so that it travels with the source
tree and is found by `megakernels.ek`.
"""

import argparse
import os
import shutil
import subprocess
import sys
import warnings
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent.parent
CSRC = PKG_ROOT / "csrc"
OUT = PKG_ROOT / "libek.so"
BINDING = PKG_ROOT / "_ekops.so"  # ek_torch.cpp
# ek_decode.cu is compiled once per kernel variant (model x prefetch paths),
# so that each kernel carries only the code its model runs.
VARIANTS = [
    ("llama", {"EK_MODEL": 0, "EK_PF": 0}),
    ("llama_pf", {"EK_MODEL": 0, "EK_PF": 1}),
    ("mixtral", {"EK_MODEL": 1, "EK_PF": 0}),
    ("mixtral_pf", {"EK_MODEL": 1, "EK_PF": 1}),
]
# translation units compiled once
SOURCES = ["ek_capi", "ek_kvcache", "ek_prefix_attn", "ek_sample"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMPILE_FLAGS = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
LINK_FLAGS = [*ARCH, "-shared", "-cudart", "static"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def gxx_path() -> str:
    for cand in (os.environ.get("CXX"), shutil.which("g++"), shutil.which("c++")):
        if cand:
            return cand
    raise RuntimeError("g++ not found")


def binding_command(out: Path) -> list[str]:
    """Compiles the tensor binding against torch's headers. It is linked against the torch libraries that the
    process has loaded by then."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = Path(nvcc_path()).resolve().parent.parent
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], str(cuda / "include")]
    lib = Path(torch.__file__).parent / "lib"
    return [gxx_path(), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-I{i}" for i in include), "-o", str(out), str(CSRC / "ek_torch.cpp"),
            f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]


def binding_problem() -> str | None:
    """What keeps the tensor binding from being built here, or None. libek.so needs nvcc only."""
    try:
        gxx_path()
        import torch
        from torch.utils import cpp_extension  # noqa: F401
    except (RuntimeError, ImportError) as e:
        return str(e)
    return None if torch.version.cuda else "torch is built without CUDA"


def expected_registers() -> dict[int, int]:
    """Registers per thread that the warpgroups of `many_rows` share out among themselves, by kind (0: bf16, 1: int8).
    With fewer at launch they would wait for good; the launch refuses that too."""
    import re

    m = re.search(r"int REGS = I8 \? (\d+) : (\d+)", (CSRC / "ek_prefix_attn.cu").read_text())
    return {0: int(m.group(2)), 1: int(m.group(1))}


def check_registers(log: str):
    """Compares what the compiler allotted to each many_rows<D, I8> with the kernel's numbers."""
    import re

    found = re.findall(r"Compiling entry function '\S*many_rowsILi(\d+)ELb([01])E\S*'.*?Used (\d+) registers", log, re.S)
    expected = expected_registers()
    for d, i8, n in found:
        if int(n) != expected[int(i8)]:
            raise RuntimeError(f"ek_prefix_attn.cu: many_rows<{d}, {i8}> got {n} registers per thread from this compiler, "
                               f"its warpgroups count on {expected[int(i8)]}")
    if len(found) != 4:
        raise RuntimeError(f"ek_prefix_attn.cu: the compiler reported registers of {len(found)} of 4 many_rows kernels")


def _stale(target: Path, kinds: tuple[str, ...]) -> bool:
    if not target.exists():
        return True
    deps = [f for kind in kinds for f in CSRC.glob(kind)]
    deps.append(PKG_ROOT.parent / "include" / "ek.h")
    return any(d.stat().st_mtime > target.stat().st_mtime for d in deps if d.exists())


def engine_stale() -> bool:
    return _stale(OUT, ("*.cu", "*.cuh", "*.h"))


def binding_stale() -> bool:
    return _stale(BINDING, ("*.cpp",))


def build(force: bool = False, verbose: bool = False) -> Path:
    """Builds what is older than its sources. libek.so comes first: what only the binding needs may be missing (a
    warning says so), and a binding that does not compile raises with the new libek.so in place."""
    engine, binding = force or engine_stale(), force or binding_stale()
    if not engine and not binding:
        return OUT
    from concurrent.futures import ThreadPoolExecutor

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        if "-v" not in cmd:
            subprocess.run(cmd, check=True, cwd=PKG_ROOT)
            return
        done = subprocess.run(cmd, cwd=PKG_ROOT, stderr=subprocess.PIPE, text=True)
        if done.returncode:
            print(done.stderr, file=sys.stderr, flush=True)
            raise subprocess.CalledProcessError(done.returncode, cmd)
        check_registers(done.stderr)

    def build_binding():
        tmp = BINDING.with_suffix(".so.tmp")
        run(binding_command(tmp))
        tmp.replace(BINDING)

    problem = binding_problem() if binding else None
    with ThreadPoolExecutor(max_workers=len(VARIANTS) + len(SOURCES) + 1) as ex:
        bound = ex.submit(build_binding) if binding and problem is None else None
        if engine:
            nvcc = nvcc_path()
            objdir = PKG_ROOT / "_build"
            objdir.mkdir(exist_ok=True)
            jobs = []
            for name, macros in VARIANTS:
                defs = [f"-D{k}={v}" for k, v in macros.items()] + [f"-DEK_NS={name}"]
                jobs.append([nvcc, *COMPILE_FLAGS, *defs, "-c", "-o", str(objdir / f"ek_decode_{name}.o"),
                             str(CSRC / "ek_decode.cu")])
            for name in SOURCES:
                report = ["-Xptxas", "-v"] if name == "ek_prefix_attn" else []  # for check_registers
                jobs.append([nvcc, *COMPILE_FLAGS, *report, "-c", "-o", str(objdir / f"{name}.o"), str(CSRC / f"{name}.cu")])
            list(ex.map(run, jobs))
            tmp = OUT.with_suffix(".so.tmp")
            objs = [str(objdir / f"ek_decode_{n}.o") for n, _ in VARIANTS] + [str(objdir / f"{n}.o") for n in SOURCES]
            run([nvcc, *LINK_FLAGS, "-o", str(tmp), *objs])
            tmp.replace(OUT)
        if bound is not None:
            bound.result()
    if problem is not None:
        warnings.warn(f"{BINDING.name} is not built: {problem}", RuntimeWarning, stacklevel=2)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=True))
