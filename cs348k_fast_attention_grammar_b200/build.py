"""Build libfa_b200.so in-tree with nvcc for sm_100a, and the torch binding.

    python -m cs348k_fast_attention_grammar_b200.build [--force] [--verbose]

The library is a plain C-ABI shared object (no torch types in its
signatures), so it is compiled by nvcc directly rather than as a torch
extension.  It links the CUDA runtime statically and needs no libcuda at link
time (tensor maps are encoded through cudaGetDriverEntryPoint).  _fa_torch*.so
is a CPython module (g++, torch's headers) that holds no kernels: the host side
of the operators whose small calls are host bound.
"""

from __future__ import annotations

import argparse
import fcntl
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_NAME = "libfa_b200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
SOURCES = ["common.cu", "attn_fwd.cu", "gemm.cu", "rotary.cu", "paged_attn.cu",
           "paged_tiles.cu"]
BINDING_SOURCE = os.path.join(CSRC, "torch_binding.cpp")
HEADERS = ["sm100_ptx.cuh", "sm100_tmem_wide.cuh", "sm100_2sm.cuh", "fa_internal.h",
           "paged.cuh", "paged_attn.h"]
PUBLIC_HEADER = os.path.join(os.path.dirname(PKG_DIR), "include", "fa_b200.h")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-shared",
              "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def _inputs():
    return ([os.path.join(CSRC, s) for s in SOURCES] +
            [os.path.join(CSRC, h) for h in HEADERS] + [PUBLIC_HEADER])


def _older(path, inputs) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(p) > t for p in inputs if os.path.exists(p))


def binding_path() -> str:
    """Where the binding for this Python and this torch lies: it holds their
    layouts through inlined code, so another version's is another file."""
    import sysconfig

    import torch
    tags = (sysconfig.get_config_var("SOABI"), "torch" + torch.__version__,
            f"abi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}")
    return os.path.join(PKG_DIR, "_fa_torch." + ".".join(map(str, tags)) + ".so")


def library_stale() -> bool:
    return _older(LIB_PATH, _inputs())


def binding_stale() -> bool:
    return _older(binding_path(), [BINDING_SOURCE, PUBLIC_HEADER])


def is_stale() -> bool:
    return library_stale() or binding_stale()


def _library_command(verbose: bool) -> list:
    cmd = [nvcc_path()] + ARCH_FLAGS + NVCC_FLAGS + ["--threads", "0"]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    return cmd + [os.path.join(CSRC, s) for s in SOURCES]


def _binding_command() -> list:
    import sysconfig

    import torch
    root = os.path.join(os.path.dirname(torch.__file__))
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path()))), "include")
    return ([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(root, "include"),
             "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
             "-I" + cuda, BINDING_SOURCE, "-L" + os.path.join(root, "lib"), "-ltorch_python",
             "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-lc10", "-lc10_cuda"])


def build(force: bool = False, verbose: bool = False, library: bool = True,
          binding: bool = True) -> str:
    """Compile the library and the binding (or one of them) if they are missing
    or older than their sources; returns the library's path.  Neither needs the
    other: the library loads where there is no g++ or no torch to build the
    binding against.

    Safe when several processes (the ranks of one job) call it at once: an
    exclusive lock on a file beside the library lets one of them compile, the
    others wait and then find the library fresh; each compile writes its own
    temporary file and renames it over the library atomically."""
    def wanted():
        return (library and (force or library_stale()), binding and (force or binding_stale()))

    if not any(wanted()):
        return LIB_PATH
    with open(LIB_PATH + ".lock", "a+") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            jobs = []
            want_library, want_binding = wanted()
            if want_library:
                jobs.append((LIB_PATH, _library_command(verbose)))
            if want_binding:
                jobs.append((binding_path(), _binding_command()))
            running, failed = [], []
            for path, cmd in jobs:
                tmp = f"{path}.{os.getpid()}.tmp"
                cmd = cmd + ["-o", tmp]
                if verbose:
                    print(" ".join(cmd), file=sys.stderr)
                try:
                    running.append((path, tmp, cmd[0], subprocess.Popen(
                        cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
                except OSError as e:                # (the others end before this is raised)
                    failed.append(f"{os.path.basename(cmd[0])} cannot be run: {e}")
            for path, tmp, tool, proc in running:
                out, _ = proc.communicate()
                if verbose or proc.returncode != 0:
                    sys.stderr.write(out)
                if proc.returncode != 0:
                    if os.path.exists(tmp):
                        os.unlink(tmp)
                    failed.append(f"{os.path.basename(tool)} failed with exit code "
                                  f"{proc.returncode}")
                else:
                    os.replace(tmp, path)
            if failed:
                raise RuntimeError("; ".join(failed))
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
