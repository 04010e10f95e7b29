"""Build libg2ptq_b200.so in-tree for sm_100a (``python -m g2ptq_b200.build``),
and the native torch binding of the operators called token by token."""

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
BINDING = os.path.join(HERE, "_lib", "_binding.so")


def _run(cmd, what, verbose):
    res = subprocess.run(cmd, stdout=None if verbose else subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout or "")
        raise RuntimeError(f"building {what} failed")


def build_binding(verbose=False):
    """Compile csrc/binding.cpp against this interpreter and this torch; skipped
    while the result is newer than its sources and made for the same torch."""
    import torch
    from torch.utils import cpp_extension
    src = os.path.join(HERE, "csrc", "binding.cpp")
    header = os.path.join(HERE, os.pardir, "include", "g2ptq_b200.h")
    made_for = f"{sys.version}\n{torch.__version__}\n"
    stamp = BINDING + ".for"
    if os.path.exists(BINDING) and os.path.exists(stamp):
        newest = max(os.path.getmtime(p) for p in (src, header))
        with open(stamp) as f:
            if os.path.getmtime(BINDING) >= newest and f.read() == made_for:
                return BINDING
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_binding",
           "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{os.path.dirname(header)}", f"-I{sysconfig.get_paths()['include']}",
           f"-I{cuda}/include"]
    cmd += [f"-I{p}" for p in cpp_extension.include_paths()]
    cmd += [src, "-o", BINDING, f"-L{lib}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
            "-ltorch_python"]
    _run(cmd, "the torch binding", verbose)
    with open(stamp, "w") as f:
        f.write(made_for)
    return BINDING


def build(jobs=None, verbose=False):
    jobs = jobs or max(1, min(16, os.cpu_count() or 1))
    _run(["make", "-C", os.path.join(HERE, "csrc"), f"-j{jobs}"], "libg2ptq_b200.so", verbose)
    try:
        build_binding(verbose)
    except (RuntimeError, OSError) as e:
        raise RuntimeError("libg2ptq_b200.so is built and runs the quantization path; its torch "
                           "binding, which the 8-bit linears and the expert routing need, is not "
                           f"(g++ and the headers of Python and torch): {e}") from e
    return os.path.join(HERE, "_lib", "libg2ptq_b200.so")


if __name__ == "__main__":
    print(build(verbose=True))
