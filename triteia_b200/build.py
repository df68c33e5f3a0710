"""Build recipe of the native library: one nvcc call, sm_100a only, output in-tree.

    python -m triteia_b200.build

produces triteia_b200/libtriteia_b200.so from triteia_b200/csrc/triteia_b200.cu (a single
translation unit; nvcc cross-compiles without a GPU) and triteia_b200/_binding.so, the Python binding
of the latency-critical operators, from triteia_b200/csrc/binding.cpp (g++ with torch's headers).
"""
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(PKG, "csrc", "triteia_b200.cu")
LIB = os.path.join(PKG, "libtriteia_b200.so")
BINDING_SRC = os.path.join(PKG, "csrc", "binding.cpp")
BINDING = os.path.join(PKG, "_binding.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
]


def sources():
    d = os.path.join(PKG, "csrc")
    return sorted(os.path.join(d, f) for f in os.listdir(d) if f.endswith((".cu", ".cuh")))


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    hdr = os.path.join(PKG, "..", "include", "triteia_b200.h")
    return any(os.path.getmtime(p) > t for p in sources() + [hdr])


def binding_tag():
    """What the extension module is built for; it holds this text.  Another Python or torch may refuse it, or crash in it."""
    import torch

    return f"triteia_b200 binding, torch {torch.__version__}, {sys.implementation.cache_tag}"


def binding_fits(path=BINDING):
    """Whether the extension module is there and built for this Python and torch."""
    try:
        with open(path, "rb") as f:
            return binding_tag().encode() + b"\0" in f.read()
    except FileNotFoundError:
        return False


def build_binding(force=False):
    """The extension module triteia_b200._binding; it finds libtriteia_b200.so next to itself."""
    hdr = os.path.join(PKG, "..", "include", "triteia_b200.h")
    if not force and binding_fits() and all(os.path.getmtime(BINDING) >= os.path.getmtime(p) for p in (BINDING_SRC, hdr)):
        return BINDING
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    cmd = (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DTRB_BINDING_TAG="{binding_tag()}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
           + [f"-I{d}" for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                                 os.path.join(cuda, "include"), sysconfig.get_paths()["include"])]
           + [BINDING_SRC, "-o", BINDING, f"-L{PKG}", "-ltriteia_b200", f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch",
              "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"])
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building _binding.so")
    return BINDING


def build(force=False, verbose=False):
    if not force and not needs_build():
        build_binding()
        return LIB
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + [SRC, "-o", LIB]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libtriteia_b200.so")
    if verbose:
        sys.stderr.write(res.stderr)
    build_binding(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
