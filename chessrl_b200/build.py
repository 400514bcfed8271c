"""Builds libchessrl_b200.so (hand-written sm_100a CUDA + the C ABI) in-tree with nvcc, and _serving.so, the module that
hands torch tensors to its serving entry points, with g++.

    python -m chessrl_b200.build [--force]

nvcc cross-compiles without a GPU. The libraries sit next to this file so that they travel with the
source tree; nothing is installed into site-packages.
"""
import os
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libchessrl_b200.so")
SERVING = os.path.join(HERE, "_serving.so")
SOURCES = ["engine.cu", "serving.cu", "chess.cpp"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def _newest_source_mtime():
    newest = 0.0
    for root in (CSRC, os.path.join(os.path.dirname(HERE), "include")):
        for name in os.listdir(root):
            newest = max(newest, os.path.getmtime(os.path.join(root, name)))
    return newest


def _serving_command():
    import torch
    root = os.path.join(os.path.dirname(torch.__file__))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    for path in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                 sysconfig.get_paths()["include"], os.path.join(cuda, "include")):
        cmd += ["-isystem", path]
    return cmd + ["-o", SERVING, os.path.join(CSRC, "serving_torch.cpp"), "-L" + os.path.join(root, "lib"), "-ltorch_python",
                  "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def _run(commands, verbose):
    """Run the commands side by side; raises with the output of the first that fails."""
    running = [(cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)) for cmd in commands]
    outputs = [(cmd, proc.communicate()[0], proc.returncode) for cmd, proc in running]
    for cmd, out, code in outputs:
        if code != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n{out}")
        if verbose:
            print(out)


def build(force=False, verbose=False):
    """Compile what is missing or older than any source; returns the library's path."""
    newest = _newest_source_mtime()
    stale = [path for path in (LIB, SERVING) if force or not os.path.exists(path) or os.path.getmtime(path) < newest]
    nvcc = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")] + NVCC_FLAGS
    with tempfile.TemporaryDirectory() as scratch:
        commands, objects = [], []
        if LIB in stale:
            for name in SOURCES:
                objects.append(os.path.join(scratch, name + ".o"))
                commands.append(nvcc + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", objects[-1], os.path.join(CSRC, name)])
        if SERVING in stale:
            commands.append(_serving_command())
        _run(commands, verbose)
        if objects:
            _run([nvcc + ["-shared", "-o", LIB] + objects], verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
