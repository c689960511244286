"""In-tree hipcc build for the simumax_hip extension (gfx950 only).

Drives hipcc directly — no torch hipify pass, no CUDA compatibility
layer: the .hip sources are native CDNA4 code. The built .so lands next
to this file so it travels to the GPU box with the repo snapshot.
"""

import os
import subprocess
from concurrent.futures import ThreadPoolExecutor
import sys
import sysconfig

import torch
import torch.utils.cpp_extension as cpp_ext

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "simumax_hip.so")
FLAGS = os.path.join(HERE, "simumax_hip.flags")  # what OUT was built with
ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")

KERNEL_SOURCES = ["rmsnorm.hip", "rope.hip", "swiglu.hip", "cross_entropy.hip", "fp8_cast.hip",
                  "attention.hip", "mfma_probe.hip", "gemm_bench.hip",
                  "grouped_gemm.hip", "vocab.hip"]
HEADERS = ["common.h", "vocab.h"]


def _newest_mtime(paths):
    return max(os.path.getmtime(p) for p in paths if os.path.exists(p))


def _recorded_flags():
    if not os.path.exists(FLAGS):
        return None
    with open(FLAGS) as f:
        return f.read()


def build(verbose: bool = True, force: bool = False) -> str:
    sources = [os.path.join(CSRC, s) for s in KERNEL_SOURCES
               if os.path.exists(os.path.join(CSRC, s))]
    sources.append(os.path.join(CSRC, "wgrad.cpp"))
    sources.append(os.path.join(CSRC, "binding.cpp"))
    headers = [os.path.join(CSRC, h) for h in HEADERS]

    inc = [f"-I{p}" for p in cpp_ext.include_paths()]
    inc.append(f"-I{sysconfig.get_paths()['include']}")
    torch_lib = cpp_ext.library_paths()[0]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)

    common = [
        f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DHIPBLAS_V2",
        "-DHIP_ENABLE_WARP_SYNC_BUILTINS=1",
        "-DTORCH_API_INCLUDE_EXTENSION_H",
        "-DTORCH_EXTENSION_NAME=simumax_hip",
        # no packed fp32 arithmetic in device code: some of its forms are
        # not reliable on this part (the host pass warns that it does not
        # know the feature; that is harmless)
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    ]

    link_flags = [
        f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10",
        "-lc10_hip", "-ltorch_python", "-lhipblas", f"-Wl,-rpath,{torch_lib}",
    ]

    # objects of other flags are no newer for being newer than their source
    flags = "\n".join(common + inc + link_flags)
    if _recorded_flags() != flags:
        force = True
        if os.path.exists(FLAGS):
            os.remove(FLAGS)
    if (not force and os.path.exists(OUT)
            and os.path.getmtime(OUT) > _newest_mtime(sources + headers)):
        return OUT

    def compile_one(src):
        obj = os.path.join(HERE, os.path.basename(src) + ".o")
        if (not force and os.path.exists(obj)
                and os.path.getmtime(obj) > _newest_mtime([src] + headers)):
            return obj
        cmd = ["hipcc", "-c", src, "-o", obj] + common
        if src.endswith(".cpp"):
            cmd += inc
        if verbose:
            print("[simumax_hip]", " ".join(cmd[:4]), "...", flush=True)
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=8) as pool:
        objs = list(pool.map(compile_one, sources))

    link = ["hipcc", "-shared", "-o", OUT] + objs + link_flags
    if verbose:
        print("[simumax_hip] linking", OUT)
    subprocess.run(link, check=True)
    with open(FLAGS, "w") as f:
        f.write(flags)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
