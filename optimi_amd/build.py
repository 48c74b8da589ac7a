"""In-tree build of the two native pieces.

* ``liboptimi_hip.so`` – the gfx950 kernels and the C ABI (hipcc, no torch), one object per ``.hip`` source.
* ``_C.*.so``          – the PyTorch-ROCm binding over that ABI (g++, host code only).

Both land next to this file so they travel with the source tree.  Run
``python -m optimi_amd.build`` to build them by hand.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
INCLUDE = os.path.join(ROOT, "include")
CSRC = os.path.join(HERE, "csrc")
LIB_PATH = os.path.join(HERE, "liboptimi_hip.so")
EXT_SUFFIX = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
BINDING_PATH = os.path.join(HERE, "_C" + EXT_SUFFIX)
ROCM_HOME = os.environ.get("ROCM_HOME", "/opt/rocm")

# -ffp-contract=off: the kernels spell out every fused multiply-add they want.
# packed-fp32-ops is switched off: hipcc must not form v_pk_*_f32 from the float code.
# -disable-vector-combine: that LLVM pass turns `pair * scalar_field` (a scalar read from the
# launch-scalars struct and splatted) into a two-float load that overlaps the next field; the
# overlapping loads then keep the optimizer from taking the struct apart, and the backend parks
# what is left of it in LDS - 768 to 1792 bytes per workgroup in every fp32 Adam, Adan and
# StableAdamW kernel, which costs a granule or two of the LDS budget that sets the occupancy
# and puts LDS reads into the element loops (fp32 AdamW over a cache-resident list: 74.5 us
# with the pass, 67.5 us without; the 16-bit kernels are unchanged within noise).
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm", "-disable-vector-combine",
]
KERNEL_SOURCES = ["optimi_hip.hip", "int8_rows.hip", "int8_gemm.hip"]
BINDING_SOURCES = ["torch_binding.cpp", "int8_binding.cpp"]


def _run(cmd: list[str]):
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"build step failed ({proc.returncode}): {' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    return proc


def _lib_commands():
    """Compile commands, link command and objects of the kernel library."""
    hipcc = shutil.which("hipcc") or os.path.join(ROCM_HOME, "bin", "hipcc")
    objs = [os.path.join(CSRC, src[:-len(".hip")] + ".hip.o") for src in KERNEL_SOURCES]
    compile_cmds = [[hipcc, *HIPCC_FLAGS, f"-I{INCLUDE}", "-c", os.path.join(CSRC, src), "-o", obj]
                    for src, obj in zip(KERNEL_SOURCES, objs)]
    return compile_cmds, [hipcc, "--offload-arch=gfx950", "-shared", *objs, "-o", LIB_PATH], objs


def _remove(paths):
    for path in paths:
        if os.path.exists(path):
            os.remove(path)


def _compile_all(cmds, verbose: bool):
    from concurrent.futures import ThreadPoolExecutor

    with ThreadPoolExecutor(max_workers=max(1, len(cmds))) as pool:
        jobs = []
        for cmd in cmds:
            if verbose:
                print(" ".join(cmd))
            jobs.append(pool.submit(_run, cmd))
        for job in jobs:
            job.result()


def _link(cmd, verbose: bool):
    if verbose:
        print(" ".join(cmd))
    _run(cmd)


def build_lib(verbose: bool = False) -> str:
    compile_cmds, link_cmd, objs = _lib_commands()
    try:
        _compile_all(compile_cmds, verbose)
        _link(link_cmd, verbose)
    finally:
        _remove(objs)
    return LIB_PATH


def _binding_commands():
    import torch
    from torch.utils import cpp_extension as ce

    inc = [f"-I{p}" for p in ce.include_paths()] + [f"-I{INCLUDE}", f"-I{ROCM_HOME}/include",
                                                     f"-I{sysconfig.get_paths()['include']}"]
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    gxx = shutil.which("g++") or "g++"
    objs = [os.path.join(CSRC, src[:-len(".cpp")] + ".o") for src in BINDING_SOURCES]
    compile_cmds = [[
        gxx, "-O2", "-std=c++17", "-fPIC", "-c", "-Wno-deprecated-declarations",
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *inc, os.path.join(CSRC, src), "-o", obj,
    ] for src, obj in zip(BINDING_SOURCES, objs)]
    link_cmd = [
        gxx, "-shared", *objs, "-o", BINDING_PATH,
        f"-L{HERE}", "-loptimi_hip", f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip",
        "-ltorch_python", f"-L{ROCM_HOME}/lib", "-lamdhip64", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}",
        f"-Wl,-rpath,{ROCM_HOME}/lib",
    ]
    return compile_cmds, link_cmd, objs


def build_binding(verbose: bool = False) -> str:
    """Compiles and links the binding; the kernel library must exist already (it is linked against)."""
    compile_cmds, link_cmd, objs = _binding_commands()
    try:
        _compile_all(compile_cmds, verbose)
        _link(link_cmd, verbose)
    finally:
        _remove(objs)
    return BINDING_PATH


def build_all(verbose: bool = False):
    """Both pieces: all translation units compile side by side, then the library is linked, then the
    binding that is linked against it."""
    lib_cmds, lib_link, lib_objs = _lib_commands()
    binding_cmds, binding_link, binding_objs = _binding_commands()
    try:
        _compile_all(lib_cmds + binding_cmds, verbose)
        _link(lib_link, verbose)
        _link(binding_link, verbose)
    finally:
        _remove(lib_objs + binding_objs)


if __name__ == "__main__":
    build_all(verbose=True)
    print("built", LIB_PATH, BINDING_PATH, file=sys.stderr)
