"""Build the in-tree CUDA library for sm_100a with nvcc.

``libflashhog_b200.so`` -- the kernels and the C ABI declared in
``include/flash_hog_b200.h`` -- is written next to this file so it travels with
the source tree, and so is ``_torch_ops.so``, the autograd nodes of dense
attention and of ``fused``'s embedding, dropout and policy loss over that ABI
(``csrc/torch_ops.cpp``). Object files are cached under ``_build/`` keyed by source and
header modification times, so an unchanged tree rebuilds in seconds; the nodes are also
built again beside another torch or Python than theirs.
"""

from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
ROOT = os.path.dirname(PKG)
BUILD_DIR = os.path.join(ROOT, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
              "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]

MAIN_SOURCES = ["capi.cu", "fwd.cu", "fwd_few.cu", "bwd.cu", "bwdbwd.cu", "sink_join.cu", "rowdot.cu", "f32.cu",
                "ln_gelu.cu", "xent.cu", "embed.cu", "dropout.cu", "policy.cu"]

MAIN_LIB = os.path.join(PKG, "libflashhog_b200.so")
TORCH_OPS_SOURCE = os.path.join(CSRC, "torch_ops.cpp")
TORCH_OPS_LIB = os.path.join(PKG, "_torch_ops.so")


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build flash_hog_b200")


def _headers_mtime() -> float:
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    inc = os.path.join(ROOT, "include")
    paths += [os.path.join(inc, f) for f in os.listdir(inc) if f.endswith(".h")]
    return max(os.path.getmtime(p) for p in paths)


def _compile(src: str, verbose: bool) -> str:
    os.makedirs(BUILD_DIR, exist_ok=True)
    path = os.path.join(CSRC, src)
    obj = os.path.join(BUILD_DIR, src.replace(".cu", ".o"))
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(path), _headers_mtime()):
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", path, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        print(res.stderr, file=sys.stderr)
    return obj


def _link(objs, out):
    cmd = [nvcc(), *ARCH, "-shared", "-o", out, *objs]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of {os.path.basename(out)} failed:\n{res.stdout}\n{res.stderr}")


def _torch_ops_origin() -> str:
    """What the nodes' library is built for: it loads beside this torch and Python alone."""
    return "\n".join([sys.version, importlib.metadata.version("torch"), importlib.util.find_spec("torch").origin])


def build_torch_ops() -> None:
    """Compile ``csrc/torch_ops.cpp`` against torch's headers (host code only), where the
    library is older than its sources or was built for another torch or Python."""
    header = os.path.join(ROOT, "include", "flash_hog_b200.h")
    stamp, origin = os.path.join(BUILD_DIR, "torch_ops.origin"), _torch_ops_origin()
    if os.path.exists(TORCH_OPS_LIB) and os.path.exists(stamp):
        with open(stamp) as f:
            same = f.read() == origin
        if same and os.path.getmtime(TORCH_OPS_LIB) >= max(os.path.getmtime(TORCH_OPS_SOURCE),
                                                           os.path.getmtime(header)):
            return
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    os.makedirs(BUILD_DIR, exist_ok=True)
    if os.path.exists(stamp):  # until the build has ended
        os.remove(stamp)
    includes = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"], os.path.dirname(header)]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *["-isystem" + i for i in includes],
           TORCH_OPS_SOURCE, "-o", TORCH_OPS_LIB, *["-L" + p for p in cpp_extension.library_paths("cuda")],
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on torch_ops.cpp:\n{res.stdout}\n{res.stderr}")
    with open(stamp, "w") as f:
        f.write(origin)


def build(verbose: bool = False) -> None:
    """Compile every CUDA source of the library for sm_100a and link it; then the torch nodes."""
    srcs = MAIN_SOURCES
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        torch_ops = ex.submit(build_torch_ops)
        objs = dict(zip(srcs, ex.map(lambda s: _compile(s, verbose), srcs)))
        torch_ops.result()
    _link([objs[s] for s in MAIN_SOURCES], MAIN_LIB)


XLA_FFI_SOURCE = os.path.join(CSRC, "xla_ffi.cc")
XLA_FFI_LIB = os.path.join(PKG, "libfh_xla_ffi.so")


def xla_ffi_include_dir():
    """jaxlib's FFI header directory, or None where JAX is not installed (this image)."""
    try:
        import jax.ffi

        return jax.ffi.include_dir()
    except Exception:  # noqa: BLE001 - any failure means the headers are not available
        return None


def build_xla_ffi():
    """Compiles ``csrc/xla_ffi.cc`` (the XLA FFI handlers FhAttnFwd, FhAttnBwd, FhBwdBwd,
    FhBwdBwdO) into ``libfh_xla_ffi.so``, linked against ``libflashhog_b200.so``.
    Returns the library path, or None without building where jaxlib's FFI headers are
    absent -- as on this image, where the handlers are therefore not built."""
    inc = xla_ffi_include_dir()
    if inc is None:
        return None
    build()
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-x", "cu", "-shared", "-I" + inc, XLA_FFI_SOURCE, "-o", XLA_FFI_LIB,
           "-L" + PKG, "-lflashhog_b200", "-Xlinker", "-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on xla_ffi.cc:\n{res.stdout}\n{res.stderr}")
    return XLA_FFI_LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv)
    print("built", MAIN_LIB)
    ffi_lib = build_xla_ffi()
    print("built", ffi_lib) if ffi_lib else print("XLA FFI handlers not built: jaxlib's FFI headers are absent")
