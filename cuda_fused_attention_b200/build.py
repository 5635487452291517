"""Build recipe for the sm_100a extension library (in-tree, no JIT cache).

    python -m cuda_fused_attention_b200.build

compiles cuda_fused_attention_b200/csrc/*.cu with nvcc for sm_100a only into
cuda_fused_attention_b200/lib/libfa_sm100.so. The library exports the C ABI of
include/fa_sm100.h and include/fa_sm100_paged.h and the C++ API of include/flash_attention_sm100.h; the CUDA
runtime is linked statically and the driver is reached only through
cudaGetDriverEntryPoint, so the .so needs nothing but libc/libstdc++ and the
NVIDIA driver at run time.

The same sources compiled with FA_SM100_DEBUG_DUMP give lib/libfa_sm100_debug.so,
whose kernel also dumps its intermediate tiles for layout checks
(fa_sm100_debug_read); only tests load it.

lib/_paged.<python>-torch<version>.so is the CPython binding of the paged-cache operators for torch tensors
(csrc/paged_binding.cpp). It is the one part that is compiled against torch's headers
and needs torch at run time; the two libraries above do not, and without torch they
alone are built. Its name holds the versions that it was compiled for, so that after an
upgrade it is missing, and built again, instead of being loaded with another binary interface.
"""
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libfa_sm100.so")
DEBUG_LIB_PATH = os.path.join(LIB_DIR, "libfa_sm100_debug.so")


def binding_name():
    """File name of the binding for this Python and the installed torch."""
    try:
        torch_version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        torch_version = "unknown"
    return f"_paged.{sys.implementation.cache_tag}-torch{torch_version}.so"


BINDING_PATH = os.path.join(LIB_DIR, binding_name())
SOURCES = ["fa_sm100.cu", "fa_sm100_host.cu", "fa_sm100_api.cu", "fa_sm100_static.cu",
           "fa_sm100_plan.cu", "fa_sm100_paged.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    candidate = os.path.join(cuda_home, "bin", "nvcc")
    return candidate if os.path.exists(candidate) else (shutil.which("nvcc") or "nvcc")


def compile_command(output=LIB_PATH, extra=()):
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    return [nvcc_path(), "-std=c++17", "-O3", "-lineinfo", *ARCH_FLAGS,
            "-shared", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
            "-I", os.path.join(ROOT, "include"), "-I", CSRC,
            *extra, *srcs, "-o", output]


def binding_command(output=BINDING_PATH):
    import sysconfig
    from torch.utils import cpp_extension
    includes = [os.path.join(ROOT, "include"), *cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    return ["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-fvisibility=hidden",
            *(flag for path in includes for flag in ("-I", path)), os.path.join(CSRC, "paged_binding.cpp"),
            *(flag for path in cpp_extension.library_paths("cuda") for flag in ("-L", path)),
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-ldl", "-o", output]


def have_torch():
    return importlib.util.find_spec("torch") is not None


def needs_build():
    outputs = (LIB_PATH, DEBUG_LIB_PATH, *((BINDING_PATH,) if have_torch() else ()))
    if not all(os.path.exists(path) for path in outputs):
        return True
    lib_time = min(os.path.getmtime(path) for path in outputs)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps += [os.path.join(ROOT, "include", f) for f in os.listdir(os.path.join(ROOT, "include"))]
    return any(os.path.getmtime(d) > lib_time for d in deps)


def build(force=False, verbose=True, ptxas_verbose=False):
    """Compile the library if a source is newer than it; returns its path."""
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_verbose else []
    cmds = [compile_command(extra=extra),
            compile_command(output=DEBUG_LIB_PATH, extra=["-DFA_SM100_DEBUG_DUMP"])]
    if have_torch():
        cmds.append(binding_command())
    elif verbose:
        print("torch is not installed: the binding of the paged-cache operators is not built", flush=True)
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    failed = 0
    for proc in procs:
        out, err = proc.communicate()
        if verbose or proc.returncode != 0:
            sys.stdout.write(out)
            sys.stderr.write(err)
        failed = failed or proc.returncode
    if failed:
        raise RuntimeError(f"the compiler failed with exit code {failed}")
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, ptxas_verbose="-v" in sys.argv)
