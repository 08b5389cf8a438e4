"""In-tree build of the CUDA library (sm_100a only).

    python -m orin_llm_b200.build          # -> orin_llm_b200/lib/liborin_attn_b200.so

nvcc cross-compiles without a GPU.  The CUDA runtime is linked statically so that the library
does not depend on which libcudart the host process has loaded.
"""
import contextlib
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "liborin_attn_b200.so")
SOURCES = ["capi.cu", "decode.cu", "decode_q4.cu", "kv_q4.cu", "prefill_mma.cu", "prefill_tc.cu", "rope_kv.cu"]
HEADERS = ["common.cuh", "attn_internal.h", "decode_merge.cuh", "f32x2.cuh", "kv_q4.cuh", os.path.join("..", "..", "include", "orin_attn_b200.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "--threads", "0",
]


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


HOST_LIB = os.path.join(LIBDIR, "liborin_attn_host.so")
HOST_SRC = os.path.join(HERE, "host", "kernels.cpp")


def build_host(force=False):
    """The C++ wrappers with the reference's names (host/kernels.h), linked against the C-ABI library."""
    build(force=False)
    deps = [HOST_SRC, os.path.join(HERE, "host", "kernels.h"), LIB]
    if not force and os.path.exists(HOST_LIB) and all(os.path.getmtime(d) <= os.path.getmtime(HOST_LIB) for d in deps):
        return HOST_LIB
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fno-exceptions", "-fno-rtti", "-o", HOST_LIB, HOST_SRC,
           "-L" + LIBDIR, "-lorin_attn_b200", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
    return HOST_LIB


BINDING_LIB = os.path.join(LIBDIR, "_q4_binding.so")
BINDING_SRC = os.path.join(HERE, "host", "torch_binding.cpp")


def build_binding(force=False):
    """The torch binding of the 4-bit cache's calls (host/torch_binding.cpp), linked against the C-ABI library.  Returns at once
    where the one that is there is newer than its source and header and was made for this torch and this Python."""
    import sysconfig

    import torch
    stamp = "%s %s" % (torch.__version__, sys.version.split()[0])       # it is bound to both
    stamp_file = BINDING_LIB + ".for"
    deps = [BINDING_SRC, os.path.join(HERE, "..", "include", "orin_attn_b200.h")]
    if (not force and os.path.exists(BINDING_LIB) and os.path.exists(stamp_file) and open(stamp_file).read() == stamp
            and all(os.path.getmtime(d) <= os.path.getmtime(BINDING_LIB) for d in deps if os.path.exists(d))):
        return BINDING_LIB
    if not os.path.exists(LIB):                             # (one that is there may be loaded already, and stays as it is)
        build()
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    made = "%s.%d" % (BINDING_LIB, os.getpid())             # put in place whole: another process may load or build it now
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-o", made, BINDING_SRC,
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI),
           "-isystem", os.path.join(root, "include"), "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"),
           "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           "-L" + LIBDIR, "-lorin_attn_b200", "-Wl,-rpath,$ORIGIN"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError("_q4_binding.so is missing or was built for another torch, Python or source (here: torch and Python %s), and "
                           "g++ does not run to build it: %s" % (stamp, e)) from e
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
    with contextlib.suppress(FileNotFoundError):
        os.remove(stamp_file)                               # (without one the file in between counts as stale)
    os.replace(made, BINDING_LIB)
    with open("%s.%d" % (stamp_file, os.getpid()), "w") as f:
        f.write(stamp)
    os.replace(f.name, stamp_file)
    return BINDING_LIB


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, s) for s in SOURCES + HEADERS]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    if not force and not needs_build():
        return LIB
    os.makedirs(LIBDIR, exist_ok=True)
    cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-shared", "-o", LIB]
    cmd += [os.path.join(CSRC, s) for s in SOURCES]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose:
        sys.stderr.write(r.stderr)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_host(force="--force" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
