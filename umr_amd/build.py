"""Build libumr_hip.so (hipcc, gfx950 only) in-tree, umr_amd/lib/libumr_hip.so, and libumr_torch.so beside it: the PyTorch operators
of include/umr_nn.h (csrc/torch_nn.cpp, host code).

`python -m umr_amd.build` or umr_amd.build.build().  The .so is git-ignored but travels with the
gpurun snapshot, so the GPU box uses the prebuilt library (hipcc is present there too).
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libumr_hip.so")
TORCH_LIB = os.path.join(LIBDIR, "libumr_torch.so")
SOURCES = ["raster.hip", "geometry.hip", "losses.hip", "perceptual.hip", "edt.hip", "atlas.hip", "regs.hip", "eval.hip"]
NN_SOURCES = ["linear.hip", "linear_f32.hip", "linear_bf16.hip", "linear_f16.hip", "balance.hip"]     # include/umr_nn.h
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC", "-shared",
         "-munsafe-fp-atomics",   # native global_atomic_add_f32 instead of CAS loops
         "-ffp-contract=off",     # branch-deciding expressions round like the reference's float code
         "-fno-slp-vectorize",    # no pairing of scalar float code
         # No packed fp32 instructions: some forms of v_pk_{add,mul,fma}_f32 have given wrong results on this target now and then, and
         # the compiler makes them from float2 code.  Two scalar operations give the same bits; the render-and-compare step
         # takes the same time (2.83 ms with and without).
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall", "-Wno-unused-function", "-Wno-bitwise-instead-of-logical"]


def _dep_files():
    return sorted([os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".h", ".cpp"))] +
                  [os.path.normpath(os.path.join(HERE, "..", "include", f)) for f in ("umr_hip.h", "umr_nn.h")])


def source_hash():
    """sha256 over the kernel sources + the C-ABI headers (file names and contents).  The build embeds it in the library
    (umr_build_id()); tests compare the two, so a stale .so is detected wherever the tests run -- file times do not
    survive the copy to the GPU box, contents do."""
    import hashlib
    h = hashlib.sha256()
    for f in _dep_files():
        h.update(os.path.basename(f).encode() + b"\0")
        h.update(open(f, "rb").read())
    return h.hexdigest()[:32]


def _stale():
    if not os.path.exists(LIB) or not os.path.exists(TORCH_LIB):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(TORCH_LIB))
    return any(os.path.getmtime(d) > t for d in _dep_files() + [os.path.abspath(__file__)])


def torch_command(hash_flag):
    """libumr_torch.so: host code against this PyTorch, linked to libumr_hip.so beside it."""
    import torch
    from torch.utils.cpp_extension import include_paths
    tl = os.path.join(os.path.dirname(torch.__file__), "lib")
    rocm = os.path.dirname(os.path.dirname(HIPCC))
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), hash_flag] + \
        [a for d in include_paths() + [os.path.join(rocm, "include")] for a in ("-isystem", d)] + \
        [os.path.join(CSRC, "torch_nn.cpp"), "-o", TORCH_LIB, "-L" + LIBDIR, "-l:libumr_hip.so", "-L" + tl, "-lc10", "-lc10_hip", "-ltorch_cpu",
         "-Wl,-rpath,$ORIGIN"]


def build(force=False, verbose=True, extra_flags=()):
    """Compile every source (one hipcc each, in parallel), link the kernel library, then the operators on top of it."""
    if not force and not _stale():
        return LIB
    import tempfile
    from concurrent.futures import ThreadPoolExecutor
    os.makedirs(LIBDIR, exist_ok=True)
    hash_flag = '-DUMR_SRC_HASH="%s"' % source_hash()
    compile_flags = [f for f in FLAGS if f != "-shared"]

    def run(cmd):
        if verbose:
            print("[umr_amd.build]", " ".join(cmd), flush=True)
        subprocess.check_call(cmd)

    with tempfile.TemporaryDirectory() as tmp:
        def one(src):
            obj = os.path.join(tmp, src + ".o")
            run([HIPCC] + compile_flags + [hash_flag] + list(extra_flags) +
                ["-c", os.path.join(CSRC, src), "-o", obj])
            return obj
        with ThreadPoolExecutor(max_workers=8) as ex:
            objs = list(ex.map(one, SOURCES + NN_SOURCES))
        run([HIPCC, "--offload-arch=gfx950", "-fPIC", "-shared"] + objs + ["-o", LIB])
    run(torch_command(hash_flag))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
