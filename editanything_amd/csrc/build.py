"""Build the gfx950 HIP library (product) and, for the CPU test-suite only, the
host emulation build of the same kernel sources.

    python -m editanything_amd.csrc.build          # libeditanything_hip.so (hipcc, gfx950)
    python -m editanything_amd.csrc.build --emu    # tests/emu/libeditanything_emu.so (host clang)
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
SOURCES = ["ea_gemm.hip", "ea_norm.hip", "ea_attn.hip", "ea_elem.hip", "ea_sam.hip", "ea_exact.hip", "ea_train.hip", "ea_fp8.hip", "ea_fp8_gemm.hip"]
HEADERS = ["ea_platform.h", "ea_gemm.h", "ea_gemm2.h", "ea_gemm8.h", "ea_prims.h", "ea_epi_tr.h", "ea_fp8.h", "ea_fp8_gemm.h", os.path.join(ROOT, "include", "editanything_hip.h")]
# experiment kernels compiled into the tools / emulation builds only (-DEA_TOOLS=1)
TOOLS_HEADERS = [os.path.join(ROOT, "tools", "kernels", "ea_gemm3.h")]
LIB = os.path.join(HERE, "libeditanything_hip.so")
# Compile flags of the product library.  `-target-feature -packed-fp32-ops`: NO packed fp32 VALU instruction (v_pk_fma_f32 /
# v_pk_mul_f32 / v_pk_add_f32 / v_pk_mov_b32) is ever emitted.  Round 5 (tools/probe_pk_swap.hip,
# profiles/r05_gn_exec_repro.*): on gfx950 such an instruction with a cross-half source selection (op_sel: the low result reads
# the HIGH half of src1 / src2 -- hipcc's code for a horizontal add, e.g. in the round-3 GroupNorm statistics loop) returns wrong
# data in lanes 48..63 while another wave of the same SIMD has MFMAs in flight -- i.e. beside any matrix-core kernel of a second
# stream.  tests/test_isa_hazards.py compiles every source with exactly these flags and fails on any instruction of the class.
HIP_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffast-math", "-fno-finite-math-only",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
EMU_DIR = os.path.join(ROOT, "tests", "emu")
EMU_LIB = os.path.join(EMU_DIR, "libeditanything_emu.so")


def _newer(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _hipcc():
    for c in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found: the MI355X library cannot be built")


def build_hip(force=False, verbose=True):
    srcs = [os.path.join(HERE, s) for s in SOURCES]
    deps = srcs + [h if os.path.isabs(h) else os.path.join(HERE, h) for h in HEADERS] + [os.path.abspath(__file__)]
    if not force and not _newer(LIB, deps):
        return LIB
    objs, jobs = [], []
    for s in srcs:                         # all at once: the longest decides
        o = s[:-4] + ".o"
        cmd = [_hipcc()] + HIP_FLAGS + ["-c", s, "-o", o]
        if verbose:
            print(" ".join(cmd), flush=True)
        jobs.append((cmd, subprocess.Popen(cmd)))
        objs.append(o)
    failed = [cmd for cmd, job in jobs if job.wait()]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


def _host_cxx():
    for c in ("/opt/rocm/lib/llvm/bin/clang++", shutil.which("clang++")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("clang++ (for _Float16 / ext_vector_type host emulation) not found")


def build_emu(force=False, verbose=True):
    """TEST INFRASTRUCTURE: same kernels, host fibers instead of a GPU."""
    srcs = [os.path.join(HERE, s) for s in SOURCES]
    emu_srcs = [os.path.join(EMU_DIR, "hip_emu.cpp")]
    deps = srcs + emu_srcs + [os.path.join(EMU_DIR, "hip_emu.h")] + \
        [h if os.path.isabs(h) else os.path.join(HERE, h) for h in HEADERS] + TOOLS_HEADERS + [os.path.abspath(__file__)]
    if not force and not _newer(EMU_LIB, deps):
        return EMU_LIB
    cmd = [_host_cxx(), "-O1", "-std=c++17", "-fPIC", "-shared", "-DEA_EMU", "-DEA_TOOLS=1", "-I", EMU_DIR, "-I", HERE,
           "-Wno-unknown-attributes", "-Wno-unused-value", "-o", EMU_LIB]
    for s in srcs:
        cmd += ["-x", "c++", s]
    for s in emu_srcs:
        cmd += ["-x", "c++", s]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return EMU_LIB


def build_emu_attn_exp(force=False, verbose=True):
    """TEST INFRASTRUCTURE: the attention kernels alone with the round-3 experiment compiled in (-DEA_ATTN_EXP=2: two query
    groups per wave, measured slower on the MI355X and not shipped) -- its own emulation library, so that the main
    emulation build dispatches exactly as the product does."""
    lib = os.path.join(EMU_DIR, "libeditanything_emu_attn_exp2.so")
    srcs = [os.path.join(HERE, "ea_attn.hip"), os.path.join(EMU_DIR, "hip_emu.cpp")]
    deps = srcs + [os.path.join(EMU_DIR, "hip_emu.h"), os.path.join(HERE, "ea_platform.h"), os.path.join(HERE, "ea_prims.h"),
                   os.path.abspath(__file__)]
    if not force and not _newer(lib, deps):
        return lib
    cmd = [_host_cxx(), "-O1", "-std=c++17", "-fPIC", "-shared", "-DEA_EMU", "-DEA_TOOLS=1", "-DEA_ATTN_EXP=2", "-I", EMU_DIR, "-I", HERE,
           "-Wno-unknown-attributes", "-Wno-unused-value", "-o", lib]
    for s in srcs:
        cmd += ["-x", "c++", s]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return lib


if __name__ == "__main__":
    if "--emu" in sys.argv:
        print(build_emu(force="--force" in sys.argv))
    else:
        print(build_hip(force="--force" in sys.argv))
