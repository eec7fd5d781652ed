"""Compiles rnnt_amd/csrc/*.hip into librnnt_mi355x.so for gfx950, and torch_binding.cpp into _native.so.

hipcc cross-compiles without a GPU, so this runs in a CPU-only container; the
built library stays in-tree (git-ignored) and travels with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
SOURCES = [os.path.join(CSRC, "rnnt_mi355x.hip"), os.path.join(CSRC, "fc_joint.hip"),
           os.path.join(CSRC, "skinny_dense.hip"), os.path.join(CSRC, "decode_step.hip")]
# operators around the joint network
OPERATOR_SOURCES = [os.path.join(CSRC, n) for n in ("dropout.hip", "beam.hip", "layer.hip", "layer_fp32.hip", "layer_bf16.hip", "layer_fp16.hip")]
OPERATOR_PIECES = [os.path.join(CSRC, n) for n in ("op_util.h", "layer_plan.h", "layer_gemm.h", "layer_gemm_launch.h")]
# rnnt_mi355x.hip is one translation unit whose kernels live in these included pieces
PIECES = [os.path.join(CSRC, n) for n in ("workspace.h", "device_util.h", "lse_rows.h", "sweep.h", "grad_rows.h", "grad_span.h", "grad_split.h", "cell_coef.h", "grad_flat.h", "lse_span.h",
                                          "small_vocab.h", "joint.h", "aux_kernels.h")]
HEADER = os.path.join(os.path.dirname(_HERE), "include", "rnnt_mi355x.h")
LIB = os.path.join(CSRC, "librnnt_mi355x.so")
# the operators' path from torch to the library (plain C++, against the torch that is installed)
BINDING = os.path.join(CSRC, "torch_binding.cpp")
NATIVE = os.path.join(_HERE, "_native.so")
# hipcc's packed float32 instructions have given wrong results on this hardware now and then: no source is built with them
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops"]
# the HIP headers and torch's want to be told their platform
NATIVE_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1"]


def sources_digest() -> str:
    """Sixteen hex digits that change whenever a source of the loss and its joints changes: measurements taken from a build (the HBM
    counter bytes of profiles/traffic.json) are stamped with it and not quoted for another one."""
    import hashlib
    h = hashlib.sha256()
    for p in sorted((*SOURCES, *PIECES)):
        with open(p, "rb") as f:
            h.update(os.path.basename(p).encode() + b"\0" + f.read() + b"\0")
    return h.hexdigest()[:16]


def hipcc_path() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: cannot build librnnt_mi355x.so")


def _stamp(*what) -> str:
    """What an artefact depends on besides its sources, as the bytes that it carries."""
    import hashlib
    return "rnnt-build-" + hashlib.sha256("\0".join(what).encode()).hexdigest()[:16]


def lib_stamp() -> str:
    return _stamp(*FLAGS)


def native_stamp() -> str:
    """The binding is built against one torch and one Python."""
    import sysconfig

    import torch
    return _stamp(torch.__version__, str(torch.version.git_version), str(sysconfig.get_config_var("SOABI")), *NATIVE_FLAGS)


def _carries(path: str, stamp: str) -> bool:
    with open(path, "rb") as f:
        return stamp.encode() in f.read()


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return not _carries(LIB, lib_stamp()) or any(os.path.getmtime(p) > t for p in (*SOURCES, *PIECES, *OPERATOR_SOURCES, *OPERATOR_PIECES, HEADER))


def newer_sources():
    """Sources that are newer than the built library."""
    if not os.path.exists(LIB):
        return [*SOURCES, *OPERATOR_SOURCES]
    t = os.path.getmtime(LIB)
    return [p for p in (*SOURCES, *PIECES, *OPERATOR_SOURCES, *OPERATOR_PIECES, HEADER) if os.path.getmtime(p) > t]


def needs_native_build() -> bool:
    if not os.path.exists(NATIVE):
        return True
    t = os.path.getmtime(NATIVE)
    return not _carries(NATIVE, native_stamp()) or any(os.path.getmtime(p) > t for p in (BINDING, HEADER))


def native_command(out: str):
    """The g++ line that compiles the torch binding."""
    import sysconfig

    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    rocm = os.path.dirname(os.path.dirname(hipcc_path()))
    if not os.path.isdir(os.path.join(rocm, "include", "hip")):
        rocm = "/opt/rocm"
    cxx = shutil.which("g++")
    if not cxx:
        raise RuntimeError("g++ not found: cannot build the torch binding")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), os.path.join(rocm, "include"),
               sysconfig.get_path("include")]
    return [cxx, *NATIVE_FLAGS, f'-DRNNT_BUILD_STAMP="{native_stamp()}"',
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in include], BINDING, "-o", out,
            f"-L{os.path.join(root, 'lib')}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]


def build_native(force: bool = False, verbose: bool = False) -> str:
    """Compiles the torch binding; as build(), one process at a time and moved into place when whole."""
    import fcntl
    import tempfile
    if not force and not needs_native_build():
        return NATIVE
    with open(NATIVE + ".lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if force or needs_native_build():
                with tempfile.TemporaryDirectory(prefix=".build-", dir=_HERE) as tmp:
                    staged = os.path.join(tmp, os.path.basename(NATIVE))
                    cmd = native_command(staged)
                    if verbose:
                        print(" ".join(cmd))
                    subprocess.check_call(cmd)
                    os.replace(staged, NATIVE)
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return NATIVE


def build(force: bool = False, verbose: bool = False, defines=(), out: str = LIB) -> str:
    """defines / out: experiment builds (`-DNAME=VALUE` variants of the library under another file name, selected
    at run time with RNNT_MI355X_LIB).

    Several processes may call this at once (ranks of one job, test workers): one of them builds, under a file
    lock, the others wait and find the library current; objects and the library are written under names of their
    own and moved into place, so nobody ever loads a half-written file."""
    import fcntl
    import tempfile
    if not force and not needs_build() and out == LIB:
        return LIB
    hipcc = hipcc_path()
    with open(out + ".lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if not force and out == LIB and not needs_build():  # another process built it while this one waited
                return LIB
            flags = [*FLAGS, f'-DRNNT_BUILD_STAMP="{lib_stamp()}"', *[f"-D{d}" for d in defines]]
            with tempfile.TemporaryDirectory(prefix=".build-", dir=os.path.dirname(out)) as tmp:
                # one object per source, compiled side by side, then one link
                sources = [*SOURCES, *OPERATOR_SOURCES]
                objs = [os.path.join(tmp, os.path.splitext(os.path.basename(src))[0] + ".o") for src in sources]
                cmds = [[hipcc, *flags, "-c", src, "-o", obj] for src, obj in zip(sources, objs)]
                if verbose:
                    for cmd in cmds:
                        print(" ".join(cmd))
                procs = [subprocess.Popen(cmd) for cmd in cmds]
                failed = [cmd for cmd, pr in zip(cmds, procs) if pr.wait() != 0]
                if failed:
                    raise subprocess.CalledProcessError(1, failed[0])
                staged = os.path.join(tmp, os.path.basename(out))
                link = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", staged, *objs]
                if verbose:
                    print(" ".join(link))
                subprocess.check_call(link)
                os.replace(staged, out)
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return out


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build_native(force=True, verbose=True))
