"""Build libcsm_hip.so (include/csm_hip.h) and libcsm_ops.so (include/csm_ops.h) for gfx950 in-tree with hipcc: plain C-ABI shared objects, no
torch involvement -- `python csm-hf_amd/build.py` makes them on a host without torch.  `python -m csm_hf_amd.build` or `build_library()`.
Behind them comes _ops_binding.so, the operators' binding for torch tensors (g++, torch and Python headers): where it cannot be built the
libraries stand all the same, and the torch entry points of csm_hf_amd.ops raise."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(HERE, "libcsm_hip.so")
UNITS = ["gemv", "gemv_w0_k1", "gemv_w0_k2", "gemv_w0_k4", "gemv_w1_k1", "gemv_w1_k2", "gemv_w1_k4", "gemv_w2_k1", "gemv_w2_k2", "gemv_w2_k4", "gemm16", "gemm32", "gemm128", "gemm_mx", "train", "attn_prefill", "launchers", "engine", "mimi"]
# gemm16 / gemm32: no implicit multiply-add contraction -- the batched decode launches of every width (16 / 32 / 64 / 128 rows,
# several template instantiations of the same epilogues) must round alike, bit for bit (tests: logits of wide launches against
# 16-row launches); the few fused operations these epilogues want are spelled out (__fmaf_rn)
UNIT_FLAGS = {"attn_prefill": ["-mllvm", "--amdgpu-mfma-vgpr-form"], "gemm16": ["-ffp-contract=off"], "gemm32": ["-ffp-contract=off"], "gemm128": ["-ffp-contract=off", "-mllvm", "--amdgpu-mfma-vgpr-form"]}
# -amdgpu-kernarg-preload-count: leading scalar kernel parameters (up to 14 dwords) arrive in SGPRs, initialised by the dispatcher, instead of
# being s_loaded by every wave at its first instruction (gemv.h GEMV_HOT_PARAMS; round 6)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-value", "-Wno-pass-failed", "-mllvm", "-amdgpu-kernarg-preload-count=16"]

# stand-alone operators (include/csm_ops.h) in a library of their own: they need no engine, and the engine library's measurement records are
# stamped with ITS sources.  packed-fp32-ops off: no v_pk_*_f32 in these kernels
OPS_SRC = os.path.join(CSRC, "ops")
OPS_LIB = os.path.join(HERE, "libcsm_ops.so")
OPS_BINDING = os.path.join(HERE, "_ops_binding.so")   # csrc/ops/binding.cpp: the same calls for torch tensors, built against the installed torch
OPS_UNITS = ["ops_api", "paged_append", "paged_attn", "sample_filtered"]
OPS_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-value", "-Wno-pass-failed",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
BINDING_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__"]
OPS_UNIT_FLAGS = {"paged_attn": ["-mllvm", "--amdgpu-mfma-vgpr-form"]}   # accumulators in VGPRs: the softmax reads every score at once


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _sources_mtime() -> float:
    m = os.path.getmtime(os.path.join(os.path.dirname(HERE), "include", "csm_hip.h"))
    for f in os.listdir(CSRC):
        if f.endswith((".hip", ".h", ".inc")):
            m = max(m, os.path.getmtime(os.path.join(CSRC, f)))
    return m


def sources_sha256() -> str:
    """sha256 over the kernel sources and the C header (sorted file names + contents): identifies the BUILD INPUT of the library.  Measurement
    records (profiles/hbm_traffic.json, profiles/launch_kinds_b*.json) are stamped with it and bench.py marks them stale when it differs --
    a rebuilt library of the same sources is the same build, whatever its bytes are."""
    import hashlib
    h = hashlib.sha256()
    files = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".hip", ".h", ".inc"))]
    files.append(os.path.join(os.path.dirname(HERE), "include", "csm_hip.h"))
    for f in files:
        h.update(os.path.basename(f).encode())
        h.update(open(f, "rb").read())
    return h.hexdigest()


def build_library(force: bool = False, verbose: bool = False, defines=(), out: str = None) -> str:
    """`defines` / `out`: A/B variants of the same ABI (e.g. ("CSM_NO_PROBE",) -> libcsm_hip_noprobe.so), selected at
    run time with the CSM_HIP_LIB environment variable.  Without them the operators' library and its binding are built too."""
    path = _build_engine(force, verbose, defines, out)
    if not defines and out is None:
        build_ops_library(force, verbose)
        try:
            build_ops_binding(force, verbose)
        except Exception as e:
            print(f"[build] no {os.path.basename(OPS_BINDING)} (csm_hf_amd.ops will raise): {e}", file=sys.stderr)
    return path


def _build_engine(force, verbose, defines, out) -> str:
    global OBJ
    lib_out = out or LIB
    if not force and not defines and os.path.exists(LIB) and os.path.getmtime(LIB) >= _sources_mtime():
        return LIB
    hipcc = _hipcc()
    obj_dir = OBJ if not defines else OBJ + "_" + "_".join(defines)
    os.makedirs(obj_dir, exist_ok=True)

    def compile_one(u):
        cmd = [hipcc, *FLAGS, *UNIT_FLAGS.get(u, []), *[f"-D{d}=1" for d in defines], "-c", os.path.join(CSRC, u + ".hip"), "-o", os.path.join(obj_dir, u + ".o")]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for {u}.hip:\n{r.stderr[-4000:]}")
        if verbose:
            print(f"[build] {u}.o", file=sys.stderr)

    with ThreadPoolExecutor(min(len(UNITS), os.cpu_count() or 4)) as ex:
        list(ex.map(compile_one, UNITS))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *[os.path.join(obj_dir, u + ".o") for u in UNITS], "-o", lib_out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
    return lib_out


def _newer(path: str, deps) -> bool:
    return os.path.exists(path) and os.path.getmtime(path) >= max(os.path.getmtime(f) for f in deps)


def build_ops_library(force: bool = False, verbose: bool = False) -> str:
    """libcsm_ops.so from csrc/ops (include/csm_ops.h); reused when it is newer than its sources unless `force`."""
    deps = [os.path.join(OPS_SRC, f) for f in os.listdir(OPS_SRC) if f.endswith((".hip", ".h"))]
    deps += [os.path.join(CSRC, "common.h"), os.path.join(os.path.dirname(HERE), "include", "csm_ops.h")]
    if not force and _newer(OPS_LIB, deps):
        return OPS_LIB
    hipcc, obj_dir = _hipcc(), os.path.join(OPS_SRC, "build")
    os.makedirs(obj_dir, exist_ok=True)

    def compile_one(u):
        cmd = [hipcc, *OPS_FLAGS, *OPS_UNIT_FLAGS.get(u, []), "-c", os.path.join(OPS_SRC, u + ".hip"), "-o", os.path.join(obj_dir, u + ".o")]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for ops/{u}.hip:\n{r.stderr[-4000:]}")
        if verbose:
            print(f"[build] ops/{u}.o", file=sys.stderr)

    with ThreadPoolExecutor(min(len(OPS_UNITS), os.cpu_count() or 4)) as ex:
        list(ex.map(compile_one, OPS_UNITS))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *[os.path.join(obj_dir, u + ".o") for u in OPS_UNITS], "-o", OPS_LIB]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
    return OPS_LIB


def binding_stamp() -> str:
    """What _ops_binding.so has to have been built for: the installed torch (its inlined layouts are compiled in), this Python, the flags."""
    import sysconfig
    import torch
    return (f"csm_ops binding for torch {torch.__version__} ({torch.version.git_version}), C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"{sysconfig.get_config_var('SOABI')}, {' '.join(BINDING_FLAGS)}")


def build_ops_binding(force: bool = False, verbose: bool = False) -> str:
    """_ops_binding.so from csrc/ops/binding.cpp; reused when it is newer than its sources and carries `binding_stamp()` unless `force`."""
    import sysconfig
    import torch
    stamp, obj_dir = binding_stamp(), os.path.join(OPS_SRC, "build")
    deps = [os.path.join(OPS_SRC, "binding.cpp"), os.path.join(os.path.dirname(HERE), "include", "csm_ops.h")]
    if not force and _newer(OPS_BINDING, deps):
        with open(OPS_BINDING, "rb") as f:
            if stamp.encode() in f.read():
                return OPS_BINDING
    os.makedirs(obj_dir, exist_ok=True)
    base = os.path.dirname(torch.__file__)
    inc, lib = os.path.join(base, "include"), os.path.join(base, "lib")
    dirs = [inc, os.path.join(inc, "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"], os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")]
    obj = os.path.join(obj_dir, "binding.o")
    for what, cmd in (("g++ failed for ops/binding.cpp", ["g++", *BINDING_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DCSM_BINDING_STAMP="{stamp}"',
                                                          *["-isystem" + d for d in dirs], "-c", deps[0], "-o", obj]),
                      ("link of the binding failed", ["g++", "-shared", obj, "-o", OPS_BINDING, "-L" + HERE, "-l:" + os.path.basename(OPS_LIB), "-Wl,-rpath,$ORIGIN",
                                                      "-L" + lib, "-ltorch_python", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip"])):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{what}:\n{r.stderr[-4000:]}")
    if verbose:
        print("[build] ops/binding.o", file=sys.stderr)
    return OPS_BINDING


if __name__ == "__main__":
    defs = tuple(a[2:] for a in sys.argv[1:] if a.startswith("-D"))
    outs = [a[6:] for a in sys.argv[1:] if a.startswith("--out=")]
    print(build_library(force="--force" in sys.argv or bool(defs), verbose=True, defines=defs, out=outs[0] if outs else None))
    if not defs and not outs:
        import importlib.util
        if importlib.util.find_spec("torch"):   # with torch there is something to bind to: a binding that could not be built is an error
            build_ops_binding()
