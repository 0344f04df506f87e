"""Build every native component in-tree.

Host-only pieces build with g++; device code builds with hipcc for gfx950
(MI355X) only — no multi-arch fatbins, no CUDA paths.  Outputs land in
sofa_amd/native/{bin,lib} so they travel with the repo snapshot to GPU boxes.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "bin")
LIB = os.path.join(HERE, "lib")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
GFX_ARCH = "gfx950"
# packed 32-bit arithmetic off for all device code: some of its forms have given
# wrong results on gfx950
HIP_FLAGS = [
    f"--offload-arch={GFX_ARCH}",
    "-O3",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _newer(dst: str, *srcs: str) -> bool:
    if not os.path.exists(dst):
        return False
    dt = os.path.getmtime(dst)
    return all(os.path.getmtime(s) <= dt for s in srcs if os.path.exists(s))


def _recipe(cmd, *uses: str) -> str:
    """What a target depends on besides its sources, wherever the tree is: the
    command, the ROCm release, and `uses`."""
    try:
        with open(os.path.join(ROCM, ".info", "version")) as f:
            rocm = f.read().strip()
    except OSError:
        rocm = "unknown"
    return "\n".join([*cmd, *uses, "ROCm " + rocm]).replace(HERE, ".") + "\n"


def _fresh(dst: str, srcs, recipe: str) -> bool:
    """dst is newer than srcs and was made by the same recipe, which is kept
    beside it."""
    try:
        with open(dst + ".made") as f:
            return f.read() == recipe and _newer(dst, *srcs)
    except OSError:
        return False


def _start(cmd, verbose: bool) -> subprocess.Popen:
    if verbose:
        print("+ " + " ".join(cmd))
    return subprocess.Popen(cmd)


def _finish(running) -> None:
    """Waits for all (dst, recipe, cmd, process), then raises if one failed."""
    failed = None
    for dst, recipe, cmd, process in running:
        if process.wait() != 0:
            failed = failed or (process.returncode, cmd)
        else:
            with open(dst + ".made", "w") as f:
                f.write(recipe)
    if failed:
        raise subprocess.CalledProcessError(*failed)


def _make(dst: str, srcs, cmd, verbose: bool, force: bool, *uses: str) -> None:
    recipe = _recipe(cmd, *uses)
    if force or not _fresh(dst, srcs, recipe):
        _finish([(dst, recipe, cmd, _start(cmd, verbose))])


def build_all(verbose: bool = False, model: bool = True, force: bool = False) -> None:
    """model: the operators of workloads.kernels as well, which recording does
    not need and which take a minute.  force: also what is up to date."""
    os.makedirs(BIN, exist_ok=True)
    os.makedirs(LIB, exist_ok=True)

    host_targets = [
        (
            os.path.join(BIN, "sofa-cpusampler"),
            [os.path.join(HERE, "cpusampler", "cpusampler.cc")],
            ["g++", "-O2", "-std=c++17"],
            [],
        ),
        (
            os.path.join(BIN, "sofa-timebase"),
            [os.path.join(HERE, "timebase", "timebase.cc")],
            ["g++", "-O2", "-std=c++17"],
            [],
        ),
        (
            os.path.join(BIN, "sofa-pktcap"),
            [os.path.join(HERE, "pktcap", "pktcap.cc")],
            ["g++", "-O2", "-std=c++17"],
            [],
        ),
        (
            os.path.join(BIN, "sofa-syscalltrace"),
            [os.path.join(HERE, "syscalltrace", "syscalltrace.cc")],
            ["g++", "-O2", "-std=c++17"],
            [],
        ),
        (
            os.path.join(LIB, "libsofarccl.so"),
            [
                os.path.join(HERE, "rccl_shim", "rccl_shim.cc"),
                os.path.join(HERE, "collector", "sgt_format.h"),
            ],
            ["g++", "-O2", "-std=c++17", "-fPIC", "-shared"],
            ["-ldl", "-lpthread"],
        ),
        (
            os.path.join(LIB, "libsofatracer.so"),
            [
                os.path.join(HERE, "collector", "sofatracer.cc"),
                os.path.join(HERE, "collector", "sgt_format.h"),
            ],
            [
                "g++",
                "-O2",
                "-std=c++17",
                "-fPIC",
                "-shared",
                "-D__HIP_PLATFORM_AMD__",
                f"-I{ROCM}/include",
            ],
            [f"-L{ROCM}/lib", "-lrocprofiler-sdk", f"-Wl,-rpath,{ROCM}/lib"],
        ),
        (
            os.path.join(LIB, "libsofahsalite.so"),
            [
                os.path.join(HERE, "hsalite", "hsalite.cc"),
                os.path.join(HERE, "collector", "sgt_format.h"),
            ],
            [
                "g++",
                "-O2",
                "-g",  # line info for crash triage; free at runtime
                "-std=c++17",
                "-fPIC",
                "-shared",
                # hsa_api_trace.h uses the in-tree "inc/" include layout
                # unless AMD_INTERNAL_BUILD; the installed headers are flat
                "-DAMD_INTERNAL_BUILD",
                f"-I{ROCM}/include",
                f"-I{ROCM}/include/hsa",
            ],
            ["-lpthread"],
        ),
    ]
    for dst, srcs, cc, link in host_targets:
        if not os.path.exists(srcs[0]):
            continue
        cc_srcs = [s for s in srcs if s.endswith((".cc", ".cpp"))]
        _make(dst, srcs, cc + ["-o", dst] + cc_srcs + link, verbose, force)

    # --- HIP device code (gfx950) ---
    hipcc = os.path.join(ROCM, "bin", "hipcc")
    ring_h = os.path.join(HERE, "hip", "trace_ring.h")
    hip_targets = [
        (
            os.path.join(LIB, "libsofahip.so"),
            [
                os.path.join(HERE, "hip", "timebase_kernel.hip"),
                os.path.join(HERE, "hip", "trace_ring.hip"),
                os.path.join(HERE, "hip", "ring_writer.hip"),
                ring_h,
            ],
        ),
        (
            os.path.join(BIN, "sofa-bandwidth"),
            [os.path.join(HERE, "hip", "bandwidth.hip"), ring_h],
        ),
    ]
    for dst, srcs in hip_targets:
        srcs = [s for s in srcs if os.path.exists(s)]
        if not srcs:
            continue
        cmd = [hipcc] + HIP_FLAGS + ["-std=c++17"]
        if dst.endswith(".so"):
            cmd += ["-fPIC", "-shared"]
        cmd += ["-o", dst] + [s for s in srcs if s.endswith(".hip")]
        if dst.endswith("sofa-bandwidth"):
            # --ring mode links the device-trace-ring machinery
            cmd += ["-L" + LIB, "-lsofahip", "-Wl,-rpath,$ORIGIN/../lib"]
        _make(dst, srcs, cmd, verbose, force)

    if model:
        _build_model_kernels(hipcc, verbose, force)


def _build_model_kernels(hipcc: str, verbose: bool, force: bool) -> None:
    """The operators of workloads.kernels: the kernels, one object per source,
    compiled side by side (their many variants take a minute each) and linked
    into libsofamodel, and their binding to torch where torch is installed."""
    src_dir = os.path.join(HERE, "hip", "model")
    dst = os.path.join(LIB, "libsofamodel.so")
    headers = [os.path.join(src_dir, n) for n in ("model_ops.h", "model_api.h")]
    srcs = [os.path.join(src_dir, n) for n in sorted(os.listdir(src_dir)) if n.endswith(".hip")]
    objs, running = [], []

    def start(obj, srcs, cmd, *uses):
        recipe = _recipe(cmd, *uses)
        if force or not _fresh(obj, srcs, recipe):
            running.append((obj, recipe, cmd, _start(cmd, verbose)))

    for src in srcs:
        obj = os.path.join(LIB, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        start(obj, [src, *headers], [hipcc] + HIP_FLAGS + ["-std=c++20", "-fPIC", "-c", src, "-o", obj])

    binding = os.path.join(src_dir, "bindings.cc")
    module, module_obj = os.path.join(LIB, "sofa_model.so"), os.path.join(LIB, "bindings.o")
    torch_lib = torch_version = None
    try:
        import torch
        from torch.utils.cpp_extension import include_paths

        torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
        torch_version = "torch " + torch.__version__
    except ImportError:
        if verbose:
            print("torch is not installed: the operators of workloads.kernels are not bound")
    if torch_lib:
        include = include_paths() + [f"{ROCM}/include", sysconfig.get_paths()["include"]]
        start(module_obj, [binding, headers[1]],
              ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
              + [f"-I{i}" for i in include] + ["-c", binding, "-o", module_obj], torch_version)

    _finish(running)
    _make(dst, objs, [hipcc, f"--offload-arch={GFX_ARCH}", "-shared", "-o", dst] + objs, verbose, force)
    if torch_lib:
        _make(module, [module_obj, dst],
              ["g++", "-shared", "-o", module, module_obj, f"-L{torch_lib}", "-ltorch_python", "-ltorch",
               "-ltorch_cpu", "-lc10_hip", "-lc10", f"-L{LIB}", "-lsofamodel", "-Wl,-rpath,$ORIGIN"],
              verbose, force, torch_version)


if __name__ == "__main__":
    build_all(verbose=True)
