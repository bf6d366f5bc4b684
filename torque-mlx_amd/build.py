"""Build recipe for libtorque_hip.so (gfx950).

    python torque-mlx_amd/build.py            # or __graft_entry__.build()
    python torque-mlx_amd/build.py --asan OUT.so   # host-only AddressSanitizer build

Compiles the csrc/*.hip sources with hipcc, side by side, and links them into
torque_hip/libtorque_hip.so, in-tree; csrc/paged_binding.cpp becomes the CPython
module torque_hip/_paged.so.  Packed-FP32 VALU ops are disabled for all device code.  The
atomic optimizer is off for device code: it rewrites a single lane's LDS
atomic (the split kernels' tile counter) into a wave-wide form that waits
for the result at once, where the kernels want it one iteration later.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
REPO = ROOT.parent
SOURCES = tuple(ROOT / "csrc" / name for name in ("torque_hip.hip", "paged_append.hip", "paged_attention.hip"))
OUTPUT = ROOT / "torque_hip" / "libtorque_hip.so"
BINDING = ROOT / "csrc" / "paged_binding.cpp"
BINDING_OUTPUT = ROOT / "torque_hip" / "_paged.so"
ARCH = os.environ.get("TORQUE_HIP_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Xarch_device",
    "-mllvm=-amdgpu-atomic-optimizer-strategy=None",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(path).exists():
        raise RuntimeError("hipcc not found")
    return path


# Host-only AddressSanitizer build (argument validation, split planning,
# workspace checks): the host pass is instrumented, the gfx950 code is not.
ASAN_FLAGS = ["-O1", "-g", "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fno-omit-frame-pointer", "-shared-libasan"]


def asan_runtime() -> Path:
    """The clang AddressSanitizer runtime a process must preload to load the ASan build."""
    hits = sorted(Path(hipcc()).resolve().parents[1].glob("lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not hits:
        raise RuntimeError("libclang_rt.asan-x86_64.so not found next to hipcc")
    return hits[-1]


def _run(cmd: list[str], verbose: bool) -> str:
    """Run one compiler command; its messages, or RuntimeError."""
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    stderr = "\n".join(line for line in proc.stderr.splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({proc.returncode}):\n{stderr}")
    return stderr


def build_library(verbose: bool = False, asan: bool = False, output: Path | None = None) -> Path:
    """Compile the library to `output` (default: the in-tree libtorque_hip.so; the ASan build has no
    default location and needs one)."""
    if asan and output is None:
        raise ValueError("the AddressSanitizer build needs an output path outside the package")
    out = Path(output) if output is not None else OUTPUT
    flags = [f for f in HIPCC_FLAGS if not (asan and f == "-O3")] + (ASAN_FLAGS if asan else [])
    with tempfile.TemporaryDirectory(prefix="torque_hip_") as tmp:
        objects = [str(Path(tmp) / (source.stem + ".o")) for source in SOURCES]
        compile_ = [hipcc(), *flags, "-I", str(REPO / "include"), "-I", str(ROOT / "csrc"), "-c"]
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            done = list(pool.map(lambda so: _run([*compile_, str(so[0]), "-o", so[1]], verbose), zip(SOURCES, objects)))
        done.append(_run([hipcc(), *flags, "-shared", *objects, "-o", str(out) + ".tmp"], verbose))
    stderr = "\n".join(text for text in done if text.strip())
    os.replace(str(out) + ".tmp", out)
    if verbose and stderr.strip():
        print(stderr, file=sys.stderr)
    return out


def build_binding(verbose: bool = False) -> Path:
    """Compile the paged cache's CPython module (host code over torch's C++ API and the library's C ABI)."""
    import torch

    base = Path(torch.__path__[0])
    includes = [base / "include", base / "include/torch/csrc/api/include", "/opt/rocm/include", sysconfig.get_paths()["include"], REPO / "include"]
    libraries = ["c10", "c10_hip", "torch", "torch_cpu", "torch_hip", "torch_python"]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in includes), str(BINDING), "-o",
           str(BINDING_OUTPUT) + ".tmp", f"-L{base / 'lib'}", *(f"-l{lib}" for lib in libraries)]
    _run(cmd, verbose)
    os.replace(str(BINDING_OUTPUT) + ".tmp", BINDING_OUTPUT)
    return BINDING_OUTPUT


def build_all(verbose: bool = False) -> Path:
    """The library and the module, side by side."""
    with ThreadPoolExecutor(1) as pool:
        binding = pool.submit(build_binding, verbose)
        library = build_library(verbose)
        binding.result()
    return library


if __name__ == "__main__":
    if "--asan" in sys.argv:
        print(build_library(verbose=True, asan=True, output=Path(sys.argv[sys.argv.index("--asan") + 1])))
    else:
        print(build_all(verbose=True))
