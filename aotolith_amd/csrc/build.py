"""Build the gfx950 code object and the C-ABI host library, in-tree.

Outputs (next to the package, so they travel with the source tree):

* ``aotolith_amd/aoto_gfx950.hsaco`` - every kernel, ``hipcc --genco`` for gfx950;
* ``aotolith_amd/libaoto_hip.so``     - the ``extern "C"`` launchers of
  ``include/aoto_hip.h``;
* ``aotolith_amd/_calls.so``          - the serving operators' calls from Python
  (``calls.cpp``: host code against torch's headers; ``ops.py`` makes the same
  calls without it, at 5 to 8 us more each).

Run ``python -m aotolith_amd.csrc.build`` or call :func:`build`.
"""

from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys
import sysconfig
import warnings

CSRC = os.path.dirname(os.path.abspath(__file__))
PACKAGE = os.path.dirname(CSRC)
ROOT = os.path.dirname(PACKAGE)
INCLUDE = os.path.join(ROOT, "include")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ROCM = os.path.dirname(os.path.dirname(HIPCC))

CODE_OBJECT = os.path.join(PACKAGE, "aoto_gfx950.hsaco")
LIBRARY = os.path.join(PACKAGE, "libaoto_hip.so")
CALLS = os.path.join(PACKAGE, "_calls.so")

# Device flags: gfx950 only; packed-FP32 VALU forms disabled (they are not used
# by hand and the compiler is told not to form them); kernel arguments preloaded
# into SGPRs (up to 14 dwords on gfx950, so a kernel's first loads need not wait
# for a scalar load of its argument buffer; kernels order their arguments for
# it).
DEVICE_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-mllvm",
    "-amdgpu-kernarg-preload-count=16",
    "-I" + CSRC,
    "-I" + INCLUDE,
]


def _run(command: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(command), flush=True)
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        sys.stderr.write(result.stdout + result.stderr)
        raise RuntimeError(f"build step failed ({result.returncode}): {' '.join(command)}")


def calls_built_for() -> str:
    """The torch and Python whose objects ``calls.cpp`` reaches into: a build for others is not to be used."""

    import torch

    return f"torch {torch.__version__} {torch.version.git_version}, {sys.implementation.cache_tag}"


def _calls_command(output: str) -> list[str]:
    import torch
    from torch.utils import cpp_extension

    libraries = os.path.join(os.path.dirname(torch.__file__), "lib")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w", "-I" + INCLUDE,
            "-I" + sysconfig.get_paths()["include"], *("-I" + path for path in cpp_extension.include_paths()),
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DAOTO_BUILT_FOR="{calls_built_for()}"', os.path.join(CSRC, "calls.cpp"), "-o", output,
            "-L" + libraries, "-ltorch_python", "-ltorch_cpu", "-lc10"]


def _build_calls(output: str, verbose: bool) -> None:
    _run(_calls_command(output), verbose)


def build(verbose: bool = False) -> tuple[str, str]:
    """Compile the code object, the host library and the Python calls; return the first two's paths.

    The calls need a host compiler, Python's headers and torch's. Where those are missing the others are built all the
    same, with a warning, and no calls of an earlier build stay.
    """

    tmp_obj, tmp_lib, tmp_calls = CODE_OBJECT + ".tmp", LIBRARY + ".tmp", CALLS + ".tmp"
    commands = (
        [HIPCC, *DEVICE_FLAGS, "--genco", "--no-gpu-bundle-output", os.path.join(CSRC, "kernels.hip"), "-o", tmp_obj],
        # The host library: the C-ABI launchers (paged.cpp and serving.cpp: those of serving), plus noalloc.hip, whose
        # device part is only the static scratch buffer of the allocation-free GEMM entry point.
        [
            HIPCC,
            "-O2",
            "-std=c++17",
            "-fPIC",
            "-shared",
            "--offload-arch=gfx950",
            "-Xclang",
            "-target-feature",
            "-Xclang",
            "-packed-fp32-ops",
            "-I" + INCLUDE,
            "-I" + CSRC,
            os.path.join(CSRC, "aoto_hip.cpp"),
            os.path.join(CSRC, "paged.cpp"),
            os.path.join(CSRC, "serving.cpp"),
            os.path.join(CSRC, "noalloc.hip"),
            "-o",
            tmp_lib,
        ],
    )
    with concurrent.futures.ThreadPoolExecutor() as pool:
        calls = pool.submit(_build_calls, tmp_calls, verbose)
        for step in [pool.submit(_run, command, verbose) for command in commands]:
            step.result()
    os.replace(tmp_obj, CODE_OBJECT)
    os.replace(tmp_lib, LIBRARY)
    try:
        calls.result()
        os.replace(tmp_calls, CALLS)
    except (RuntimeError, OSError, ImportError) as error:
        if os.path.exists(CALLS):
            os.remove(CALLS)
        warnings.warn(f"_calls.so is not built, ops.py makes the serving operators' calls itself: {error}")
    return CODE_OBJECT, LIBRARY


if __name__ == "__main__":
    for path in build(verbose=True):
        print(path, os.path.getsize(path))
