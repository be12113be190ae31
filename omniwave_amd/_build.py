"""Builds libomniwave_amd.so in-tree with hipcc for gfx950.

The library is a plain C-ABI shared object (include/omniwave_amd.h): host route tables
(route.cpp) and the HIP kernels + launchers (bigemm_fwd.hip).  It is written next to this
file so it travels with the source tree, as is the Python module _glue.so (torch_glue.cpp): the
small operators' calls and autograd nodes over that library, host code against torch's headers.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
import tempfile
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
LIB_PATH = PKG_DIR / "libomniwave_amd.so"
SOURCES = ["route.cpp", "bigemm_fwd.hip", "bigemm_fwd_resident.hip", "bigemm_fwd_wave16.hip", "bigemm_fwd_persist.hip", "bigemm_fwd_split.hip", "bigemm_fwd_f32.hip", "bigemm_fwd_x3.hip", "bigemm_bwd.hip", "bigemm_bwd_f32.hip", "bigemm_bwd_x3.hip", "bwd_block.hip", "stem.hip", "fwd_noalloc.hip",
           "block_norms.hip", "layer_norm.hip", "adamw.hip", "cross_entropy.hip", "distillation.hip", "gated_linear.hip", "gated_linear_bwd.hip"]
GLUE_PATH = PKG_DIR / "_glue.so"
GLUE_SOURCE = "torch_glue.cpp"
ARCH = "gfx950"


def hipcc() -> str:
    found = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(found).exists():
        raise RuntimeError("hipcc not found (expected /opt/rocm/bin/hipcc)")
    return found


def compile_flags() -> list[str]:
    return [
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-Wall",
        "-Wno-unused-function",
        # Packed-FP32 VALU ops stay off: scalar float code only.
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        # MFMA accumulators in VGPRs: the SiLU and epilogue read them with VALU instructions.
        "-mllvm", "-amdgpu-mfma-vgpr-form=1",
        f"-I{INCLUDE}",
        f"-I{CSRC}",
    ]


def glue_commands(obj: str, out: str, lib_dir: str) -> tuple[list[str], list[str]]:
    """Compile and link commands of the Python module (host compiler, torch's headers and libraries)."""
    import torch

    root = Path(torch.__file__).resolve().parent
    rocm = Path(hipcc()).resolve().parent.parent
    if not (rocm / "include" / "hip").exists():
        rocm = Path("/opt/rocm")
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", rocm / "include", INCLUDE,
               sysconfig.get_paths()["include"]]
    cc = shutil.which("g++") or "g++"
    compile_cmd = [cc, "-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
                   f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *[f"-I{p}" for p in include], "-c",
                   str(CSRC / GLUE_SOURCE), "-o", obj]
    link_cmd = [cc, "-shared", obj, "-o", out, f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
                "-lc10_hip", f"-L{rocm / 'lib'}", "-lamdhip64", f"-L{lib_dir}", f"-l:{LIB_PATH.name}", "-Wl,-rpath,$ORIGIN"]
    return compile_cmd, link_cmd


def build(verbose: bool = False) -> Path:
    """Compile every source into LIB_PATH and GLUE_PATH (always recompiles); returns the library path.

    The module needs more than the library does (a host compiler, Python's and torch's headers).  Where it cannot
    be built, a warning says why and there is none: the norms and the loss then run through their operators, and
    only ``AdamW`` is refused."""
    cc = hipcc()
    with tempfile.TemporaryDirectory(prefix="ow_build_") as tmp:
        objs = [str(Path(tmp) / (Path(src).stem + ".o")) for src in SOURCES]
        cmds = [[cc, *compile_flags(), "-c", str(CSRC / src), "-o", obj] for src, obj in zip(SOURCES, objs)]
        out_tmp, glue_tmp = Path(tmp) / LIB_PATH.name, Path(tmp) / GLUE_PATH.name

        def compile_glue() -> list[str]:
            """Compiles the module; returns its link command, which needs the library."""
            compile_cmd, link_cmd = glue_commands(str(Path(tmp) / "torch_glue.o"), str(glue_tmp), tmp)
            _run(compile_cmd, verbose)
            return link_cmd

        with ThreadPoolExecutor(max_workers=min(len(cmds) + 1, os.cpu_count() or 1)) as pool:
            futures = [pool.submit(_run, cmd, verbose) for cmd in cmds]
            glue = pool.submit(compile_glue)
            for future in futures:
                future.result()
        _run([cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", str(out_tmp)], verbose)
        _install(out_tmp, LIB_PATH)
        try:
            _run(glue.result(), verbose)
            _install(glue_tmp, GLUE_PATH)
        except Exception as exc:  # whatever it is that is missing
            GLUE_PATH.unlink(missing_ok=True)  # one that is there is of another library
            warnings.warn(f"{GLUE_PATH.name} was not built: {exc}", RuntimeWarning, stacklevel=2)
    return LIB_PATH


def _install(built: Path, path: Path) -> None:
    staged = path.with_suffix(".so.tmp")
    shutil.copyfile(built, staged)
    os.replace(staged, path)


def _run(cmd: list[str], verbose: bool = False) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        noise = "is not a recognized feature for this target"
        stderr = "\n".join(line for line in proc.stderr.splitlines() if noise not in line)
        raise RuntimeError(f"build failed ({proc.returncode}): {' '.join(cmd)}\n{stderr}")


if __name__ == "__main__":
    print(build(verbose=True))
