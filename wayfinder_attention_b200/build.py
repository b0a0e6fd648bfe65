"""Build libwayfinder_sm100.so in-tree with nvcc (sm_100a only), and _wf_torch.so with g++.

Usage: python -m wayfinder_attention_b200.build [--verbose]

The shared libraries are written next to this file so that they travel with the
source tree; the Python package loads them from there and refuses to run
without them.  The first holds the kernels behind the C ABI; the second the
PyTorch calls (argument checks, autograd nodes) of the operators that have them.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "libwayfinder_sm100.so"
LIB_PATH = PKG_DIR / LIB_NAME

SOURCES = ["wf_abi.cu", "wf_topk.cu", "wf_topk_tc.cu", "wf_attn.cu", "wf_attn_bf16.cu", "wf_attn_f16.cu",
           "wf_attn_f32.cu", "wf_addr_proj.cu",
           "wf_attn_bwd.cu", "wf_keymask.cu", "wf_bench.cu",
           "wf_gemm.cu", "wf_linear.cu", "wf_linear_few.cu",
           "wf_layer_norm.cu", "wf_logprobs.cu"]
TORCH_SOURCE = "wf_torch.cpp"
TORCH_LIB_PATH = PKG_DIR / "_wf_torch.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or put /usr/local/cuda/bin on PATH")
    return cand


def _sources() -> list[Path]:
    return [CSRC / s for s in SOURCES]


def _deps() -> list[Path]:
    return _sources() + [CSRC / TORCH_SOURCE] + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [REPO_DIR / "include" / "wayfinder.h"]


def up_to_date() -> bool:
    if not (LIB_PATH.exists() and TORCH_LIB_PATH.exists()):
        return False
    t = min(LIB_PATH.stat().st_mtime, TORCH_LIB_PATH.stat().st_mtime)
    return all(p.stat().st_mtime <= t for p in _deps())


def torch_command(out: Path) -> list[str]:
    """g++ on the PyTorch calls, against the headers and libraries of the torch that is installed."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include"]
    return [
        os.environ.get("CXX") or shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
        "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
        "-I", sysconfig.get_path("include"), *[a for p in include for a in ("-isystem", str(p))],
        str(CSRC / TORCH_SOURCE), "-o", str(out), "-L", str(root / "lib"),
        "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ldl",
    ]


def build(verbose: bool = False, force: bool = False) -> Path:
    if not force and up_to_date():
        return LIB_PATH
    nvcc = nvcc_path()
    obj_dir = PKG_DIR / "_build"
    obj_dir.mkdir(exist_ok=True)
    common = [
        "-O3",
        "-std=c++17",
        "-lineinfo",
        "-Xcompiler",
        "-fPIC",
        "-Xcompiler",
        "-fvisibility=hidden",
        "-I",
        str(REPO_DIR / "include"),
        *ARCH_FLAGS,
    ]
    if verbose:
        common += ["-Xptxas", "-v"]
    # translation units compile concurrently (the attention instantiations dominate)
    jobs = []
    torch_tmp = TORCH_LIB_PATH.with_suffix(".so.tmp")
    torch_job = subprocess.Popen(torch_command(torch_tmp), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    for src in _sources():
        obj = obj_dir / (src.stem + ".o")
        cmd = [nvcc, *common, "-c", str(src), "-o", str(obj)]
        jobs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    objs = []
    errors = []
    for src, obj, proc in jobs:
        _, err = proc.communicate()
        if proc.returncode != 0:
            errors.append(f"nvcc failed on {src.name}:\n{err}")
        elif verbose and err:
            sys.stderr.write(err)
        objs.append(str(obj))
    _, err = torch_job.communicate()
    if torch_job.returncode != 0:
        errors.append(f"g++ failed on {TORCH_SOURCE}:\n{err}")
    if errors:
        raise RuntimeError("\n".join(errors))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *objs, "-cudart", "static"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc link failed:\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    os.replace(torch_tmp, TORCH_LIB_PATH)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/smem usage")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force))


if __name__ == "__main__":
    main()
