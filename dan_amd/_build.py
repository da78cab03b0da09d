"""Build recipe for the gfx950 shared library (hipcc, in-tree) and the host
modules of the plain calls (g++).

    python -m dan_amd._build          # -> dan_amd/_lib/libdan_tree_attn.so, _decode_calls.so, _layer_calls.so

Flags:
  --offload-arch=gfx950            CDNA4 only, no other targets.
  -mcode-object-version=5          accepted by every ROCm 6/7 runtime (torch
                                   ships its own HIP runtime).
  -target-feature -packed-fp32-ops no packed fp32 VALU instructions.
  -amdgpu-mfma-vgpr-form           matrix-core results in VGPRs, so the softmax
                                   reads the score tile without AGPR copies
                                   (every source but fp8_gemm.hip, whose
                                   accumulators fill the AGPRs).
  -fno-honor-nans -mno-amdgpu-ieee tree_attn.hip only: v_max_f32 without a
                                   canonicalizing max in front of every operand
                                   (the attention's running-max raise). The
                                   other sources keep IEEE NaN semantics, and
                                   host-side argument checks read float bits.

Each source compiles to its own object with its own flags; one link makes
the library.
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRCS = [os.path.join(HERE, "csrc", f) for f in ("tree_attn.hip", "tree_attn_grad.hip", "qkv_front.hip", "tree_plan.hip", "fp8_quant.hip", "fp8_gemm.hip",
                                                 "gdn.hip", "gdn_chunk.hip", "gdn_conv.hip", "gdn_norm.hip", "gdn_proj.hip",
                                                 "paged_append.hip", "paged_attn.hip", "logprobs.hip", "add_norm.hip", "adapt.hip")]
# Extra flags per source (file name -> flags).
SRC_FLAGS = {"tree_attn.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"]}
# Matrix-core results in VGPRs, for every source but the GEMM, whose 256
# accumulators per lane live in the accumulation registers (AGPRs).
MFMA_VGPR_FORM = ["-mllvm", "-amdgpu-mfma-vgpr-form"]
ACC_IN_AGPRS = {"fp8_gemm.hip"}
# The host side of the plain calls: CPython modules on torch's headers (g++).
CALLS = {"_decode_calls.so": os.path.join(HERE, "csrc", "decode_calls.cpp"), "_layer_calls.so": os.path.join(HERE, "csrc", "layer_calls.cpp")}
INCLUDE = os.path.join(ROOT, "include")
OUT_DIR = os.path.join(HERE, "_lib")
OUT = os.path.join(OUT_DIR, "libdan_tree_attn.so")

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    "-mcode-object-version=5",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-command-line-argument",
]


def hipcc():
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found (ROCm is required to build the gfx950 library)")
    return path


def calls_command(src, out):
    import sysconfig

    import torch

    home = os.path.dirname(torch.__file__)
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I", INCLUDE,
            *(f for d in (os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"),
                          sysconfig.get_paths()["include"], os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")) for f in ("-isystem", d)),
            src, "-o", out, "-L", os.path.join(home, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python", "-lamdhip64"]


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature: harmless.
    noise = "is not a recognized feature for this target"
    diag = "\n".join(line for line in (res.stderr or "").splitlines() if noise not in line)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n{diag}")
    if diag.strip() and verbose:
        print(diag, file=sys.stderr)


def build(out=OUT, extra=(), verbose=False):
    """Compile the library; always recompiles. Returns the output path."""
    from concurrent.futures import ThreadPoolExecutor

    os.makedirs(os.path.dirname(out), exist_ok=True)
    obj_dir = os.path.join(os.path.dirname(out), "_obj")
    os.makedirs(obj_dir, exist_ok=True)
    objs = [os.path.join(obj_dir, os.path.basename(src) + ".o") for src in SRCS]
    def flags(src):
        name = os.path.basename(src)
        return [*HIPCC_FLAGS, *([] if name in ACC_IN_AGPRS else MFMA_VGPR_FORM), *SRC_FLAGS.get(name, [])]

    cmds = [[hipcc(), *flags(src), *extra, "-I", INCLUDE, "-c", src, "-o", obj] for src, obj in zip(SRCS, objs)]
    calls = {os.path.join(os.path.dirname(out), name): src for name, src in CALLS.items()}
    cmds = [calls_command(src, path + ".tmp") for path, src in calls.items()] + cmds
    with ThreadPoolExecutor(max_workers=min(len(cmds), max(1, (os.cpu_count() or 1)))) as pool:
        for f in [pool.submit(_run, c, verbose) for c in cmds]:
            f.result()
    tmp = out + ".tmp"
    _run([hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", tmp], verbose)
    os.replace(tmp, out)
    for path in calls:
        os.replace(path + ".tmp", path)
    return out


if __name__ == "__main__":
    print(build(verbose=True))
