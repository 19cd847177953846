"""Builds x_amd/csrc/libatl_hip.so for gfx950 with hipcc (in-tree, no JIT cache).

Flags: -ffp-contract=off keeps every fp32 expression rounded op by op (the index and cut-off arithmetic must
match the reference's CPU rounding), -munsafe-fp-atomics emits hardware float atomics, and packed FP32 is
disabled (-Xclang -target-feature -Xclang -packed-fp32-ops)."""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parents[1]
SOURCES = ["abi.hip", "events.hip", "tiles.hip", "pairs.hip", "fastpair.hip", "knn.hip", "embed.hip", "rmsnorm.hip", "gscan.hip", "headrot.hip", "decay.hip", "decay_f32.hip",
           "decay_bf16.hip", "decay_f16.hip"]
OUT = HERE / "libatl_hip.so"
ARCH = os.environ.get("ATL_HIP_ARCH", "gfx950")


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (Path(cand).exists() or cand == "hipcc"):
            return cand
    raise RuntimeError("hipcc not found")


def build(verbose: bool = False) -> Path:
    """Compiles the sources side by side (the largest take a minute each) and links them."""
    srcs = [HERE / s for s in SOURCES if (HERE / s).exists()]
    flags = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-munsafe-fp-atomics",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-command-line-argument",
             f"-I{ROOT / 'include'}"]

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")

    with tempfile.TemporaryDirectory() as tmp:
        objs = [str(Path(tmp) / (s.stem + ".o")) for s in srcs]
        with ThreadPoolExecutor(max_workers=8) as pool:
            list(pool.map(lambda so: run([hipcc(), *flags, "-c", str(so[0]), "-o", so[1]]), zip(srcs, objs)))
        out = OUT.with_suffix(".so.tmp")
        run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(out), *objs])
    os.replace(out, OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
