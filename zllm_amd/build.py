"""Build libzs.so (gfx950) in-tree with hipcc.

The library is the product: hand-written HIP kernels + the C ABI of
include/zs.h. `python -m zllm_amd.build` or `build()` compiles every source
each time it is called.
"""
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libzs.so")

SOURCES = ["zs_api.cpp", "zs_grammar.cpp", "zs_regex.cpp", "zs_schema.cpp", "zs_tokens.cpp", "zs_wire.cpp", "zs_sample.hip", "zs_row.hip", "zs_sums.hip", "zs_dfa.hip", "zs_lane.hip", "zs_spec.hip",
           "zs_head.hip", "zs_beam.hip", "zs_distill.hip", "zs_ce.hip", "zs_q4.hip"]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # IEEE f32 behaviour the exact paths rely on: keep denormals, no contraction
    "-fno-gpu-flush-denormals-to-zero",
    "-ffp-contract=off",
    "-fno-fast-math",
    # some forms of packed fp32 VALU ops have given wrong results
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I" + os.path.join(ROOT, "include"),
    "-Wno-unused-result",
]


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("hipcc failed building libzs.so")


def build(verbose=False):
    """The sources side by side (one behind the other they take four minutes), then the library."""
    with tempfile.TemporaryDirectory(dir=HERE, prefix=".build") as tmp, ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        objs = [os.path.join(tmp, s + ".o") for s in SOURCES]
        # (the longest first)
        list(pool.map(lambda s: _run([HIPCC] + FLAGS + ["-c", os.path.join(CSRC, s), "-o", os.path.join(tmp, s + ".o")], verbose),
                      reversed(SOURCES)))
        _run([HIPCC, "--offload-arch=gfx950", "-fPIC", "-shared"] + objs + ["-o", LIB + ".tmp"], verbose)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
