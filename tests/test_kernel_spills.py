"""The two-tile tcgen05 kernel over whole segments keeps its loops in registers for Q8_0 rows: its dequantisers have 80 each,
and what shares code with the paged instance has made it spill before."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "backburner_b200", "csrc")


def test_two_tile_kernel_does_not_spill(tmp_path):
    src = tmp_path / "k.cu"
    src.write_text('#include <cuda.h>\n#include "pa_prefill.cuh"\n'
                   "template __global__ void pa::pre::prefill_kernel<1, 2, 128, false>(const __grid_constant__ CUtensorMap, const pa::pre::Params);\n")
    nvcc = "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc"
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xptxas=-v", "-I", CSRC, "-c",
                        "-o", str(tmp_path / "k.o"), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    spills = re.findall(r"(\d+) bytes spill stores, (\d+) bytes spill loads", r.stdout + r.stderr)
    assert spills and all(s == ("0", "0") for s in spills), spills
