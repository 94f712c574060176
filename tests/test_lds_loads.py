"""Loads to LDS in assembly set m0, the address register that the compiler keeps for its own loads to LDS too."""
import os
import re
import subprocess

from conftest import ROOT

KERNEL = r"""
#include "kernels/seq_attn.hpp"
extern "C" __global__ void both(const float* p, float* out, i4 buffer) {
    __shared__ float mine[64];
    __attribute__((address_space(3))) void* to = (__attribute__((address_space(3))) void*)mine;
    const __attribute__((address_space(1))) void* from = (const __attribute__((address_space(1))) void*)p;
    __builtin_amdgcn_global_load_lds(from, to, 4, 0, 0);
    load_to_lds(buffer, threadIdx.x * 16, 1024);
    __builtin_amdgcn_global_load_lds(from, to, 4, 256, 0);
    vm_wait();
    __syncthreads();
    out[threadIdx.x] = mine[threadIdx.x];
}
"""


def test_the_compiler_knows_that_m0_changes(tmp_path):
    """Behind the load in assembly the compiler sets m0 again before a load of its own to the same place as before."""
    src, asm = tmp_path / "both.hip", tmp_path / "both.s"
    src.write_text(KERNEL)
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-S", "--cuda-device-only", "--offload-arch=gfx950", "-O1",
                    "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I", os.path.join(ROOT, "prism-inference_amd", "csrc"), str(src), "-o", str(asm)], check=True, timeout=300,
                   stderr=subprocess.DEVNULL)
    body = re.search(r"^both:(.*?)s_endpgm", asm.read_text(), re.S | re.M).group(1)
    lines = [x.strip() for x in body.split("\n")]
    mine = [i for i, x in enumerate(lines) if x.startswith("global_load_lds")]
    theirs = [i for i, x in enumerate(lines) if x.startswith("buffer_load_dwordx4") and x.endswith("lds")]
    assert len(mine) == 2 and len(theirs) == 1 and mine[0] < theirs[0] < mine[1]
    assert any(re.match(r"s_\w+ m0,", x) for x in lines[theirs[0] + 1:mine[1]])
