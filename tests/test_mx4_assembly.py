"""Assembly of the 4-bit convolution's device helpers, without a GPU."""
import os
import re
import subprocess

from conftest import ROOT

PROBE = """
#include "srx_conv_mx4.h"
using namespace srx::dev;
// Loads of the compiler's own, which set m0 to `base`, on both sides of one of the helper's, to `base` + 4096.
__global__ void probe(const uint8_t* p, unsigned base, unsigned* out)
{
    extern __shared__ uint8_t lds[];
    const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, 0x1000, 0x27000);
    auto* to = (__attribute__((address_space(3))) uint8_t*)lds + base;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, to, 4, threadIdx.x * 4, 0, 0, 0);
    LOAD(descriptor(p, 0x1000), threadIdx.x * 16, base + 4096);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, to, 4, threadIdx.x * 4 + 64, 0, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    out[threadIdx.x] = lds[threadIdx.x];
}
"""


def test_loads_to_lds_set_their_address_register_in_the_compilers_sight(tmp_path):
    """Otherwise the compiler keeps its own value in m0 over the helper's load, and its next one goes to the wrong place."""
    source = tmp_path / "probe.hip"
    source.write_text(PROBE)
    for load in ("loadToLds", "loadWordToLds"):
        out = tmp_path / (load + ".s")
        subprocess.check_call(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-DLOAD=" + load, "-I" + os.path.join(ROOT, "superresolution_amd", "csrc"),
                               "--offload-device-only", "-S", "-o", str(out), str(source)])
        # the order of writes of m0 and of loads to LDS
        order = re.findall(r"^\s+(s_\w+ m0,|buffer_load_\w+ .* lds)", out.read_text(), re.M)
        assert ["m0" if "m0" in o else "load" for o in order] == ["m0", "load"] * 3, order
