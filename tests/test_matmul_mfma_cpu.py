"""csrc/matmul_mfma.cuh as the compiler sees it (no GPU: the assembly of a small kernel built here)."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# the compiler's own LDS DMA to one address, before and after dma16 to another
KERNEL = """
#include <hip/hip_runtime.h>
#include "matmul_mfma.cuh"
using namespace ngp::mm;
__global__ void around(const char* p, int* out) {
	__shared__ __attribute__((aligned(1024))) char lds[4096];
	const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 1024, 0x00020000);
	__builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds_of(lds), 4, threadIdx.x * 4, 0, 0, 0);
	dma16(i32x4{(int)(uint32_t)(uint64_t)p, (int)((uint64_t)p >> 32), 1024, 0x00020000}, lds_of(lds) + 2048, threadIdx.x * 16);
	__builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds_of(lds), 4, threadIdx.x * 4, 0, 512, 0);
	wait_and_sync();
	out[threadIdx.x] = ((int*)lds)[threadIdx.x];
}
"""


def test_the_dma_says_that_it_writes_m0(tmp_path):
    """m0 is the LDS address of both kinds of load: behind dma16 the compiler has to set it again, not to go on with the value it had"""
    src, out = str(tmp_path / "around.hip"), str(tmp_path / "around.s")
    open(src, "w").write(KERNEL)
    r = subprocess.run([os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc"), "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "--cuda-device-only", "-S", "-I" + os.path.join(ROOT, "blender-ngp_amd", "csrc"), "-I" + os.path.join(ROOT, "include"), "-o", out, src], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    seen = re.findall(r"s_mov_b32 (m0), (\S+)|(buffer_load_dwordx?4?) ", open(out).read())
    order = ["m0 " + value if m0 else load for m0, value, load in seen]
    assert [o.split()[0] for o in order] == ["m0", "buffer_load_dword", "m0", "buffer_load_dwordx4", "m0", "buffer_load_dword"], order
    assert order[0] == order[4] != order[2], order
