"""The kernels' bounded wait (``csrc/umma.cuh``), compiled alone: a barrier that nothing arrives at
ends the wait after some two seconds with a result the host reads, and the context stays usable; a
barrier that is arrived at is seen."""
import ctypes
import os
import subprocess

import pytest
import torch

from halftone_quantizedkvcache_b200.csrc import build

pytestmark = pytest.mark.gpu

SOURCE = r"""
#include "umma.cuh"
__global__ void wait_kernel(int arrive, int* seen, unsigned long long* ns) {
  __shared__ uint64_t bar;
  hq::mbar_init(&bar, 1);
  hq::fence_mbar_init();
  if (arrive) hq::mbar_arrive(&bar);
  const uint64_t from = hq::global_ns();
  *seen = hq::tc::wait_bar(&bar, 0);
  *ns = hq::global_ns() - from;
}
extern "C" __attribute__((visibility("default"))) int run(int arrive, int* seen, unsigned long long* ns) {
  wait_kernel<<<1, 1>>>(arrive, seen, ns);
  return cudaDeviceSynchronize();
}
"""


def test_a_wait_that_nothing_ends_gives_up(tmp_path):
    src, lib = tmp_path / "wait.cu", tmp_path / "wait.so"
    src.write_text(SOURCE)
    subprocess.run([build.nvcc(), *build.ARCH, *build.FLAGS, "-I", build.HERE, "-shared", "-cudart", "static",
                    str(src), "-o", str(lib)], check=True, timeout=300)
    run = ctypes.CDLL(os.fspath(lib)).run
    run.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    seen = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    ns = torch.zeros(2, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    assert run(1, seen[0:].data_ptr(), ns[0:].data_ptr()) == 0
    assert run(0, seen[1:].data_ptr(), ns[1:].data_ptr()) == 0
    assert seen.tolist() == [1, 0]
    # 2^19 polls of 2 to 4 us; a poll's length is the hardware's, so the bounds are wide
    assert ns[0] < 1_000_000 and 500_000_000 < ns[1] < 4_000_000_000
