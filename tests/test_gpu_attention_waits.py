"""The attention kernels' bounded waits, in a kernel of their own: a barrier that nobody signals ends every wait of the CTA and is reported, and a
CTA that gives up waits for its copies in flight.  Nothing here hangs: each wait has its limit of about a second, which is what the test lets run out."""
import ctypes as C
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "micro-expert-router-ssd-streamed-moe-mer_b200", "csrc")

SOURCE = r"""
#include <cuda_runtime.h>
#include "attend_wait.cuh"

// 0: nothing signals; 1: warp 0's barrier has been signalled.  said: what each of two warps' waits returned, the flag, words of the copy that are there.
__global__ void k_wait(int signalled, const uint32_t *src, uint32_t *said, uint32_t *status) {
  __shared__ uint64_t bars[3];
  __shared__ volatile uint32_t stop;
  __shared__ __align__(16) uint32_t got[256];
  const uint32_t tid = threadIdx.x, warp = tid / 32;
  if (tid == 0) {
    for (int i = 0; i < 3; i++) mbar_init(&bars[i], 1);
    stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (tid == 0) {
    if (signalled) mbar_arrive(&bars[0]);
    mbar_expect_tx(&bars[2], sizeof got);
    bulk_g2s(got, src, sizeof got, &bars[2]);
  }
  __syncwarp();
  const bool ok = wait_or_stop(&bars[warp], 0, &stop, status);
  __syncthreads();
  if (tid % 32 == 0) said[warp] = ok;
  if (tid == 0) said[2] = stop;
  if (tid == 0 && stop) drain_copies(&bars[2]);
  __syncthreads();
  uint32_t right = 0;
  for (int i = 0; i < 256; i++) right += got[i] == src[i];
  if (tid == 0) said[3] = right;
}
extern "C" int run(int signalled, const uint32_t *src, uint32_t *said, uint32_t *status, cudaStream_t s) {
  k_wait<<<1, 64, 0, s>>>(signalled, src, said, status);
  return cudaGetLastError();
}
"""


@pytest.fixture(scope="module")
def kernel(tmp_path_factory):
    d = tmp_path_factory.mktemp("waits")
    src, lib = d / "waits.cu", d / "libwaits.so"
    src.write_text(SOURCE)
    nvcc = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no CUDA compiler here")
    subprocess.check_call([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", "-I", CSRC, str(src),
                           "-o", str(lib)])
    k = C.CDLL(str(lib))
    k.run.argtypes = [C.c_int] + [C.c_void_p] * 4
    return k


@pytest.mark.parametrize("signalled", [0, 1])
def test_a_wait_that_runs_out_stops_the_cta_and_leaves_no_copy_in_flight(kernel, signalled):
    src = torch.arange(1, 257, dtype=torch.int32, device="cuda")
    said, status = torch.full((4,), 9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert kernel.run(signalled, src.data_ptr(), said.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert said.tolist() == [signalled, 0, 1, 256]
    assert status.item() == 4  # MER_DEVSTAT_TIMEOUT
