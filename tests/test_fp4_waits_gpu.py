"""GPU: the limit of waits inside the attention kernels, and the count of those
that ran out."""
import subprocess

import pytest
import torch

from flexkv_b200 import fp4_cache
from flexkv_b200.build import ARCH_FLAGS, CSRC, _nvcc

pytestmark = pytest.mark.gpu

# One thread waits for a barrier at which nobody arrives, eight tries and then one; another barrier has been met.
PROGRAM = """
#include <cstdio>
#include <cuda_runtime.h>
#include "fp4_wait.cuh"
__global__ void waits(int *tries) {
  __shared__ uint64_t never, met;
  if (threadIdx.x) return;
  fkv::mbar_init(&never, 1), fkv::mbar_init(&met, 1);
  fkv::mbar_arrive(&met);
  fkv::Patience patience{8};
  patience.wait(&met, 0);
  tries[0] = patience.tries;
  patience.wait(&never, 0);
  tries[1] = patience.tries;
  patience.wait(&never, 0);
  patience.wait(&met, 0);
  tries[2] = patience.tries;
}
int main() {
  int *tries, host[3] = {-1, -1, -1};
  unsigned long long n = 99;
  if (cudaMalloc(&tries, sizeof(host))) return 1;
  for (int i = 0; i < 3; ++i) waits<<<1, 32>>>(tries);
  if (cudaDeviceSynchronize() || cudaMemcpy(host, tries, sizeof(host), cudaMemcpyDeviceToHost) ||
      cudaMemcpyFromSymbol(&n, fkv::g_wait_timeouts, sizeof(n)))
    return 2;
  std::printf("%d %d %d %llu\\n", host[0], host[1], host[2], n);
}
"""


def test_a_wait_that_runs_out_is_counted_once(tmp_path):
    """The thread goes on, with a single try for each later wait, and the kernel ends without an error."""
    (tmp_path / "w.cu").write_text(PROGRAM)
    exe = str(tmp_path / "w")
    subprocess.run([_nvcc(), *ARCH_FLAGS, "-std=c++17", "-I", CSRC, "-o", exe, str(tmp_path / "w.cu")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.split() == ["8", "1", "1", "3"], out


def test_the_count_waits_for_every_stream():
    """For streams that do not synchronise with the default one, too."""
    assert fp4_cache.fp4_wait_timeouts() == 0
    stream, event = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(500_000_000)  # a quarter of a second
        event.record()
    assert not event.query()
    assert fp4_cache.fp4_wait_timeouts(torch.device("cuda", torch.cuda.current_device())) == 0
    assert event.query()
