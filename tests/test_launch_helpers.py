"""Host-side launch helpers (csrc/launch.cuh) compiled for the CPU against a fake of the two runtime calls they make."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "triattention_b200" / "csrc"

PROGRAM = r"""
#include "launch.cuh"

#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <thread>

static std::mutex m;
static std::condition_variable cv;
static int attribute = 0, calls = 0, big_entered = 0, small_done = 0;

extern "C" cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
// The attribute is what the last call set.  A call for 150000 bytes returns only after the thread that wants 100000 is through, or
// after a while, if that one has to wait.
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
  std::unique_lock<std::mutex> lock(m);
  attribute = value;
  ++calls;
  if (value == 150000) {
    big_entered = 1;
    cv.notify_all();
    cv.wait_for(lock, std::chrono::milliseconds(500), [] { return small_done != 0; });
  }
  return cudaSuccess;
}
static void kernel(int) {}

int main() {
  std::thread big([] { if (!triattn::ensure_dynamic_smem<kernel>(150000)) std::abort(); });
  std::thread small([] {
    std::unique_lock<std::mutex> lock(m);
    cv.wait(lock, [] { return big_entered != 0; });
    lock.unlock();
    if (!triattn::ensure_dynamic_smem<kernel>(100000)) std::abort();
    lock.lock();
    small_done = 1;
    cv.notify_all();
  });
  big.join();
  small.join();
  const int after_both = attribute;
  if (!triattn::ensure_dynamic_smem<kernel>(120000) || !triattn::ensure_dynamic_smem<kernel>(150000)) return 1;
  std::printf("%d %d %d\n", after_both, attribute, calls);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_shared_memory_opt_in_is_never_lowered_by_another_thread(tmp_path):
    """Two threads raise one kernel's dynamic shared memory to different sizes at the same time (kernels sized by the width of a
    block table): the attribute ends at the larger one, so later launches of either size go through."""
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"
    src = tmp_path / "smem.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "smem"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{cuda}", f"-I{CSRC}", "-x", "c++", str(src), "-o", str(exe)], check=True,
                   capture_output=True, text=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
    assert [int(x) for x in out] == [150000, 150000, 1]
