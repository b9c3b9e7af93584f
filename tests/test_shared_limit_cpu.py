"""The limit of a kernel's dynamic shared memory under calls from several threads, on a runtime that is told to be slow."""
import shutil
import subprocess
from pathlib import Path

import pytest

from ghost_flow_b200.csrc.build import HERE, _nvcc

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>
#include "gf_host.h"

// one kernel's limit; setting it takes its time, another with each call
static std::atomic<int> limit[2], calls;
static thread_local int device;
extern "C" cudaError_t CUDARTAPI cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t CUDARTAPI cudaFuncSetAttribute(const void*, enum cudaFuncAttribute, int bytes) {
  const int d = device, n = calls.fetch_add(1);
  std::this_thread::sleep_for(std::chrono::microseconds(n * 7919 % 400));
  limit[d].store(bytes);
  std::this_thread::sleep_for(std::chrono::microseconds(n * 104729 % 400));
  return bytes > 200000 ? cudaErrorInvalidValue : cudaSuccess;
}
static void kernel() {}

int main() {
  int low = 0;
  for (int round = 0; round < 50; ++round) {
    gf::SharedLimit shared;
    limit[0] = limit[1] = 0;
    std::atomic<int> missed{0}, begun{0};
    std::vector<std::thread> threads;
    for (int t = 0; t < 6; ++t)
      threads.emplace_back([&, t] {
        device = t % 2;
        for (begun.fetch_add(1); begun < 6;) std::this_thread::yield();
        for (int i = 0; i < 5; ++i) {
          const int bytes = 50000 + (t * 31 + i * 17 + round) % 97 * 100;
          if (!shared.raise(kernel, bytes) || limit[device] < bytes) missed.fetch_add(1);      // what a launch would then find
        }
      });
    for (auto& t : threads) t.join();
    low += missed;
  }
  gf::SharedLimit shared;
  const bool refused = !shared.raise(kernel, 300000) && !shared.raise(kernel, 250000) && shared.raise(kernel, 60000);
  const int before = calls;
  const bool known = shared.raise(kernel, 60000) && shared.raise(kernel, 100) && calls == before;
  std::printf("%d %d %d\n", low, refused, known);
}
"""


def test_no_launch_finds_less_than_it_asked_for(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    source, exe = tmp_path / "limit.cpp", tmp_path / "limit"
    source.write_text(PROGRAM)
    include = Path(_nvcc()).resolve().parent.parent / "include"
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-I", str(HERE), "-I", str(include), str(source), "-o", str(exe), "-lpthread"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    assert subprocess.run([str(exe)], capture_output=True, text=True, timeout=120).stdout.split() == ["0", "1", "1"]
