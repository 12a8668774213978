"""The bounded waits (csrc/waits.cuh) compiled for the host over fake barriers and a fake clock: what a kernel whose
wait gave up still waits for."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from tilegen_b200 import _lib

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <vector>
#define __device__
#define __forceinline__ inline
namespace tg {
constexpr unsigned long long kWaitLimitNs = 1000;
unsigned long long g_clock = 0, g_tick = 0;
unsigned int g_device_status = 0;
void atomicOr(unsigned int* p, unsigned int v) { *p |= v; }
unsigned long long globaltimer_ns() { return g_clock += g_tick; }
struct Poll { uint64_t bar; uint32_t parity; };
std::vector<Poll> g_done;   // the waits that ended, in order
int g_polls = 0;            // of the wait under way
uint64_t g_stuck = ~0ull;   // the barrier that never completes
bool mbar_try_wait(uint64_t* bar, uint32_t parity) {  // completes at its 100th poll
  g_clock += 1;
  if (*bar == g_stuck || ++g_polls < 100) return false;
  g_polls = 0;
  g_done.push_back({*bar, parity});
  return true;
}
}
#include "waits.cuh"
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  using namespace tg;
  uint64_t bars[5] = {0, 1, 2, 3, 4};
  for (int stages = 1; stages <= 5; ++stages)
    for (int issued = 0; issued <= 14; ++issued) {
      g_done.clear();
      ring_drain(bars, issued, stages, 1u);
      const int last = issued < stages ? issued : stages;
      CHECK(int(g_done.size()) == last);  // each is waited for until it completes
      for (int j = 0; j < last; ++j) {
        const int i = issued - last + j;
        CHECK(g_done[j].bar == uint64_t(i % stages) && g_done[j].parity == uint32_t(i / stages % 2));
      }
    }
  CHECK(g_device_status == 0);
  g_done.clear();
  g_stuck = 2;
  const unsigned long long t0 = g_clock;
  ring_drain(bars, 9, 4, 4u);  // a load that never lands: its limit, then the others
  CHECK(g_device_status == 4 && g_done.size() == 3 && g_clock - t0 > kWaitLimitNs && g_clock - t0 < 2 * kWaitLimitNs);
  const unsigned long long t1 = g_clock;
  g_tick = 1;
  wait_out();
  CHECK(g_clock - t1 > kWaitLimitNs && g_clock - t1 < 2 * kWaitLimitNs);
  return 0;
}
"""


def test_loads_in_flight_are_waited_for(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "waits.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "waits"
    subprocess.run([compiler, "-std=c++17", "-O1", "-I", _lib.CSRC_DIR, "-o", str(exe), str(src)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_the_four_bit_kernel_drains_its_ring_with_them():
    """Not with the wait that ends as soon as another role has given up: the loads would land after the CTA has left."""
    with open(os.path.join(_lib.CSRC_DIR, "gemv_i4.cuh")) as f:
        text = f.read()
    tail = text[text.index("++filled"):text.index("named_barrier(1, WK * WR * 32)")]
    assert "ring_drain(full_bar, filled, p.stages" in tail and "mbar_wait(&scale_bar" in tail


def test_the_grouped_kernel_leaves_nothing_in_flight():
    """Once all roles of the CTA are done, not before: a flag that a slower role sets later would be missed."""
    with open(os.path.join(_lib.CSRC_DIR, "gemm_grouped.cuh")) as f:
        text = f.read()
    tail = text[text.index("if (lane == 0) bulk_wait<0>();"):text.index("tmem_dealloc_pair(")]
    assert tail.index("__syncthreads()") < tail.index("if (abort_flag && threadIdx.x == 0) wait_out()") < tail.index("cluster_sync()")


def test_the_tiled_kernel_leaves_nothing_in_flight():
    with open(os.path.join(_lib.CSRC_DIR, "gemm_i8.cuh")) as f:
        text = f.read()
    tail = text[text.index("\ndone:"):text.index("tmem_dealloc_pair(tmem_base")]
    assert tail.index("__syncthreads()") < tail.index("if (abort_flag && threadIdx.x == 0) wait_out()") < tail.index("cluster_sync()")
