"""csrc/once.h, which guards the kernels' first call on a device, under host
threads (no GPU needed)."""
import os
import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

#include "once.h"

int main() {
  static amass::DeviceOnce once;
  std::atomic<int> ready[3] = {}, calls[3] = {}, bad{0};
  std::vector<std::thread> all;
  for (int i = 0; i < 24; ++i)
    all.emplace_back([&, i] {
      const int dev = i % 3;
      const bool ok = once.run(dev, [&] {
        calls[dev]++;
        std::this_thread::sleep_for(std::chrono::milliseconds(30));
        ready[dev] = 1;
        return true;
      });
      if (!ok || !ready[dev]) bad++;
    });
  for (auto& t : all) t.join();
  for (int d = 0; d < 3; ++d)
    if (calls[d] != 1) return 1;
  if (bad) return 2;
  // a failure is not taken for done, and leaves the other devices alone
  int tries = 0;
  const auto set = [&] { return ++tries > 2; };
  if (once.run(5, set) || once.run(5, set)) return 3;
  if (!once.run(5, set) || !once.run(5, set) || tries != 3) return 4;
  if (!once.run(0, [] { return false; })) return 5;
  int far = 0;
  for (int k = 0; k < 2; ++k)
    if (!once.run(69, [&] { return ++far > 0; })) return 6;
  return far == 2 ? 0 : 7;
}
"""


def test_threads_wait_for_the_setup(tmp_path):
    src, exe = tmp_path / "once.cpp", tmp_path / "once"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I",
                    os.path.join(ROOT, "amass_kv_b200", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    for _ in range(5):
        assert subprocess.run([str(exe)], timeout=60).returncode == 0
