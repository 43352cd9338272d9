"""The loop of the device's bounded waits, compiled for the host: it ends when it should, with and
without a flag that calls it off."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "mlx-batch-invariant_b200", "csrc")

SOURCE = r"""
#include <cstdio>
#include "bounded_wait.h"

int main() {
  long long polls = 0, clock = 1000, looks = 0;
  auto now = [&] { ++looks; return clock += 7; };
  auto after = [&](long long n) { return [&polls, n] { return ++polls > n; }; };
  auto run = [&](long long ready_after, const volatile int* flag, long long budget) {
    polls = looks = 0;
    const bool ok = bi::bounded_wait(after(ready_after), now, flag, budget);
    std::printf("%d %lld %lld\n", ok, polls, looks);
  };
  const long long never = 1LL << 60;
  volatile int down = 0, up = 1;
  run(0, nullptr, 70);       // ready at once
  run(3, &up, 70);           // soon: the flag is not looked at yet
  run(1000, nullptr, 70);    // late, within the budget, nothing to call it off
  run(never, nullptr, 70);   // the budget ends it
  run(never, &down, 70);
  run(never, &up, 1LL << 50);  // the flag ends it
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_the_loop(tmp_path):
    src, exe = tmp_path / "wait.cpp", tmp_path / "wait"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-I" + CSRC, str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.returncode  # (a null flag that is read ends it with a signal)
    # the clock moves 7 a look: the 12th look is the first more than 70 behind the first
    assert r.stdout.split("\n")[:-1] == [
        "1 1 0", "1 4 0", "1 1001 3", "0 %d 12" % (12 * 256), "0 %d 12" % (12 * 256), "0 256 1"]


def test_the_kernels_use_it():
    """The drain of the paged kernel's products passes no flag."""
    with open(os.path.join(CSRC, "paged_sdpa_tc.cu")) as f:
        text = f.read()
    assert '#include "bounded_wait.h"' in text and "bounded_wait(" in text
    assert "*abort_flag ||" not in text
