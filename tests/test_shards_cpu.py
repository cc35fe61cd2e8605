"""A call's work on several devices when threads cannot be started (csrc/shards.h)."""
import os
import shutil
import subprocess

import pytest

from tests.conftest import ROOT

PROGRAM = r"""
#include <sys/resource.h>
#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <string>
#include "shards.h"

int main(int, char **argv) {
  const int n = std::atoi(argv[1]);
  const long room = std::atol(argv[2]);  // of address space, in MiB; 0 for any
  if (room) {
    long pages = 0;
    std::ifstream("/proc/self/statm") >> pages;
    rlimit r;
    r.rlim_cur = r.rlim_max = pages * 4096 + (room << 20);
    setrlimit(RLIMIT_AS, &r);
  }
  std::vector<int> done(n), mine(n), here(n);
  const auto caller = std::this_thread::get_id();
  auto work = [&](int i) {
    ++done[i];
    mine[i] = std::this_thread::get_id() == caller;
  };
  mfb200::run_shards(n, work, [&](int i) {
    here[i] = 1;
    work(i);
  });
  for (int i = 0; i < n; ++i) std::printf("%d%d%d ", done[i], mine[i], here[i]);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("shards")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "metalfish_b200", "csrc"),
                    "-o", str(d / "main"), str(d / "main.cpp")], check=True)

    def run(n, room):
        out = subprocess.run(["bash", "-c", 'ulimit -s 8192; exec "$@"', "run", str(d / "main"), str(n), str(room)],
                             check=True, capture_output=True, text=True, timeout=60)
        return out.stdout.split()
    return run


def test_each_shard_on_a_thread_of_its_own(program):
    assert program(1, 0) == ["110"]
    assert program(5, 0) == ["100"] * 5


def test_shards_without_a_thread_run_on_the_calling_one(program):
    assert program(4, 2) == ["111"] * 4  # no room for a stack of 8 MiB
    some = program(6, 20)  # room for one or two
    assert some[0] == "100" and some[-1] == "111" and set(some) == {"100", "111"}
