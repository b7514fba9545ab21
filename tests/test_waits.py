"""The give-up protocol of waits that a group of threads acts on together (csrc/agree.cuh), compiled for
the host: whatever another thread writes meanwhile, all of the group go on or all leave."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

HARNESS = r"""
#include <atomic>
#include <barrier>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>
#include "agree.cuh"

// argv[1]: when an outsider raises the abort flag: 0 never, 1 before the leader looks, 2 behind the
// barrier, when the first thread has its answer and the others have not
int main(int, char** argv) {
  const int when = std::atoi(argv[1]);
  constexpr int N = 4;
  std::barrier<> gate(N);
  volatile int answer = -1;
  std::atomic<int> abort_flag{when == 1}, first_out{0}, reads_behind{0};
  int got[N];
  std::vector<std::thread> group;
  for (int i = 0; i < N; ++i)
    group.emplace_back([&, i] {
      bool behind = false;
      got[i] = moe::agree(i == 0, &answer, [&] {
        if (behind || i != 0) ++reads_behind;
        return abort_flag.load() == 0;
      }, [&] {
        gate.arrive_and_wait();
        behind = true;
        if (i == 0) return;
        while (!first_out) std::this_thread::yield();
        if (when == 2) abort_flag = 1;
      });
      if (i == 0) first_out = 1;
    });
  for (auto& t : group) t.join();
  for (int i = 0; i < N; ++i) std::printf("%d ", got[i]);
  std::printf("%d\n", reads_behind.load());
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    where = tmp_path_factory.mktemp("agree")
    (where / "main.cpp").write_text(HARNESS)
    subprocess.run([shutil.which("g++") or "c++", "-std=c++20", "-O1", "-pthread", "-I",
                    os.path.join(ROOT, "nanospeaker_b200", "csrc"), str(where / "main.cpp"), "-o",
                    str(where / "main")], check=True)
    return str(where / "main")


@pytest.mark.parametrize("when,go", [(0, 1), (1, 0), (2, 1)])
def test_a_group_goes_on_or_leaves_as_one(harness, when, go):
    out = subprocess.run([harness, str(when)], check=True, capture_output=True, text=True, timeout=60)
    *got, reads_behind = map(int, out.stdout.split())
    assert got == [go] * 4            # (an abort raised behind the barrier counts at the next wait)
    assert reads_behind == 0


def test_waits_end_early_for_waits_that_ran_out_and_not_for_reported_inputs(tmp_path):
    """csrc/status.cuh: an expert id or a run start out of range, reported by this call or an earlier one, stops
    nobody."""
    (tmp_path / "main.cpp").write_text('#include "status.cuh"\n#include <cstdio>\nint main() {\n'
                                       "  for (int code = -1; code < 5; ++code)\n"
                                       '    std::printf("%d ", moe::status_ends_waits(code));\n}\n')
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-I",
                    os.path.join(ROOT, "nanospeaker_b200", "csrc"), str(tmp_path / "main.cpp"), "-o",
                    str(tmp_path / "main")], check=True)
    out = subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["0", "0", "1", "0", "0", "0"]


def test_unseen_uses_are_the_copies_that_may_be_in_flight(tmp_path):
    """csrc/ring.cuh against the ring itself: a reader that gives up at use `first` has seen all before; a writer that
    waits for a stage to be freed can have started `stages` more. Each with the parity of the phase that it ends
    (a barrier's phases count from 0, one per use of its stage)."""
    (tmp_path / "main.cpp").write_text(
        '#include "ring.cuh"\n#include <cstdio>\n#include <cstdlib>\nint main(int, char** v) {\n'
        "  moe::unseen_uses(std::atoi(v[1]), std::atoi(v[2]), [](uint32_t s, uint32_t p) {\n"
        '    std::printf("%u.%u ", s, p);\n  });\n}\n')
    exe = str(tmp_path / "main")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-I",
                    os.path.join(ROOT, "nanospeaker_b200", "csrc"), str(tmp_path / "main.cpp"), "-o", exe], check=True)
    for stages in (1, 2, 3, 6):
        for first in range(20):
            freed, started, phase, flying = set(range(stages)), 0, [-1] * stages, {}
            while started % stages in freed:          # the writer: a stage's first use needs no one
                at = started % stages
                if started < first:                   # (seen, and given back)
                    phase[at] += 1
                else:
                    freed.discard(at)
                    phase[at] += 1
                    flying[at] = phase[at] & 1
                started += 1
            out = subprocess.run([exe, str(first), str(stages)], check=True, capture_output=True, text=True).stdout
            assert dict(map(int, w.split(".")) for w in out.split()) == flying and len(out.split()) == stages
