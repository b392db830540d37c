"""How the copies of a CTA pair are brought to an end when a wait has run out (csrc/pair_copies.h), on the CPU: a model of the ring's barriers, with
both CTAs stopped anywhere."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nncv_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "pair_copies.h"
using namespace nncv_b200::pair_copies;

// The barrier of a stage on the first CTA: a phase completes with the first CTA's arrival, which announces two shares of bytes, and both shares.
struct Barrier {
  long long phase = 0;
  bool arrived = false;
  int shares = 0;
  void look() {
    if (arrived && shares == 2) { ++phase; arrived = false; shares = 0; }
  }
};

// waits(parity): whether a wait for that parity returns, as the hardware has it
static bool waits(const Barrier& b, unsigned parity) { return ((b.phase & 1) ^ 1) == parity; }

int main() {
  long long wrong = 0, unequal = 0, older = 0;
  srand(7);
  for (int run = 0; run < 200000; ++run) {
    const int stages = 1 + rand() % 20;
    const long long total = 1 + rand() % 70;
    std::vector<Barrier> full(stages);
    long long issued[2] = {0, 0}, used = 0;      // blocks whose copies are issued, and whose MMAs have ended
    std::vector<std::pair<int, int>> flying;     // copies under way: stage, CTA
    auto issue = [&](int cta) {
      const int st = (int)spot_of(issued[cta]++, stages).stage;
      if (cta == 0) { if (full[st].arrived) ++wrong; full[st].arrived = true; }
      flying.push_back({st, cta});
    };
    auto land = [&](size_t k) {
      Barrier& b = full[flying[k].first];
      if (++b.shares > 2) ++wrong;
      b.look();
      flying[k] = flying.back();
      flying.pop_back();
    };
    for (int steps = rand() % 400; steps > 0; --steps) {
      const int what = rand() % 4;
      if (what < 2 && issued[what] < total && issued[what] < used + stages) issue(what);        // the stage was given back
      else if (what == 2 && !flying.empty()) land(rand() % flying.size());
      else if (what == 3 && used < issued[0] && used < issued[1] && full[used % stages].phase > used / stages) ++used;
    }
    unequal += issued[0] != issued[1];
    const long long end0 = meet_at(issued[0], issued[1]), end1 = meet_at(issued[1], issued[0]);
    if (end0 != end1 || end0 - issued[0] > stages || end0 - issued[1] > stages) ++wrong;
    // without meeting: the first CTA's waits for the stages that it used itself, copies left behind
    if (issued[1] > issued[0]) ++older;
    for (int cta = 0; cta < 2; ++cta)
      while (issued[cta] < end0) issue(cta);
    // the first CTA's waits all return, whatever the order in which the copies land, and not before the last has
    while (!flying.empty()) {
      bool all = true;
      for (long long n = wait_from(end0, stages); n < end0; ++n) all = all && waits(full[spot_of(n, stages).stage], spot_of(n, stages).parity);
      if (all) ++wrong;
      land(rand() % flying.size());
    }
    for (long long n = wait_from(end0, stages); n < end0; ++n)
      if (!waits(full[spot_of(n, stages).stage], spot_of(n, stages).parity)) ++wrong;
    for (int st = 0; st < stages; ++st)
      if (full[st].arrived || full[st].shares) ++wrong;
  }
  printf("%lld %lld %lld\n", wrong, unequal, older);
}
"""


def test_no_copy_is_left_under_way(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", "t.cpp", "-o", "t"], cwd=tmp_path, check=True)
    wrong, unequal, older = map(int, subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split())
    assert wrong == 0
    assert unequal > 50000 and older > 20000      # the CTAs stood apart, and the second ahead of the first
