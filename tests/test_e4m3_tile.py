"""The choice of tile and split of the 8-bit product (csrc/e4m3_tile.h), on the CPU, for GPUs that hold different numbers of clusters."""
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nncv_b200", "csrc")
TILES = [(128, 64), (128, 128), (256, 128), (256, 256)]

PROGRAM = r"""
#include <cstdio>
#include "e4m3_tile.h"
using namespace nncv_b200::e4m3;
int main() {
  int M, N, KB, sms, f[2][4];
  while (scanf("%d %d %d %d %d %d %d %d %d %d", &M, &N, &KB, &sms, f[0] + 1, f[0] + 2, f[0] + 3, f[1] + 1, f[1] + 2, f[1] + 3) == 10) {
    int of[2][9] = {};
    for (int i = 0; i < 2; ++i) {
      of[i][1] = sms;
      for (int k = 1; k < 4; ++k) of[i][1 << k] = f[i][k];
    }
    const Room room{{of[0], of[1]}, sms};
    const Choice c = choose(M, N, KB, room);
    printf("%d %d", c.tile, c.splits);
    for (int i = -1; i <= 4; ++i)
      for (int s = 0; s <= 16; ++s) printf(" %d", (int)fits(i, s, M, N, KB, room));
    printf("\n");
  }
}
"""


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    d = tmp_path_factory.mktemp("tile")
    (d / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", "t.cpp", "-o", "t"], cwd=d, check=True)

    def run(cases):
        """cases: (M, N, blocks of K, SMs, clusters of two, four and eight of either single tile) -> ((tile, split), {(tile, split) that fit})."""
        text = "\n".join(" ".join(map(str, (m, n, kb, sms, *a, *b))) for m, n, kb, sms, a, b in cases)
        out = []
        for line in subprocess.run([str(d / "t")], input=text, capture_output=True, text=True, check=True).stdout.splitlines():
            v = list(map(int, line.split()))
            out.append(((v[0], v[1]), {(i - 1, s) for i in range(6) for s in range(17) if v[2 + i * 17 + s]}))
        return out

    return run


def room(rng):
    sms = rng.choice((148, 148, 132, 160, 16))
    return sms, *[tuple(rng.randint(max(1, sms // s // 2), sms // s) for s in (2, 4, 8)) for _ in range(2)]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def test_what_fits_and_what_is_chosen(choose):
    rng = random.Random(3)
    cases = [(_log(rng, 1, 9000), _log(rng, 1, 9000), _log(rng, 1, 70), *room(rng)) for _ in range(4000)]
    cases += [(1, 1, 1, 148, (74, 36, 16), (74, 36, 16)), (2 ** 30, 1, 1, 148, (74, 36, 16), (74, 36, 16)), (1, 2 ** 30, 2 ** 23, 148, (74, 36, 16), (74, 36, 16))]
    seen = set()
    for (m, n, kb, sms, a, b), (got, fit) in zip(cases, choose(cases)):
        want = set()
        for i, (tm, tn) in enumerate(TILES):
            tiles = -(-m // tm) * -(-n // tn)
            for k, s in enumerate((1, 2, 4, 8)):
                if s == 1 or (i < 2 and tiles <= (a, b)[i][k - 1] and kb >= s):
                    want.add((i, s))
        assert fit == want and got in fit
        seen.add(got)
    assert seen == {(i, s) for i in range(2) for s in (1, 2, 4, 8)} | {(2, 1), (3, 1)}    # nothing stays that no product reaches
