"""How a prompt's work is cut, on the host: every sequence's items, states and cut tiles,
as the device finds them from the lengths, fit in what the launch and the workspace were
sized for without them."""
import random
import subprocess

import pytest

from prismkv_amd import build

PROGRAM = r"""
#include "prompt_plan.h"
#include <cstdio>
#include <vector>
using namespace prismkv;
int main() {
  long long sequences, kv_heads, group, row_bytes, fp32, slots, rows;
  while (scanf("%lld %lld %lld %lld %lld %lld", &sequences, &kv_heads, &group, &row_bytes, &fp32, &slots) == 6) {
    std::vector<long long> m(sequences), n(sequences);
    rows = 0;
    for (int b = 0; b < sequences; ++b) {
      if (scanf("%lld %lld", &m[b], &n[b]) != 2) return 1;
      rows += m[b];
    }
    const int tokens = tile_tokens(row_bytes);
    auto tiles = [&](int b) { return (m[b] * group + kTileRows - 1) / kTileRows; };
    auto key_tiles = [&](int b) { return (n[b] + tokens - 1) / tokens; };
    uint64_t work = 0;
    long long all = 0, items = 0, states = 0, cut = 0, longest = 0;
    for (int b = 0; b < sequences; ++b) work += tiles(b) * key_tiles(b) * kv_heads, all += tiles(b) * kv_heads;
    const PromptPlan plan = prompt_cuts(work, (int)all, fp32);
    for (int b = 0; b < sequences; ++b) {
      const long long most = plan.chunks((int)key_tiles(b));
      items += tiles(b) * most * kv_heads;
      if (most > 1) states += tiles(b) * most * kv_heads, cut += tiles(b) * kv_heads;
    }
    const PromptLayout l = prompt_layout(rows, sequences, kv_heads, group, 64, slots, row_bytes, fp32);
    // (a launch without states cuts nothing)
    if (!l.states) items = all, states = cut = 0;
    printf("%lld %lld %lld %lld %lld %lld\n", items, (long long)l.items, states, (long long)l.states, cut, (long long)l.cut_tiles);
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    path = tmp_path_factory.mktemp("plan")
    (path / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{build.CSRC}", str(path / "plan.cpp"), "-o", str(path / "plan")], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, (len(new), heads, group, row, int(fp32), slots))) + "\n" +
                         "\n".join(f"{m} {n}" for m, n in zip(new, lengths))
                         for new, lengths, heads, group, row, fp32, slots in cases)
        out = subprocess.run([str(path / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]

    return run


def check(plan, cases):
    found = plan(cases)
    assert len(found) == len(cases)
    for case, (items, most, states, room, cut, most_cut) in zip(cases, found):
        assert items <= most and states <= room and cut <= most_cut, (case[2:], len(case[0]), sum(case[0]))


def test_random_sequences(plan):
    rng = random.Random(1)
    cases = []
    for _ in range(400):
        count = rng.choice([1, 1, 2, 3, 9, 70, 500])
        slots = int(2 ** rng.uniform(0, 22))
        lengths = [rng.choice([0, 1, slots, rng.randint(0, slots), int(2 ** rng.uniform(0, 1 + slots.bit_length())) % slots])
                   for _ in range(count)]
        new = [rng.choice([0, 1, rng.randint(0, n), n, rng.randint(0, 300)]) for n in lengths]
        cases.append((new, lengths, rng.choice([1, 2, 8, 40]), rng.choice([1, 3, 4, 16, 200]), rng.choice([128, 256, 512, 1024]),
                      rng.random() < 0.3, slots))
    check(plan, cases)


def test_the_longest_sequences(plan):
    """2^30 slots (pages may stand in a table many times), of rows that are staged 32 at a time."""
    cases = []
    for rows in (100, 5000, 1 << 16, 1 << 20):
        for slots in ((1 << 29) + 12345678, 1 << 30):
            cases += [([rows], [slots], heads, group, row, False, slots)
                      for heads in (1, 2) for group in (1, 16) for row in (128, 512)]
            cases.append(([rows, 3], [slots, 4000], 2, 8, 512, False, slots))
    check(plan, cases)
