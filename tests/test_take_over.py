"""Which items the CTAs of a prompt call do, run on the CPU with the kernel's own rule
(csrc/frn_take_over.h): CTAs take over the numbers of CTAs that were not launched, in whatever
order the hardware hands them out.  The rule that takes the first number without work for the end,
and throws the rest of the answers away, is run as a planted mistake."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "kimi26-h100-rmsnorm-swiglu-fusion_b200", "csrc")

HARNESS = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "frn_take_over.h"

struct Device {               // CTAs of a grid that have not been launched
  std::vector<int> waiting;
  std::mt19937 rng;
  int order;                  // 0 rising, 1 falling, 2 any
  int take() {                // -1: none left
    if (waiting.empty()) return -1;
    size_t at = order == 0 ? 0 : order == 1 ? waiting.size() - 1 : rng() % waiting.size();
    int number = waiting[at];
    waiting.erase(waiting.begin() + at);
    return number;
  }
};

struct Cta {
  int own;
  bool started = false, ended = false, asked = false, refused = false;
  int answer = -1;
};

int main(int argc, char** argv) {
  const int grid = atoi(argv[1]), work = atoi(argv[2]), sms = atoi(argv[3]);
  const bool broken = atoi(argv[6]);
  Device dev{{}, std::mt19937(atoi(argv[5])), atoi(argv[4])};
  for (int i = 0; i < grid; ++i) dev.waiting.push_back(i);
  std::vector<int> done(work, 0);
  std::vector<Cta> running;
  auto launch = [&] {         // an SM takes the lowest CTA that is left
    if (dev.waiting.empty()) return;
    Cta c;
    c.own = dev.waiting.front();
    dev.waiting.erase(dev.waiting.begin());
    running.push_back(c);
  };
  for (int i = 0; i < sms; ++i) launch();
  int bad = 0;
  while (!running.empty()) {
    const size_t at = dev.rng() % running.size();
    Cta& c = running[at];
    auto ask = [&] {
      if (c.asked || c.refused) bad = 1;  // two under way, or one after the end
      c.asked = true;
      c.answer = dev.take();
    };
    auto hear = [&](int& number) {
      if (!c.asked) { bad = 2; return false; }  // waits for good
      c.asked = false;
      c.refused = c.answer < 0;
      number = c.refused ? 0 : c.answer;
      return !c.refused;
    };
    int found = -1;
    auto has_work = [&](int number) {
      if (number < work) found = number;
      return number < work;
    };
    bool some;
    if (!broken) {
      some = frn::next_number(!c.started, c.own, ask, hear, has_work);
    } else {
      int number = c.own;
      const bool more = !c.started || hear(number);
      if (more) ask();
      some = more && has_work(number);
      if (!some && more) while (hear(number)) ask();
    }
    c.started = true;
    if (some) {
      ++done[found];
    } else {
      if (c.asked) bad = 3;   // an answer would arrive after the CTA's end
      running.erase(running.begin() + at);
      launch();
    }
    if (bad) break;
  }
  int lost = 0, twice = 0;
  for (int n : done) lost += n == 0, twice += n > 1;
  printf("%d %d %d\n", bad, lost, twice);
}
"""


@pytest.fixture(scope="module")
def simulate(tmp_path_factory):
    folder = tmp_path_factory.mktemp("take_over")
    source, binary = folder / "harness.cpp", folder / "harness"
    source.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(source), "-o", str(binary)],
                   check=True)

    def run(*args):
        out = subprocess.run([str(binary), *map(str, args)], check=True, capture_output=True,
                             text=True, timeout=60).stdout
        return tuple(map(int, out.split()))
    return run


@pytest.mark.parametrize("order", [0, 1, 2], ids=["rising", "falling", "any"])
@pytest.mark.parametrize("grid,work", [(1, 0), (1, 1), (5, 3), (148, 148), (400, 390), (500, 0),
                                       (1200, 1199), (1200, 700)])
def test_every_item_is_done_once(simulate, grid, work, order):
    for seed in range(5):
        assert simulate(grid, work, 148, order, seed, 0) == (0, 0, 0)
        assert simulate(grid, work, 3, order, seed, 0) == (0, 0, 0)


def test_the_first_number_without_work_is_not_the_end(simulate):
    lost = [simulate(1200, 700, 3, 2, seed, 1)[1] for seed in range(5)]
    assert any(lost)
