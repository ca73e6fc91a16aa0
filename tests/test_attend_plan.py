"""How prompt attention is cut into equal shares (csrc/lw_attend_plan.h), replayed on the CPU: the closed form of the units in
front of a pair against the sum over the pairs, and the shares against the formula that names a unit's block.  Compiled with the
compiler's checks for undefined behaviour, so an overflow fails too."""
import os
import subprocess

import pytest

from tests.conftest import ROOT

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <random>

#include "lw_attend_plan.h"

using namespace lw;

static long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// from the definition: the tokens of pair i see max(0, p - window + 1) .. p each
static long long units_of_pair(const PromptShape& s, const PromptSeq& q, int i, const PairRange& r) {
  const long long p0 = static_cast<long long>(q.len) - q.rows, t0 = static_cast<long long>(i) * s.pair_tokens;
  const long long t1 = t0 + s.pair_tokens < q.rows ? t0 + s.pair_tokens : q.rows;
  const long long hi = p0 + t1;
  long long lo = s.window > 0 ? p0 + t0 - s.window + 1 : 0;
  if (lo < 0) lo = 0;
  const long long first = lo / kPosBlock, last = hi > lo ? ceil_div(hi, kPosBlock) : first + 1;
  if (r.first != first || r.last != last || r.lo != lo || (hi > lo && r.hi != hi)) {
    std::printf("pair %d of %d rows at %d, window %d, %d tokens: blocks %d..%d, not %lld..%lld\n", i, q.rows, q.len, s.window, s.pair_tokens, r.first, r.last, first, last);
    std::exit(1);
  }
  return s.lead + last - first;
}

static void check(const PromptShape& s, const PromptSeq& q, std::mt19937& rng) {
  const int pairs = prompt_pairs(s, q);
  long long sum = 0;
  for (int i = 0; i < pairs; ++i) {
    if (pairs < 40 || rng() % 16 == 0 || i + 1 == pairs)
      if (const long long got = units_before(s, q, i); got != sum) {
        std::printf("%d rows at %d, window %d, %d tokens, lead %d: %lld units before pair %d, not %lld\n", q.rows, q.len, s.window, s.pair_tokens, s.lead, got, i, sum);
        std::exit(1);
      }
    sum += units_of_pair(s, q, i, pair_range(s, q, i));
  }
  if (const long long got = units_before(s, q, pairs); got != sum) {
    std::printf("%d rows at %d, window %d, %d tokens, lead %d: %lld units, not %lld\n", q.rows, q.len, s.window, s.pair_tokens, s.lead, got, sum);
    std::exit(1);
  }
}

int main(int, char** argv) {
  std::mt19937 rng(std::atoi(argv[1]));
  const int runs = std::atoi(argv[2]);
  auto upto = [&](int n) { return static_cast<int>(rng() % (static_cast<unsigned>(n) + 1u)); };
  const int most = 2147483647;
  for (int n = 0; n < runs; ++n) {
    PromptShape s;
    s.pair_tokens = 2 * (128 / (1 + upto(upto(127))));
    s.lead = upto(3);
    switch (upto(5)) {
      case 0: s.window = 0; break;
      case 1: s.window = 1 + upto(5000); break;
      case 2: s.window = most - upto(3); break;
      case 3: s.window = most - upto(400); break;
      case 4: s.window = (1 << 30) + upto((1 << 30) - 1); break;
      default: s.window = 1 + upto(most - 1);
    }
    PromptSeq q;
    q.len = upto(3) ? upto(upto(20000)) : upto(1 << 30);
    q.rows = 1 + upto(upto(3) ? upto(3000) : 300 * s.pair_tokens);
    check(s, q, rng);
  }
  // many rows before position 0
  for (int window : {0, 1, 1000, most}) check({2, window, 2}, {1 << 20, 5}, rng);
  // shares: unit u is block floor(((u + 1) blocks - 1) / units)'s
  for (int n = 0; n < runs; ++n) {
    const int blocks = 1 + upto(200);
    const long long units = blocks + (upto(3) ? upto(5000) : static_cast<long long>(upto(most)) * upto(1 << 20));
    for (int c = 0; c < blocks; ++c) {
      const long long u0 = share(units, c, blocks), u1 = share(units, c + 1, blocks);
      if (u0 >= u1 || ((u0 + 1) * blocks - 1) / units != c || (u1 * blocks - 1) / units != c) {
        std::printf("block %d of %d, %lld units: %lld..%lld\n", c, blocks, units, u0, u1);
        return 1;
      }
    }
    if (share(units, 0, blocks) != 0 || share(units, blocks, blocks) != units) return 1;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "lazyweights_b200", "csrc"),
                    str(at / "plan.cpp"), "-o", str(at / "plan")], check=True)
    return str(at / "plan")


@pytest.mark.parametrize("seed", range(4))
def test_units_and_shares(program, seed):
    done = subprocess.run([program, str(seed), "4000"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
