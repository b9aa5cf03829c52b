"""Whether strided memory meets itself or other such memory (csrc/strided.cuh), against marking its bytes."""
import os
import subprocess

SOURCE = r'''
#include "vectorstorekit_b200/csrc/strided.cuh"
#include <cstdio>
#include <random>
#include <vector>
using namespace vsk;
int main() {
  std::mt19937 g(1);
  auto pick = [&](int lo, int hi) { return (int64_t)(lo + (int)(g() % (unsigned)(hi - lo + 1))); };
  long long meets = 0, own = 0, n = 400000;
  for (long long i = 0; i < n; ++i) {
    const int64_t row = pick(0, 40), part = pick(0, 40);   // (often shared)
    auto make = [&]() {
      return Strided{pick(0, 120), pick(1, 5), g() % 2 ? row : pick(0, 60), pick(1, 4), g() % 2 ? part : pick(0, 60), pick(1, 9)};
    };
    const Strided a = make(), b = make();
    std::vector<int> marked(1000, 0);
    bool itself = false, other = false;
    auto bytes = [](const Strided& s, auto f) {
      for (int64_t r = 0; r < s.rows; ++r)
        for (int64_t o = 0; o < s.outer; ++o)
          for (int64_t k = 0; k < s.inner; ++k) f(s.at + r * s.row + o * s.part + k);
    };
    bytes(a, [&](int64_t at) { itself |= marked[at]++ > 0; });
    bytes(b, [&](int64_t at) { other |= marked[at] > 0; });
    if (itself != meets_itself(a) || other != meet(a, b) || other != meet(b, a)) {
      for (const Strided& s : {a, b})
        printf("at %d: %d rows %d apart, %d parts %d apart of %d\n", (int)s.at, (int)s.rows, (int)s.row, (int)s.outer, (int)s.part, (int)s.inner);
      return 1;
    }
    meets += other;
    own += itself;
  }
  if (meets < n / 4 || meets > n * 3 / 4 || own < n / 8) return 2;   // both answers occur
  // caches of a whole model in one block: keys and values of each layer side by side in a row, and of other widths
  const int64_t rows = 64, heads = 8, steps = 1024, step = 256, layers = 80;
  const int64_t keys = heads * steps * step, values = keys / 2, layer = keys + values, row = layers * layer;
  const int64_t base = 0x7f0000000000;
  for (int64_t i = 0; i < layers; ++i)
    for (int64_t j = 0; j < layers; ++j) {
      const Strided k{base + i * layer, rows, row, heads, steps * step, steps * step / 2}, v{base + j * layer + keys, rows, row, heads, steps * step / 2, steps * step / 2};
      if (meet(k, v) || meets_itself(k)) return 3;
      Strided into = v;
      into.at -= step;
      if (meet(k, into)) return 4;                     // between the heads' used halves
      into.at = base + i * layer + 3 * steps * step + steps * step / 2 - 1;
      if (!meet(k, into)) return 5;
    }
  return 0;
}
'''


def test_strided_memory_against_marked_bytes(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source, exe = tmp_path / "strided.cpp", str(tmp_path / "strided")
    source.write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", root, str(source), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
