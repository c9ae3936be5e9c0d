"""Which kernel the sizes of the GPU tests take (csrc/chosen_rules.hpp, compiled for the host): each of them is reached by a test that is
named after it, whatever becomes of the rules; and the workspace of x A^T holds the shares of every call that it was asked for."""
import os
import subprocess

import pytest

from tests import test_gpu_adapters, test_gpu_adapters_shares, test_gpu_experts, test_gpu_experts_activations

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "intel-extension-for-tensorflow_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "chosen_rules.hpp"
using namespace itexhip;
int main() {
  char what;
  while (std::scanf(" %c", &what) == 1) {
    if (what == 'p') {          // product: tokens top_k experts K N up gated -> kernel
      long t, k, e, K, N; int up, gated;
      if (std::scanf("%ld %ld %ld %ld %ld %d %d", &t, &k, &e, &K, &N, &up, &gated) != 7) return 1;
      const ProductSizes s{t * k, k, (int)e, (K + 63) / 64 * 64, N, up != 0, gated != 0};
      const char* const names[] = {"strips of 4", "strips of 8", "tiles of 128", "tiles of 256"};
      if (!up && few_down(s)) std::puts("one launch");
      else if (up && few_up(s)) std::puts(few_strips(s) ? "fused strips of 8" : "fused strips of 4");
      else std::puts(names[product_kernel(s)]);
    } else if (what == 'a') {   // adapters: tokens adapters rank n_slices in columns width -> once long_tiles splits long_expand
      long t, n, rank, slices, in, columns; int width;
      if (std::scanf("%ld %ld %ld %ld %ld %ld %d", &t, &n, &rank, &slices, &in, &columns, &width) != 7) return 1;
      std::printf("%d %d %d %d\n", one_launch(t, n, rank, slices, in, columns), long_tiles(t, n), splits_of(t, n, slices * shrink_parts(rank), in), long_expand(t, n, columns, width));
    } else if (what == 'w') {   // every call of fewer tokens fits: tokens * shares against the rows of the middle
      long bad = 0, most = 0;
      for (int n : {1, 2, 5, 64, 1000}) for (int parts : {1, 2, 4, 16}) for (long in : {1, 256, 257, 1024, 4096, 1 << 20}) {
        most = 0;
        for (long t = 1; t < 2000000; t += t < 70000 ? 13 : 9973) {
          const long rows = t * splits_of(t, n, parts, in);
          if (rows > middle_rows(t) || middle_rows(t) < most) ++bad;
          most = middle_rows(t);
        }
      }
      std::printf("%ld\n", bad);
    }
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cc").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(d / "rules.cc"), "-o", str(d / "rules")], check=True)

    def run(lines):
        return subprocess.run([str(d / "rules")], input="\n".join(" ".join(str(v) for v in l) for l in lines), check=True, stdout=subprocess.PIPE, text=True).stdout.splitlines()
    return run


@pytest.mark.parametrize("kernel", list(test_gpu_experts_activations.SIZES))
def test_activations_reach_the_kernel_they_are_named_after(ask, kernel):
    t, k, e, K, N = test_gpu_experts_activations.SIZES[kernel]
    for got in ask([("p", t, k, e, K, N, 1, gated) for gated in (0, 1)]):
        assert got.startswith(kernel.split(",")[0]), got


def test_every_kernel_of_the_products_is_reached(ask):
    sizes = test_gpu_experts.SIZES
    activations = test_gpu_experts_activations.SIZES.values()
    up = set(ask([("p", t, k, e, K, N, 1, gated) for t, k, e, K, N in [s[:5] for s in sizes] + list(activations) for gated in (0, 1)]))
    assert up == {"fused strips of 4", "fused strips of 8", "strips of 4", "strips of 8", "tiles of 128", "tiles of 256"}
    down = set(ask([("p", t, k, e, K, N, 0, 0) for t, k, e, K, N, _ in sizes]))
    assert down == {"one launch", "strips of 4", "strips of 8", "tiles of 128", "tiles of 256"}


def test_shares_reach_tiles_of_64_places(ask):
    lines = [("a", t, n, rank, len(ends), K, ends[-1], 512) for t, n, rank, K, ends, _ in test_gpu_adapters_shares.SIZES]
    rules = [[int(v) for v in l.split()] for l in ask(lines)]
    assert all(once == 0 and long and splits > 1 for once, long, splits, _ in rules), rules
    assert {r[3] for r in rules} == {0, 1}              # the product with B in tiles of 64 and of 16
    assert len({r[2] for r in rules}) >= 3
    for (t, n, rank, K, ends, _), (_, _, splits, _) in zip(test_gpu_adapters_shares.SIZES, rules):
        steps = (K + 31) // 32
        if K == 1096:
            assert steps % splits != 0                   # a last share that is shorter
    other = [[int(v) for v in l.split()] for l in ask([("a", t, n, rank, len(ends), K, ends[-1], 512) for t, n, rank, K, ends, _ in test_gpu_adapters.SIZES])]
    assert any(r[0] for r in other) and any(r[1] for r in other) and any(r[2] > 1 for r in other)


def test_the_middle_holds_the_shares_of_every_call(ask):
    assert ask([("w",)]) == ["0"]
