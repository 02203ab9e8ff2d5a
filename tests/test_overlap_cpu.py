"""Whether two strided tensors share an element (plast_b200/csrc/overlap.h), against the sets of their elements."""
import itertools
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

PROBE = r"""
#include "overlap.h"
#include <stdio.h>
static int read_tensor(Tensor *t) { // offset in bytes, dims, shape, strides
  long long offset, dims, v;
  *t = Tensor{};
  if (scanf("%lld %lld", &offset, &dims) != 2) return 0;
  t->data = (void *)(1000000 + offset);
  t->ndim = dims;
  for (int d = 0; d < dims; ++d) { if (scanf("%lld", &v) != 1) return 0; t->shape[d] = v; }
  for (int d = 0; d < dims; ++d) { if (scanf("%lld", &v) != 1) return 0; t->strides[d] = (u64)v; }
  return 1;
}
int main() {
  Tensor a, b;
  while (read_tensor(&a) && read_tensor(&b))
    printf("%d%d%d\n", pb::share_an_element(pb::extent_of(&a), pb::extent_of(&b)), pb::same_elements(&a, &b), pb::has_repeated_elements(&a));
  return 0;
}
"""


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    folder = tmp_path_factory.mktemp("overlap")
    (folder / "probe.cpp").write_text(PROBE)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", f"-I{ROOT / 'include'}", f"-I{ROOT / 'plast_b200' / 'csrc'}",
                    str(folder / "probe.cpp"), "-o", str(folder / "probe")], check=True)

    def ask(pairs):
        lines = [" ".join(map(str, [off, len(shape), *shape, *strides])) for pair in pairs for off, shape, strides in pair]
        out = subprocess.run([str(folder / "probe")], input="\n".join(lines) + "\n", text=True, check=True, capture_output=True)
        return [[c == "1" for c in line] for line in out.stdout.split()]
    return ask


def elements(tensor):
    """The bytes of every element, by index."""
    offset, shape, strides = tensor
    return [offset + 4 * sum(i * s for i, s in zip(index, strides)) for index in itertools.product(*map(range, shape))]


def share(a, b):
    one, other = elements(a), elements(b)
    if (a[0] - b[0]) % 4:       # elements out of step: whether the ranges of the two meet
        return bool(one and other) and min(one) < max(other) + 4 and min(other) < max(one) + 4
    return not set(one).isdisjoint(other)


def test_small_tensors_of_any_strides(probe):
    rng = random.Random(3)

    def tensor():
        dims = rng.randint(0, 4)
        shape = [rng.choice([0, 1, 2, 3, 4]) if rng.random() < 0.2 else rng.randint(1, 4) for _ in range(dims)]
        strides = [rng.choice([0, 1, 2, 3, 4, 5, 7, 12, 16, 30, -1, -6]) for _ in range(dims)]
        return 4 * rng.randint(0, 60) + (2 if rng.random() < 0.05 else 0), shape, strides

    pairs = [(tensor(), tensor()) for _ in range(4000)]
    found = probe(pairs)
    assert [f[0] for f in found] == [share(*p) for p in pairs]
    assert 500 < sum(f[0] for f in found) < 3500


def test_slices_of_a_fused_row(probe):
    """Queries, keys and values of one row, large as in use, share nothing; a slice that begins a head early does."""
    t, h, kv, d = 4096, 32, 8, 128
    row = (h + 2 * kv) * d

    def heads(first, n, rows=t):
        return 4 * first * d, [2, rows, n, d], [t * row, row, d, 1]

    q, k, v = heads(0, h), heads(h, kv), heads(h + kv, kv)
    by_heads = (q[0], [2, h, t, d], [t * row, d, row, 1])
    early = heads(h - 1, kv)
    odd = (4 * 5, [2, t, h, d], [t * row, row, d, 1])
    answers = probe([(q, k), (k, v), (by_heads, v), (q, early), (early, k), (q, q), (q, by_heads), (q, odd)])
    assert [a[0] for a in answers] == [False, False, False, True, True, True, True, True]
    assert [a[1] for a in answers] == [False] * 5 + [True, False, False]


def test_elements_at_two_indices(probe):
    rng = random.Random(4)
    tensors = []
    for _ in range(4000):
        dims = rng.randint(0, 4)
        shape = [rng.choice([0, 1, 2, 3, 4]) if rng.random() < 0.2 else rng.randint(1, 4) for _ in range(dims)]
        strides = [rng.choice([1, 2, 3, 4, 5, 7, 12, 16, 48, -1, -6]) if rng.random() < 0.95 else 0 for _ in range(dims)]
        tensors.append((0, shape, strides))
    found = [a[2] for a in probe([(t, t) for t in tensors])]
    assert found == [len(set(elements(t))) < len(elements(t)) for t in tensors]
    assert 500 < sum(found) < 3500
    large = [(0, [2, 4096, 32, 128], [4096 * 6144, 6144, 128, 1]), (0, [2, 32, 4096, 128], [4096 * 6144, 128, 6144, 1]),
             (0, [2, 4096, 32, 128], [4096 * 6144, 6000, 192, 1]), (0, [8192, 65536], [65535, 1])]
    assert [a[2] for a in probe([(t, t) for t in large])] == [False, False, True, True]
