"""The scratch of the feature operators' sort holds every list up to the length
it was made for: a call taken in turns sorts its shorter last turn in the
scratch of a full one.  Host arithmetic alone, no GPU."""
import os
import subprocess

import pytest

from ns_fps_b200 import build
from tests.test_feature_host import _attention, _rows
from tests import capi

# pairs of a full turn and of the last one
TURNS = [(786_432, 393_216), ((1 << 19) + 1, 1 << 19), (1 << 21, 1 << 19), (1 << 24, 1 << 19),
         (1 << 24, 300_000), (1 << 19, 5000), (4097, 4096), (5000, 1), (1, 1)]

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "nsfps_sort.cuh"
int main(int argc, char **argv) {
  using namespace nsfps;
  for (int i = 1; i + 1 < argc; i += 2) {
    const uint32_t n = strtoul(argv[i], 0, 10), tail = strtoul(argv[i + 1], 0, 10);
    SortScratch s;
    WorkCarver c((void *)(1ull << 20));
    s.carve(c, n);
    const unsigned long long have = s.total - s.hist;
    const unsigned long long want = 256ull * ceil_div(tail, kSortTile);
    printf("%llu %llu\n", have, want);
  }
}
"""


def test_every_turn_fits_the_digit_counts(tmp_path):
    """One count per digit value and tile, of the turn's own tiles."""
    if not os.path.exists(build.NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "sizes.cu", tmp_path / "sizes"
    src.write_text(PROGRAM)
    subprocess.run([build.NVCC, *build.NVCC_FLAGS, str(src), "-o", str(exe)], check=True)
    args = [str(x) for turn in TURNS for x in turn]
    lines = subprocess.run([str(exe), *args], check=True, capture_output=True, text=True).stdout
    for (full, tail), line in zip(TURNS, lines.splitlines(), strict=True):
        have, want = map(int, line.split())
        assert have >= want, f"a turn of {tail} in the scratch of {full}: {want} counts, {have} fit"


def test_scratch_of_a_longer_list_is_no_smaller():
    for a, b in [(1 << 19, (1 << 19) + 1), (4096, 4097), (393_216, 786_432), (1 << 19, 1 << 20)]:
        assert (capi.gather_rows_grad_workspace(_rows(count=a)) <=
                capi.gather_rows_grad_workspace(_rows(count=b)))
        for backward in (False, True):
            few, more = (_attention(queries=n, top=1, heads=1, kv_heads=1, head_dim=8,
                                    keys=10_000_000) for n in (a, b))
            assert (capi.block_attention_workspace(few, backward) <=
                    capi.block_attention_workspace(more, backward))
