"""The cases of tests/rows_cases.py against the plan, in a host build: each is carried out by the form that it stands for, and every form is among them."""
import os
import shutil
import subprocess

import pytest

from tests.rows_cases import CASES, KINDS, NEVER, SHARES, TILES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pika-h3-flex_amd", "csrc")

# one line a case: kind, M, N, K in; rows and columns of the tiles, cuts, turns of the busiest workgroup, chunks of the shortest part out
PROGRAM = r"""
#include "pkh3_rows_index.h"
#include <stdio.h>
using namespace pkh3;
int main() {
  int kind, M, N, K;
  while (scanf("%d %d %d %d", &kind, &M, &N, &K) == 4) {
    const int mode = kind == 1 ? kGated : kind == 3 ? kGrad : kind == 4 ? kGatedGrad : kPlain;
    const ProductPlan p = plan_product(M, N, K, kind < 2, mode, mode >= kGrad, kind == 5);
    const ProductShare& s = p.share;
    if (p.thin) printf("%d %d 0 1 %d\n", thin_rows(M), mode == kGated || thin_narrow(M, N) ? 16 : 32, (K + kChunk - 1) / kChunk);
    else printf("%d %d %d %d %d\n", 32 * p.tb, 32 * p.fb, s.cuts, s.rounds + (s.rest ? part_turns(s) : 0), s.chunks / s.cuts);
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_every_form_is_among_the_cases(tmp_path):
    src, exe = tmp_path / "forms.cpp", tmp_path / "forms"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    asked = "\n".join(f"{KINDS.index(kind)} {M} {N} {K}" for kind, _, _, M, N, K in CASES)
    got = subprocess.run([str(exe)], input=asked, capture_output=True, text=True, check=True).stdout.splitlines()
    assert len(got) == len(CASES)
    for case, line in zip(CASES, got):
        rows, columns, cuts, turns, chunks = map(int, line.split())
        share = "thin" if cuts == 0 else f"{'cut' if cuts > 1 else 'whole'} {'multi' if turns > 1 else 'single'}"
        assert (case[1], case[2]) == ((rows, columns), share), (case, line)
        assert case[5] % 64 and (chunks >= 9 or (share == "thin" and case[3] > 64)), (case, line)
    there = {c[:3] for c in CASES}
    tiles = {(kind, tile, share) for kind in KINDS for tile in TILES for share in SHARES}
    few = {("plain", (rows, columns), "thin") for rows in (16, 32, 64) for columns in (16, 32)} | {("gated", (rows, 16), "thin") for rows in (16, 32, 64)}
    assert there == tiles - NEVER | few
