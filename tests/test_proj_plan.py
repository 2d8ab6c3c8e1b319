"""How the few-row projection shares out its launch (csrc/proj_lora.cuh, `plan`), compiled from the source with g++ and asked for devices that hold no cluster of
some widths, or none at all (no GPU needed): no division by what is not there, and no launch of a width that does not run."""

import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama_rs_b200", "csrc")

MAIN = r"""
// arguments: eight counts of resident clusters, then (rows, n, k) triples; prints cs kw clusters bytes two
template <int NT> void one(const int (&r)[2][4], int rows, int n, int k) {
  const Plan p = plan<NT>(r, rows, n, k);
  const int groups = k / 128;
  const size_t bytes = p.clusters ? Shape<NT>::bytes(128 * ((groups + p.cs - 1) / p.cs)) : 0;
  printf("%d %d %d %zu %d\n", p.cs, p.kw, p.clusters, bytes, bytes <= SMEM_TWO);
}
int main(int argc, char** argv) {
  int r[2][4];
  for (int i = 0; i < 8; ++i) r[i / 4][i % 4] = atoi(argv[1 + i]);
  for (int i = 9; i + 2 < argc; i += 3) {
    const int rows = atoi(argv[i]), n = atoi(argv[i + 1]), k = atoi(argv[i + 2]);
    rows <= 8 ? one<1>(r, rows, n, k) : rows <= 16 ? one<2>(r, rows, n, k) : rows <= 24 ? one<3>(r, rows, n, k) : one<4>(r, rows, n, k);
  }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    with open(os.path.join(CSRC, "proj_lora.cuh")) as f:
        s = f.read()
    line = lambda name: re.search(rf"^constexpr [^\n]*\b{name} = [^\n]*$", s, re.M).group(0)
    struct = s[s.index("template <int NT>\nstruct Shape {") :]
    struct = struct[: struct.index("\n};\n") + 4]
    fn = s[s.index("struct Plan {") :]
    fn = fn[: fn.index("\n}\n") + 3]
    consts = [line(n) for n in ("MAX_RANK", "CW", "SUB", "DEPTH", "PP", "SMEM_MAX", "V_BYTES")]
    d = tmp_path_factory.mktemp("plan")
    src = "\n".join(["#include <stdio.h>", "#include <stdlib.h>", "#include <stddef.h>", *consts, struct, fn, MAIN])
    (d / "plan.cpp").write_text(src)
    exe = str(d / "plan")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-o", exe, str(d / "plan.cpp")], check=True)
    return exe


FULL = (148, 74, 32, 14, 296, 148, 66, 30)  # what a full device may hold
SHAPES = [(rows, n, k) for rows in (1, 8, 9, 17, 32, 33, 300, 65535 * 32) for n in (1, 15, 257, 8192, 280_000) for k in (128, 256, 2048, 2176, 8192)]


def plans(exe, resident):
    args = [str(v) for v in (*resident, *(v for s in SHAPES for v in s))]
    out = subprocess.run([exe, *args], check=True, capture_output=True, text=True).stdout
    return [tuple(map(int, l.split())) for l in out.splitlines()]


@pytest.mark.parametrize("gone", [(), (3, 7), (2, 3, 6, 7), (0, 1, 2, 3), (4, 5, 6, 7), (0, 4), (0, 1, 4, 5), tuple(range(8))])
def test_no_plan_for_clusters_that_do_not_run(program, gone):
    resident = [0 if i in gone else v for i, v in enumerate(FULL)]
    got = plans(program, resident)
    assert len(got) == len(SHAPES)
    for (rows, n, k), (cs, kw, clusters, nbytes, two) in zip(SHAPES, got):
        if clusters == 0:
            assert gone, (rows, n, k)
            continue
        assert cs in (1, 2, 4, 8) and cs <= k // 128 and kw in (1, 2, 4) and nbytes <= 232448
        assert resident[4 * two + {1: 0, 2: 1, 4: 2, 8: 3}[cs]] > 0, (rows, n, k, cs)
        assert clusters <= -(-n // 16) * kw
    if len(gone) == 8:
        assert all(g[2] == 0 for g in got)
