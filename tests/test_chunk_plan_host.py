"""How chunk attention is cut into CTAs: launch_plan.h compiled for the host, over the range of sizes that the call takes."""
import subprocess

import pytest

PROGRAM = r"""
#include <cstdio>
#include "launch_plan.h"
int main()
{
    long long n = 0, b, kv, t, tile, ctx;
    while (std::scanf("%lld %lld %lld %lld %lld", &b, &kv, &t, &tile, &ctx) == 5) {
        const auto p = gb200::chunk_plan(int(b), int(kv), int(t), int(tile), int(ctx));
        std::printf("%d %d %d\n", p.tiles, p.units, p.splits);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    from pathlib import Path

    import garnet_b200
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(Path(garnet_b200.__file__).parent / "csrc"), str(folder / "plan.cpp"), "-o", str(folder / "plan")], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(folder / "plan")], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        return [tuple(map(int, line.split())) for line in out if line]
    return run


def test_plans_of_all_sizes_are_kinds_that_exist(plan):
    cases = [(b, kv, t, tile, ctx) for b in (1, 2, 7, 24, 300, 65535) for kv in (1, 4, 8, 128) for t in (1, 5, 200, 4096, 1 << 20)
             for tile in (1, 16, 64, 128) for ctx in (1, 64, 4096, 131072, 0x7fff0000) if t >= b or t == 1]
    for case, (tiles, units, splits) in zip(cases, plan(cases), strict=True):
        assert (tiles, units) in ((1, 2), (1, 6), (2, 5)), case
        assert splits in (1, 2, 4, 8), case


def test_plan_follows_the_work(plan):
    one, long_one, piece, prompt = plan([(1, 8, 4, 64, 1024), (1, 8, 1, 64, 30000), (1, 8, 512, 64, 30512), (1, 8, 8192, 64, 8192)])
    assert one == (1, 2, 8)            # few rows, few keys: many small CTAs
    assert long_one == (1, 6, 8)       # few rows, many keys: a deep ring
    assert piece == (2, 5, 4)
    assert prompt == (2, 5, 1)         # enough tiles for every SM: keys are not shared out


def test_every_kind_is_taken_somewhere(plan):
    kinds = {(1, 2, n) for n in (1, 2, 4, 8)} | {(1, 6, n) for n in (1, 2, 4, 8)} | {(2, 5, n) for n in (1, 2, 4, 8)}
    cases = [(b, kv, b * t, tile, -(-(s + t) // 16) * 16 + 16) for b in (1, 3, 6, 16) for kv, tile in ((1, 64), (8, 64), (8, 128), (2, 42))
             for t in (1, 64, 130, 300) for s in (0, 500, 1500, 3000, 4500)]
    assert set(plan(cases)) == kinds
