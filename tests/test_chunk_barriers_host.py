"""The named barriers between the warps of a tile of chunk attention (garnet_b200/csrc/chunk_barriers.h), played through on the host: no
schedule, and no wait in shared memory that gives up early or late, may mix two phases of a barrier or leave a warp waiting for ever."""
import subprocess
from pathlib import Path

import pytest

import garnet_b200

# Warps as lists of what they do, one of those that can go on chosen at random each time.  A named barrier counts arrivals (32 per
# warp) and is complete when its number is reached, as the hardware's are; `sync` goes on when the phase that it came to is complete.
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>
#include "chunk_barriers.h"
using namespace gb200;

enum Kind { Sync, Arrive, Wait, Signal };
struct Op { Kind kind; int id, threads, step; };        // barrier or event; arrivals that complete a phase; the step that it is about
struct Warp { std::vector<Op> ops; size_t at = 0; bool good = true, came = false; long long phase = 0; };
struct Barrier { int count = 0; long long phase = 0; std::set<int> steps; };

constexpr int kTurn = 1, kScores = 3, kP = 7;
constexpr int kFull = 0, kDone = 1000;                   // events: a unit is there; scores of a step are there

int play(int tiles, const int* steps, double gives_up, int lost, unsigned seed)
{
    std::mt19937 rng(seed);
    int most = 0;
    for (int q = 0; q < tiles; ++q) most = steps[q] > most ? steps[q] : most;
    const int turns = tiles == 2 ? (steps[0] < steps[1] ? steps[0] : steps[1]) : 0;
    std::vector<Warp> warps;
    Warp loader;                                         // the unit of step `lost` and those behind it never come
    for (int u = 0; u < most + 2 && u != lost; ++u) loader.ops.push_back({Signal, kFull + u, 0, u});
    warps.push_back(loader);
    for (int q = 0; q < tiles; ++q) {
        const int n = steps[q];
        Warp scout, issuer;
        chunk_scout(
            n, [&](int i) { scout.ops.push_back({Sync, kP + 2 * q + (i & 1), kWeightsThreads, i}); },
            [&](int i) { scout.ops.push_back({Wait, kDone + 1000 * q + i, 0, i}); },
            [&](int i) { scout.ops.push_back({Arrive, kScores + 2 * q + (i & 1), kScoresThreads, i}); });
        for (int u = 0; most && u < most + 2; ++u) {
            issuer.ops.push_back({Wait, kFull + u, 0, u});
            if (u >= 2 && u < n + 2) issuer.ops.push_back({Sync, kP + 2 * q + (u & 1), kWeightsThreads, u - 2});
            if (u < n + 2) issuer.ops.push_back({Signal, kDone + 1000 * q + u, 0, u});
        }
        warps.push_back(scout), warps.push_back(issuer);
        for (int w = 0; w < 4; ++w) {
            Warp softmax;
            for (int j = 0; j < n; ++j) {
                softmax.ops.push_back({Sync, kScores + 2 * q + (j & 1), kScoresThreads, j});
                if (j && rng() % 4 == 0) softmax.ops.push_back({Wait, kDone + 1000 * q + j + 1, 0, j});      // O is rescaled
                if (j < turns && (q == 1 || j > 0)) softmax.ops.push_back({Sync, kTurn + q, 256, q == 0 ? j - 1 : j});
                if (j < turns && !(q == 1 && j + 1 == turns)) softmax.ops.push_back({Arrive, kTurn + 1 - q, 256, j});
                softmax.ops.push_back({Arrive, kP + 2 * q + (j & 1), kWeightsThreads, j});
            }
            if (n) for (int i = n; i < n + 2; ++i) softmax.ops.push_back({Sync, kScores + 2 * q + (i & 1), kScoresThreads, i});
            warps.push_back(softmax);
        }
    }
    std::map<int, Barrier> barriers;
    std::set<int> events;
    std::uniform_real_distribution<double> unit(0, 1);
    const auto come = [&](const Op& o) {
        Barrier& b = barriers[o.id];
        b.steps.insert(o.step);
        if (b.steps.size() > 1) return false;            // arrivals of two steps in one phase
        b.count += 32;
        if (b.count == o.threads) b.count = 0, ++b.phase, b.steps.clear();
        return true;
    };
    for (;;) {
        std::vector<int> can;
        bool left = false, waits = false;
        for (size_t w = 0; w < warps.size(); ++w) {
            Warp& v = warps[w];
            if (v.at == v.ops.size()) continue;
            left = true;
            const Op& o = v.ops[v.at];
            if (o.kind == Sync && v.came && barriers[o.id].phase == v.phase) continue;
            if (o.kind == Wait && v.good && !events.count(o.id)) { waits = true; if (unit(rng) >= gives_up) continue; }
            can.push_back(int(w));
        }
        if (!left) return 0;
        if (can.empty()) {
            if (!waits) return 1;                        // every warp that is left waits at a named barrier
            if (gives_up == 0.0 && lost < 0) return 2;   // nothing was lost: no wait may run out
            for (Warp& v : warps)                        // time passes until a wait runs out
                if (v.at < v.ops.size() && v.ops[v.at].kind == Wait && v.good && !events.count(v.ops[v.at].id)) { v.good = false; break; }
            continue;
        }
        Warp& v = warps[can[rng() % can.size()]];
        const Op& o = v.ops[v.at];
        if (o.kind == Sync && !v.came) {
            v.came = true, v.phase = barriers[o.id].phase;
            if (!come(o)) return 3;
            continue;
        }
        if (o.kind == Sync) v.came = false;
        if (o.kind == Arrive && !come(o)) return 3;
        if (o.kind == Wait && v.good && !events.count(o.id)) v.good = false;
        if (o.kind == Signal && v.good) events.insert(o.id);
        ++v.at;
    }
}

int main(int argc, char** argv)
{
    const double gives_up = std::atof(argv[1]);
    const bool loses = std::atoi(argv[2]);
    long long bad[4] = {};
    unsigned seed = 0;
    for (int tiles = 1; tiles <= 2; ++tiles)
        for (int a = 0; a <= 9; ++a)
            for (int b = 0; b <= (tiles == 2 ? 9 : 0); ++b)
                for (int k = 0; k < 12; ++k) {
                    const int steps[2] = {a, b}, most = a > b ? a : b;
                    ++bad[play(tiles, steps, gives_up, loses && most ? int(++seed % (most + 2)) : -1, ++seed)];
                }
    std::printf("%lld %lld %lld %lld\n", bad[0], bad[1], bad[2], bad[3]);
    return 0;
}
"""


@pytest.fixture(scope="module")
def played(tmp_path_factory):
    folder = tmp_path_factory.mktemp("barriers")
    (folder / "play.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(Path(garnet_b200.__file__).parent / "csrc"), str(folder / "play.cpp"), "-o", str(folder / "play")], check=True)
    return lambda *args: [int(n) for n in subprocess.run([str(folder / "play"), *map(str, args)], capture_output=True, text=True, check=True).stdout.split()]


@pytest.mark.parametrize("gives_up,loses", [(0.0, 0), (0.0, 1), (0.002, 0), (0.05, 1), (0.5, 0)])
def test_every_warp_comes_through(played, gives_up, loses):
    """Nothing lost; copies that stop; waits that give up now and then, whether what they wait for would have come or not."""
    through, stuck, ran_out, mixed = played(gives_up, loses)
    assert (stuck, ran_out, mixed) == (0, 0, 0) and through == 12 * (10 + 100)
