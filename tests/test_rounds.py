"""The producers' rounds of the paged prefill (tb_rounds.h) on the CPU: threads in the place of warps,
a meeting that notes who waits for one that no other comes to."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tabinfer_b200", "csrc")

PROGRAM = r"""
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <thread>
#include <vector>
#include "tb_rounds.h"

constexpr int P = 4;
struct Meeting {                     // all P, or a note after two seconds
    std::mutex m;
    std::condition_variable c;
    int here = 0, turn = 0;
    bool any = false, result = false, stuck = false;
    bool operator()(bool dead)
    {
        std::unique_lock<std::mutex> l(m);
        any = any || dead;
        const int t = turn;
        if (++here == P) {
            here = 0;
            turn++;
            result = any;
            any = false;
            c.notify_all();
            return result;
        }
        if (!c.wait_for(l, std::chrono::seconds(2), [&] { return turn != t || stuck; })) stuck = true;
        if (stuck) {
            c.notify_all();
            return true;
        }
        return result;
    }
};

// argv: tiles, then for each producer the tile at which its wait gives up (-1: none)
int main(int argc, char** argv)
{
    const int tiles = atoi(argv[1]);
    Meeting meet;
    std::vector<int> done(P, 0), told(P, 0);
    std::vector<std::thread> all;
    for (int p = 0; p < P; p++)
        all.emplace_back([&, p] {
            const int at = atoi(argv[2 + p]);
            int known = tiles < 3 ? tiles : 3;
            producer_rounds(
                tiles > 0, tiles > 1, tiles > 2, [&](int it) { told[p] = it; }, [&](bool dead) { return meet(dead); },
                [&] { return ++known <= tiles; },
                [&](int it, bool next) {
                    if (next != (it + 1 < tiles) || (next && told[p] != it + 1)) abort();
                    if (it == at) return false;
                    done[p]++;
                    return true;
                });
        });
    for (auto& t : all) t.join();
    printf("%d", (int)meet.stuck);
    for (int p = 0; p < P; p++) printf(" %d", done[p]);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("rounds")
    src, exe = d / "rounds.cpp", d / "rounds"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I" + CSRC, str(src), "-o", str(exe)], check=True)
    return str(exe)


def _run(program, tiles, at):
    out = subprocess.run([program, str(tiles)] + [str(a) for a in at], check=True, capture_output=True, text=True,
                         timeout=60).stdout.split()
    return out[0] == "1", [int(x) for x in out[1:]]


@pytest.mark.parametrize("tiles", [0, 1, 2, 3, 4, 9])
def test_every_tile_once(program, tiles):
    assert _run(program, tiles, [-1] * 4) == (False, [tiles] * 4)


@pytest.mark.parametrize("tiles", [1, 2, 3, 6])
@pytest.mark.parametrize("who", [[0], [3], [1, 2], [0, 1, 2, 3]])
def test_one_that_gives_up_holds_nobody(program, tiles, who):
    """at each tile, the last one too, where the others come to no further meeting"""
    for at in range(tiles):
        stuck, done = _run(program, tiles, [at if p in who else -1 for p in range(4)])
        assert not stuck, (tiles, who, at)
        for p in range(4):
            assert done[p] == (at if p in who else at + 1)


def test_two_that_give_up_at_other_tiles(program):
    stuck, done = _run(program, 5, [2, -1, 4, -1])
    assert not stuck and done == [2, 3, 3, 3]
