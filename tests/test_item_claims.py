"""The rule by which workgroups take a launch's items (csrc/item_claims.hpp), compiled
for the host and run over simulated workgroups."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "item_claims.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace pcl;
typedef std::vector<uint32_t> Counts;

struct Group : ItemClaims {
    double free_at = 0;
    uint32_t part = 0; // whose items it takes
    uint32_t next = 0; // taken ahead
    int vain = 0, moves = 0, ran = 0;
};

// settle with the counters, which nobody else counts up meanwhile
static uint32_t settled(Group &g, Counts &taken, uint32_t n)
{
    const uint32_t before = g.part;
    auto add = [&](uint32_t part) {
        const uint32_t i = taken[part]++;
        g.vain += g.place(part, i) >= g.items;
        return i;
    };
    n = g.settle(n, g.part, [&](uint32_t part) { return taken[part]; }, add);
    g.moves += g.part != before;
    return n;
}

static uint32_t took(Group &g, Counts &taken)
{
    const uint32_t i = taken[g.part]++;
    g.vain += g.place(g.part, i) >= g.items;
    return settled(g, taken, g.place(g.part, i));
}

// `items` of random length over `grid` workgroups: "once" items, vain, moves, ended
static void run(uint32_t items, uint32_t grid, bool others, unsigned seed)
{
    const uint32_t parts = grid % kItemParts ? 1 : kItemParts;
    std::srand(seed);
    Counts taken(kItemParts, grid / parts), times(items, 0);
    std::vector<Group> groups(grid);
    for (uint32_t w = 0; w < grid; ++w) {
        groups[w].ItemClaims::operator=({items, grid, grid / parts, others && parts > 1});
        groups[w].part = w % parts;
        groups[w].next = groups[w].place(groups[w].part, w / parts);
    }
    bool wrong = false;
    uint32_t busy = grid;
    std::vector<bool> done(grid, false);
    while (busy) {
        uint32_t w = grid;
        for (uint32_t i = 0; i < grid; ++i)
            if (!done[i] && (w == grid || groups[i].free_at < groups[w].free_at))
                w = i;
        Group &g = groups[w];
        if (g.next >= items) {
            done[w] = true;
            --busy;
            // every count in vain has led to another part or to the end
            const bool taker = g.ran > 0;
            wrong |= g.vain != g.moves + (taker ? 1 : 0);
            continue;
        }
        const uint32_t now = g.next;
        ++times[now];
        ++g.ran;
        // lengths differ most between the parts
        g.free_at += 1 + std::rand() % (now % grid / g.each == 2 ? 400 : 20);
        g.next = took(g, taken);
    }
    int missed = 0, twice = 0, moves = 0;
    for (uint32_t t : times) {
        missed += t == 0;
        twice += t > 1;
    }
    for (const Group &g : groups)
        moves += g.moves;
    std::printf("%d %d %d %d\n", missed, twice, moves, (int)wrong);
}

int main(int argc, char **argv)
{
    if (argc > 1) {
        run(std::atoi(argv[1]), std::atoi(argv[2]), std::atoi(argv[3]) != 0, std::atoi(argv[4]));
        return 0;
    }
    // 8 parts of 4 items a round, 10 rounds; all parts but 1, 5 and 6 are used up
    for (uint32_t part = 0; part < kItemParts; ++part) {
        Group g;
        g.ItemClaims::operator=({320, 32, 4, true});
        g.part = part;
        Counts taken = {40, 38, 40, 40, 40, 12, 39, 44};
        std::printf("%u:", part);
        for (int i = 0; i < 4; ++i) {
            const uint32_t n = took(g, taken);
            std::printf(" %u/%u", n < 320 ? n / 4 % 8 : 99, g.part);
        }
        std::printf(" vain %d\n", g.vain);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("claims")
    source, binary = folder / "claims.cpp", folder / "claims"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas",
                    "-I" + os.path.join(ROOT, "power-cpu-llm_amd", "csrc"), str(source), "-o",
                    str(binary)], check=True)
    return str(binary)


def output(program, *args):
    return subprocess.run([program] + [str(a) for a in args], check=True, capture_output=True,
                          text=True).stdout.split("\n")[:-1]


def test_a_workgroup_goes_on_where_it_found_an_item(program):
    # "item's part/part that the workgroup takes from next", four items each
    want = {0: ("1/1 1/1 5/5 5/5", 2), 1: ("1/1 1/1 5/5 5/5", 1), 2: ("5/5 5/5 5/5 5/5", 1),
            3: ("5/5 5/5 5/5 5/5", 1), 4: ("5/5 5/5 5/5 5/5", 1), 5: ("5/5 5/5 5/5 5/5", 0),
            6: ("6/6 1/1 1/1 5/5", 2), 7: ("1/1 1/1 5/5 5/5", 2)}
    for line in output(program):
        part = int(line[0])
        items, vain = line[3:].split(" vain ")
        assert items == want[part][0], line
        assert int(vain) == want[part][1], line


@pytest.mark.parametrize("grid", [1, 7, 8, 64, 200, 256])
@pytest.mark.parametrize("others", [0, 1])
def test_every_item_is_taken_once(program, grid, others):
    for items in (0, 1, 3, grid - 1, grid, grid + 1, 5 * grid + 3, 40 * grid):
        for seed in (1, 2):
            missed, twice, moves, wrong = map(int, output(program, items, grid, others, seed)[0]
                                              .split())
            assert (missed, twice, wrong) == (0, 0, 0), (items, seed)
            assert moves == 0 or (others and grid % 8 == 0)
            # (where part 2's items are long the other parts' workgroups take some)
            if items == 40 * grid and others and grid % 8 == 0:
                assert moves > 0
