"""Places in a table of the keys of a tile and of those behind it, up to the longest tables: the kernels' own arithmetic, on the host.  No GPU."""
from pathlib import Path

from test_cache_index import build_and_run

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <random>
#include "cache_index.hpp"
using namespace gatgpu;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    std::mt19937_64 g(11);
    const auto below = [&](uint64_t n) { return uint32_t(g() % n); };
    for (int i = 0; i < 200000; ++i) {
        CacheSizes c;
        c.page_log = 4 + below(5);
        const uint32_t most = uint32_t((uint64_t(1) << 32 >> c.page_log) - 1);  // blocks * page < 2^32
        c.blocks = i % 3 ? most - below(3) : below(40);
        const uint64_t tokens = uint64_t(c.blocks) << c.page_log;
        const uint32_t keys = uint32_t(i % 2 ? tokens - below(tokens < 200 ? tokens + 1 : 200) : tokens ? g() % (tokens + 1) : 0);
        const uint32_t tiles = uint32_t((uint64_t(keys) + 63) / 64);
        // Tiles up to three behind the last one are asked for, and up to 128 keys of each: sums that pass 32 bits stay within the table.
        const uint32_t tile = i % 5 ? (tiles > 3 ? tiles - 3 : 0) + below(7) : below(uint64_t(tiles) + 4);
        for (uint32_t at = 0; at < 128; at += 1 + below(16)) {
            const uint64_t key = uint64_t(tile) * 64 + at;
            const uint32_t block = block_of(c, keys, uint32_t(key));
            CHECK(block == kNoPage || block < c.blocks);
            if (key >> 32 == 0) CHECK(block == (key < keys ? uint32_t(key >> c.page_log) : kNoPage));
        }
    }
    std::puts("fine");
}
"""


def test_tiles_at_the_end_of_long_tables(tmp_path):
    r = build_and_run(tmp_path, PROGRAM, ROOT / "gat-tfs_amd" / "csrc")
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stdout + r.stderr
