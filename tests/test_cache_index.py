"""Where a request's rows and a page's bytes lie, whatever the device arrays hold: the kernels' own arithmetic, on the
host.  And the layout of the call descriptions in Python, against the header's.  No GPU."""
import ctypes
import subprocess
from pathlib import Path

import gatgpu
import pytest

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "cache_index.hpp"
using namespace gatgpu;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    std::mt19937_64 g(7);
    const auto below = [&](uint64_t n) { return uint32_t(g() % n); };
    const auto any = [&]() -> uint32_t {
        switch (below(5)) {
            case 0: return 0xffffffffu - below(3);
            case 1: return below(4);
            case 2: return 0x80000000u + below(3);
            default: return below(70000);
        }
    };
    for (int i = 0; i < 400000; ++i) {
        CacheSizes c;
        c.kv_heads = 1 + below(8);
        c.group = 1 + below(8);
        c.heads = c.kv_heads * c.group;
        c.dim = 16 * (1 + below(8));
        c.page_log = 4 + below(5);
        c.pages = 1 + below(i % 2 ? 20 : (uint64_t(1) << 32 >> c.page_log) - 1);
        c.blocks = below(i % 3 ? 40 : (uint64_t(1) << 32 >> c.page_log));
        c.rows = below(i % 5 ? 300 : (uint64_t(1) << 31) / c.heads);
        c.most = any();
        c.requests = 1;
        const CacheRequest q = cache_request(c, any(), any(), any());
        CHECK(uint64_t(q.begin) + q.rows <= c.rows);
        CHECK(q.rows <= c.most);
        CHECK(q.keys <= uint64_t(c.blocks) << c.page_log);
        CHECK(uint64_t(row_tiles(c, q)) * kCacheRows >= uint64_t(q.rows) * c.group);
        CHECK(key_tiles(q) >= 1 && uint64_t(key_tiles(q)) * kCacheTile >= q.keys);
        if (q.rows) CHECK(cache_seen(q, q.rows - 1) <= q.keys);
        for (int j = 0; j < 4; ++j) {
            const uint32_t key = j ? below(uint64_t(q.keys) + 200) : any(), block = block_of(c, q.keys, key);
            CHECK(block == kNoPage ? key >= q.keys : block < c.blocks);
            const uint32_t page = some_page(c, any()), head = below(c.kv_heads), col = 16 * below(c.dim / 16);
            CHECK(page < c.pages);
            const uint64_t size = (uint64_t(c.pages) * c.kv_heads * c.dim) << c.page_log;
            // 16 keys of a page from a multiple of 16 on, 16 columns each; 16 columns of a key, each of 16 keys
            const uint32_t at = key & ~15u;
            CHECK(key_byte(c, page, head, at + 15) + col + 16 <= size);
            CHECK(key_byte(c, page, head, at + 15) == key_byte(c, page, head, at) + 15 * c.dim);
            CHECK(value_byte(c, page, head, at, col + 15) + 16 <= size);
            CHECK(value_byte(c, page, head, at, col + 15) == value_byte(c, page, head, at, col) + (uint64_t(15) << c.page_log));
            CHECK(value_byte(c, page, head, at, col) % 16 == 0 && key_byte(c, page, head, at) % 16 == 0);
        }
    }
    std::puts("fine");
}
"""


def build_and_run(tmp_path, source, *include):
    (tmp_path / "t.cpp").write_text(source)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", *(f"-I{i}" for i in include),
                    "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True)
    return subprocess.run([str(tmp_path / "t")], check=False, capture_output=True, text=True, timeout=100)


def test_nothing_outside_the_arrays(tmp_path):
    r = build_and_run(tmp_path, PROGRAM, ROOT / "gat-tfs_amd" / "csrc")
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stdout + r.stderr


@pytest.mark.parametrize("python,name", [(gatgpu.RotateIO, "gatgpu_rotate_io"), (gatgpu.BlocksIO, "gatgpu_blocks_io"), (gatgpu.Cache, "gatgpu_cache"),
                                         (gatgpu.AppendIO, "gatgpu_append_io"), (gatgpu.CacheAttentionIO, "gatgpu_cache_attention_io")])
def test_structures_lie_as_in_the_header(tmp_path, python, name):
    lines = [f'std::printf("%zu %zu\\n", offsetof({name}, {f}), sizeof(((({name}*)0)->{f})));' for f, _ in python._fields_]
    source = f'#include <cstddef>\n#include <cstdio>\n#include "gatgpu.h"\nint main() {{ {" ".join(lines)} std::printf("%zu\\n", sizeof({name})); }}\n'
    r = build_and_run(tmp_path, source, ROOT / "include")
    want = [f"{getattr(python, f).offset} {getattr(python, f).size}" for f, _ in python._fields_] + [str(ctypes.sizeof(python))]
    assert r.stdout.split("\n")[:-1] == want


@pytest.mark.parametrize("entry,args", [
    ("gatgpu_rotate_forward", (None, None)), ("gatgpu_rotate_backward", (None, None, None, 0)), ("gatgpu_rotate_workspace", (None, None, None)),
    ("gatgpu_blocks_assign", (None, None, None, 0)), ("gatgpu_blocks_release", (None, None, None, 0)), ("gatgpu_blocks_workspace", (None, None, None)),
    ("gatgpu_cache_append", (None, None, None)), ("gatgpu_cache_attention", (None, None, None, None, 0)),
    ("gatgpu_cache_attention_workspace", (None, None, None, None))])
def test_null_handles(entry, args):
    lib = gatgpu.load_library()
    assert getattr(lib, entry)(*args) == gatgpu.EINVAL
    assert b"null" in lib.gatgpu_last_error(None)


def test_plain_e4m3_is_the_format():
    """The oracle's own rounding: every byte is its own nearest value, and so is torch's rounding of values between them."""
    import torch

    from cache_cases import bytes_of, values
    every = torch.arange(256, dtype=torch.uint8)
    v = values(every)
    assert torch.equal(bytes_of(v[~torch.isnan(v)]), every[~torch.isnan(v)])
    assert torch.equal(torch.nan_to_num(v.float(), nan=999.0), torch.nan_to_num(every.view(torch.float8_e4m3fn).float(), nan=999.0))
    g = torch.Generator().manual_seed(1)
    x = torch.cat((torch.randn(20000, generator=g) * 100, torch.randn(20000, generator=g) * 0.01, (v[:126] + v[1:127]).float() / 2)).clamp(-448, 448)
    assert torch.equal(values(bytes_of(x.double())).float(), x.to(torch.float8_e4m3fn).float())
