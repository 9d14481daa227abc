"""The attention kernels' index arithmetic (csrc/attn_index.hpp), compiled for the
host: rows of packed sequences, pages of a cache, bad ones among them."""
from __future__ import annotations

import os
import subprocess

import pytest

from conftest import PKG_DIR

PROGRAM = r"""
#include "attn_index.hpp"
#include <cassert>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
using namespace dgm_attn;

static uint64_t state = 12345;
static uint32_t next() { state = state * 6364136223846793005ull + 1442695040888963407ull; return uint32_t(state >> 33); }

int main() {
    // Quotients: every divisor's neighbours of multiples up to 2^31 - 1.
    for (uint32_t d : {1u, 2u, 3u, 7u, 8u, 16u, 24u, 100u, 127u, 128u, 1000u, 65535u, 65536u, 1000003u, 0x7fffffffu}) {
        const Div div(d);
        for (int i = 0; i < 200000; ++i) {
            const uint32_t n = next() & 0x7fffffff, q = n / d;
            for (uint64_t m : {uint64_t(n), uint64_t(q) * d, uint64_t(q) * d + d - 1, uint64_t(0x7fffffff)})
                if (m < (1ull << 31)) assert(div(uint32_t(m)) == m / d);
        }
    }
    // Tile slots: every row of every sequence in exactly one, all within the count.
    for (int trial = 0; trial < 2000; ++trial) {
        const int nseq = 1 + next() % 40, per = 32 << (next() % 4);
        std::vector<int32_t> starts{int32_t(next() % 50)};
        for (int s = 0; s < nseq; ++s) starts.push_back(starts.back() + (next() % 3 ? next() % 300 : 0));
        const int64_t rows = starts.back() + next() % 40;
        std::vector<int> seen(rows, 0);
        for (int64_t slot = 0; slot < slot_count(rows, nseq, per); ++slot) {
            int64_t s = -1;
            for (int64_t i = 0; i < nseq; ++i)
                if (slot_base(clamped(starts.data(), i, rows), i, per) <= slot) s = i;
            if (s < 0) continue;
            const int first = clamped(starts.data(), s, rows), len = clamped(starts.data(), s + 1, rows) - first;
            const int64_t tile = slot - slot_base(first, s, per);
            for (int64_t r = tile * per; r < (tile + 1) * per && r < len; ++r) ++seen[first + r];
        }
        for (int64_t r = 0; r < rows; ++r) assert(seen[r] == (r >= starts[0] && r < starts.back()));
    }
    // Starts that are wrong stay within the rows.
    const int32_t wild[] = {-1, INT_MIN, INT_MAX, 101, 100, 0};
    for (int i = 0; i < 6; ++i) assert(clamped(wild, i, 100) >= 0 && clamped(wild, i, 100) <= 100);
    // Pages: each (position, head) of a permuted table has a row of its own; bad ids have none.
    for (int page : {1, 7, 16, 100}) {
        const int KVH = 3, numPages = 40, maxPages = 10;
        const Div div(page);
        std::vector<int32_t> table(4 * maxPages);
        for (int i = 0; i < 40; ++i) table[i] = (i * 7 + 3) % 40;
        std::set<int> rows;
        for (int s = 0; s < 4; ++s)
            for (int pos = 0; pos < maxPages * page; ++pos)
                for (int h = 0; h < KVH; ++h) {
                    const int r = cache_row(table.data(), div, numPages, maxPages, KVH, s, pos, h);
                    assert(r >= 0 && r < numPages * KVH * page && rows.insert(r).second);
                    assert(r == (table[s * maxPages + pos / page] * KVH + h) * page + pos % page);
                }
        for (int32_t id : {-1, INT_MIN, 40, 41, INT_MAX}) {
            table[5] = id;
            assert(cache_row(table.data(), div, numPages, maxPages, KVH, 0, 5 * page, 0) == -1);
        }
    }
    // The largest cache: rows just below 2^31.
    const int32_t last = (1 << 24) - 1;
    assert(cache_row(&last, Div(16), 1 << 24, 1, 8, 0, 15, 7) == INT_MAX);
    puts("ok");
}
"""


@pytest.mark.parametrize("compiler", ["g++"])
def test_index_arithmetic(tmp_path, compiler):
    src = tmp_path / "index.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "index")
    subprocess.run([compiler, "-std=c++17", "-O1", "-g", "-fsanitize=undefined,bounds", "-fno-sanitize-recover=all",
                    "-I", os.path.join(PKG_DIR, "csrc"), str(src), "-o", exe], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stderr


def test_workspace_sizes_are_host_arithmetic(dgm):
    """-1 for sizes that are refused; one float a (row, head) for the backward; partial rows of every worker and sequence for decoding."""
    import ctypes
    lib = dgm.load_library()
    a = dgm.AttnCfg(type=0, H=12, KVH=4, D=64, causal=1, scale=0.125, rows=1000, nseq=3)
    assert lib.dgm_attnPackedBwd_ws_bytes(ctypes.byref(a)) >= 1000 * 12 * 4
    a.rows = -1
    assert lib.dgm_attnPackedBwd_ws_bytes(ctypes.byref(a)) == -1 == lib.dgm_attnPackedBwd_ws_bytes(None)
    c = dgm.CacheCfg(type=1, KVH=8, D=128, pageSize=16, numPages=100, maxPages=10)
    size = lib.dgm_attnPagedDecode_ws_bytes
    assert size(ctypes.byref(c), 4, 32) > size(ctypes.byref(c), 1, 32) > 0
    assert size(ctypes.byref(c), -1, 32) == size(ctypes.byref(c), 1, 9) == size(None, 1, 8) == -1
    assert size(ctypes.byref(c), 65537, 32) == size(ctypes.byref(c), 65536, 128) == -1
    for name, value in (("D", 100), ("D", 264), ("type", 7), ("pageSize", 0), ("numPages", 1 << 30)):
        broken = dgm.CacheCfg.from_buffer_copy(c)
        setattr(broken, name, value)
        assert size(ctypes.byref(broken), 4, 32) == -1
