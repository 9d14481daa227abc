"""Report words of contexts (csrc/reports.hpp), compiled for the host."""
from __future__ import annotations

import os
import subprocess

from conftest import PKG_DIR

PROGRAM = r"""
#include "reports.hpp"
#include <cassert>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <thread>
#include <vector>

int main() {
    // Many contexts, more than a block holds: words of their own, clear, in memory that was asked for.
    dgm::ReportWords pool;
    int blocks = 0;
    std::set<uintptr_t> seen;
    const auto alloc = [&](size_t bytes) -> void* {
        ++blocks;
        return calloc(1, bytes);
    };
    const int n = 5 * dgm::ReportWords::kContexts + 3;
    std::vector<std::vector<uint32_t*>> got(4);
    std::vector<std::thread> threads;
    for (auto& mine : got)
        threads.emplace_back([&] {
            for (int i = 0; i < n; ++i) {
                uint32_t* w = pool.take(alloc);
                assert(w && w[0] == 0 && w[1] == 0);
                w[0] = w[1] = 1;   // a report, which another context's creation must leave alone
                mine.push_back(w);
            }
        });
    for (auto& t : threads) t.join();
    for (auto& mine : got)
        for (uint32_t* w : mine) {
            assert(w[0] == 1 && w[1] == 1);
            for (int i = 0; i < 2; ++i) assert(seen.insert(reinterpret_cast<uintptr_t>(w + i)).second);
        }
    assert(blocks == (4 * n + dgm::ReportWords::kContexts - 1) / dgm::ReportWords::kContexts);
    // Without memory: none, and the next one asks again.
    dgm::ReportWords poor;
    assert(!poor.take([](size_t) -> void* { return nullptr; }));
    assert(poor.take(alloc));
    puts("ok");
}
"""


def test_every_context_has_words_of_its_own(tmp_path):
    src = tmp_path / "reports.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "reports")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-pthread", "-fsanitize=undefined,bounds",
                    "-fno-sanitize-recover=all", "-I", os.path.join(PKG_DIR, "csrc"), str(src), "-o", exe], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stderr
