"""How attention over a paged cache divides its work, without a GPU: paged_runs.hpp through a small library of its own. Every
unit of every item is some block's and no other's, parts of an item lie side by side in runs that follow one another, and no
two parts have one slot or counter."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]

SOURCE = r"""
#include <algorithm>
#include <vector>

#include "paged_runs.hpp"
using namespace vvli;

struct Call {
    PageDiv group;
    uint32_t room, window, kv_heads;
};
struct Item {
    uint64_t start;
    Units un;
};
struct Had {
    uint32_t run;
    Part p;
};

// 0, or the number of what does not hold; out: runs, units a run, cut items, most parts of one, items.
template <class S>
int look(const int32_t* counts, const int32_t* starts, uint32_t n, const Call& a, uint32_t blocks, uint64_t* out) {
    std::vector<Item> items;
    uint64_t total = 0;
    for (uint32_t r = 0; r < n; ++r)
        for (uint32_t h = 0; h < a.kv_heads; ++h) {
            const Request q{0, counts[r] * a.group.d, starts[r]};
            for (uint32_t m0 = 0; m0 < q.vecs; m0 += S::M) {
                items.push_back(Item{total, units_of<S>(a, q, m0)});
                total += items.back().un.count;
            }
        }
    const Borders b = borders_of<S>(total, blocks);
    if (b.runs > blocks || b.near_lo + b.near_hi >= b.per || b.per < S::kFewest) return 1;
    std::vector<std::vector<Had>> had(items.size());
    std::vector<char> seen(blocks, 0);
    uint32_t there = 0;
    for (uint32_t block = 0; block < blocks; ++block) {
        const uint32_t run = run_of_block(block, blocks, b.runs);
        if (run >= b.runs) continue;
        if (seen[run]) return 2;
        seen[run] = 1, ++there;
        const uint64_t from = b.per * run, to = std::min(from + b.per, total);
        size_t i = std::upper_bound(items.begin(), items.end(), from, [](uint64_t u, const Item& x) { return u < x.start; }) - items.begin() - 1;
        const uint32_t unit = static_cast<uint32_t>(from - items[i].start);
        bool begun = true;
        for (; i < items.size() && items[i].start < to; ++i, begun = false) {
            Part p;
            const Share s = part_of<S>(b, items[i].un, items[i].start, to, unit, begun, p);
            if (s == Share::kEnd) break;
            if (s == Share::kNone) continue;
            had[i].push_back(Had{run, p});
            if (p.cut) break;
        }
    }
    if (there != b.runs) return 3;
    std::vector<char> slots(2 * blocks, 0), counters(blocks, 0);
    uint64_t cut = 0, most = 0;
    for (size_t i = 0; i < items.size(); ++i) {
        auto& h = had[i];
        const uint32_t count = items[i].un.count;
        std::sort(h.begin(), h.end(), [](const Had& x, const Had& y) { return x.run < y.run; });
        if (h.empty() || h.front().p.t0 != 0 || h.back().p.t1 != count) return 4;
        for (size_t k = 0; k < h.size(); ++k) {
            if (h[k].p.t0 >= h[k].p.t1 || (k && h[k].p.t0 != h[k - 1].p.t1)) return 5;   // every unit once
            if (h[k].p.cut != (k + 1 < h.size())) return 6;
            if (k && h[k].p.t0 <= S::kItem) return 7;                                     // no cut in front of the keys
        }
        if (h.size() == 1) continue;
        if (count <= S::kWhole) return 8;
        const uint64_t border = first_border(b, items[i].start);
        if (h.size() != parts_of(b, items[i].start, count)) return 9;
        if (border == 0 || border - 1 >= blocks || counters[border - 1]) return 10;
        counters[border - 1] = 1;
        for (size_t k = 0; k < h.size(); ++k) {
            if (h[k].run != border - 1 + k) return 11;                                    // where the join looks for it
            char& slot = slots[2 * h[k].run + (h[k].p.t0 == 0)];
            if (slot) return 12;
            slot = 1;
        }
        ++cut, most = std::max<uint64_t>(most, h.size());
    }
    out[0] = b.runs, out[1] = b.per, out[2] = cut, out[3] = most, out[4] = items.size();
    return 0;
}

extern "C" int t_look(const int32_t* counts, const int32_t* starts, uint32_t n, uint32_t group, uint32_t room, uint32_t window,
                      uint32_t kv_heads, uint32_t blocks, uint32_t kernel, uint64_t* out) {
    const Call a{page_div(group), room, window, kv_heads};
    switch (kernel) {
    case 0: return look<FewCuts<1>>(counts, starts, n, a, blocks, out);
    case 1: return look<FewCuts<2>>(counts, starts, n, a, blocks, out);
    case 2: return look<ChunkCuts<true>>(counts, starts, n, a, blocks, out);
    default: return look<ChunkCuts<false>>(counts, starts, n, a, blocks, out);
    }
}
"""
KERNELS = ["few rows, f32", "few rows, 16 bits", "chunks, f32", "chunks, 16 bits"]


@pytest.fixture(scope="module")
def look(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("paged_runs")
    (d / "t.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-I", str(ROOT / "vvli_amd" / "csrc"), "-o", str(d / "t.so"),
                    str(d / "t.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "t.so"))

    def run(spec, group, kv_heads, kernel, blocks, window=0, room=1 << 20):
        starts, counts = (np.ascontiguousarray(x, np.int32) for x in zip(*spec))
        out = (ctypes.c_uint64 * 5)()
        wrong = lib.t_look(ctypes.c_void_p(counts.ctypes.data), ctypes.c_void_p(starts.ctypes.data), len(spec), group, room, window,
                           kv_heads, blocks, kernel, out)
        assert wrong == 0, (wrong, KERNELS[kernel], group, kv_heads, blocks, window, room, spec[:20])
        return dict(zip(("runs", "per", "cut", "most", "items"), out))

    return run


def layout(rng):
    """Requests of one of several makes: single tokens, drafts, prompts, a mixture, many idle ones; some at negative positions."""
    n = int(np.exp(rng.uniform(0, np.log(400))))
    past = int(np.exp(rng.uniform(0, np.log(40000))))
    make = rng.randint(5)
    if make == 2:
        n = min(n, 12)
    new = {0: lambda: 1, 1: lambda: rng.randint(0, 13), 2: lambda: rng.randint(1, 3000), 3: lambda: 1 if rng.rand() < 0.9 else rng.randint(0, 900),
           4: lambda: rng.randint(1, 40) if rng.rand() < 0.1 else 0}[make]
    spec = [(int(rng.randint(0, past + 1)), int(new())) for _ in range(n)]
    return [(-c if rng.rand() < 0.05 else -3 if rng.rand() < 0.02 else p, c) for p, c in spec]


@pytest.mark.parametrize("kernel", range(4), ids=KERNELS)
def test_every_unit_is_one_blocks(look, kernel):
    rng = np.random.RandomState(kernel)
    seen = dict(long=0, cut=0, many=0, idle=0)
    for _ in range(2500):
        spec = layout(rng)
        blocks = int(rng.choice([512, 512, 768, 768, 16, 8, 1, 3, 608, 304, 100]))
        got = look(spec, int(rng.choice([1, 2, 3, 4, 7, 8, 40])), int(rng.choice([1, 2, 4, 8, 16])), kernel, blocks,
                   int(rng.choice([0, 0, 0, 1, 33, 1000, 5000])), int(rng.choice([1 << 20, 1 << 20, 5000, 64])))
        seen["long"] += got["per"] >= 16
        seen["cut"] += got["cut"] > 0
        seen["many"] += got["most"] >= 8
        seen["idle"] += got["runs"] < blocks
    assert min(seen.values()) >= 40, seen


@pytest.mark.parametrize("kernel", range(4), ids=KERNELS)
def test_batches_about_as_large_as_the_runs_borders(look, kernel):
    """Items of every length about a run's, and runs of every length from the least: where borders fall on an item's ends."""
    for per in (1, 2, 3, 5, 8, 17, 40):
        for length in range(1, 60):
            look([(length * 16, 1)] * 40, 1, 1, kernel, max(1, 40 * length // (4 * per)))
            look([(length * 32 + i, 1 + i % 3) for i in range(20)], 4, 2, kernel, 8 * per)


def test_no_rows_are_no_runs(look):
    for kernel in range(4):
        assert look([(5, 0), (0, 0)], 4, 2, kernel, 512)["runs"] == 0


def test_batches_of_the_gpu_tests_have_long_runs(look):
    """What test_attention_runs_of_many_units counts on (heads, kv heads, blocks of 256 compute units)."""
    import test_gpu_paged_ops as G

    for what, heads, kv, blocks, kernels in (("tokens", 28, 4, 512, (0, 1)), ("drafts", 32, 8, 768, (0, 1)), ("prompts", 28, 4, 512, (2, 3)),
                                             ("prompts", 32, 8, 512, (2, 3)), ("mixed", 28, 4, 512, (0, 1)), ("prompts", 16, 4, 512, (2, 3))):
        for kernel in kernels:
            got = look(G.RUNS[what], heads // kv, kv, kernel, blocks)
            assert got["per"] >= 16 and got["cut"] >= 100, (what, heads, KERNELS[kernel], got)
