"""The host side of attention over a 4-bit KV cache (csrc/attention_q4_plan.hpp),
compiled on its own."""
import os
import random
import subprocess

import pytest

from test_gpu_kv_edges import PROMPT_CALLS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "barq-inference_amd", "csrc")

MAIN = r"""
#include "attention_q4_plan.hpp"
#include <cstdio>
using namespace barq;
// shapes on stdin -> prompt, G, groups, tiles, n_split, chunk, fits
int main() {
    long long nh, nkv, hd, q, kv;
    while (scanf("%lld %lld %lld %lld %lld", &nh, &nkv, &hd, &q, &kv) == 5) {
        const Q4Plan p = q4_plan(nh, nkv, hd, q, kv, 256);
        printf("%d %d %d %d %d %d %d\n", (int)p.prompt, p.G, p.groups, p.tiles, p.n_split, p.chunk, (int)q4_fits(p, nh, hd, q));
    }
}
"""

WALK = r"""
#include "attention_q4_plan.hpp"
#include <cstdio>
using namespace barq;
// Of four waves' walks over n positions: each step is the one fetched before it, and no fetch begins behind the
// range's whole tiles, where the descriptors end.
int main() {
    for (int n = 1; n < 2000; n++)
        for (int first = 0; first < 128 && first < n; first += 32) {
            int held = first;
            for (int at = first; at < n; at += 128) {
                if (held != at) return printf("%d %d: %d\n", n, at, held), 1;
                held = q4_ahead(at, 128, n);
                if (held < 0 || held > (n + 7) / 8 * 8) return printf("%d %d: %d\n", n, at, held), 1;
            }
        }
}
"""


ENDS = r"""
#include "attention_q4_plan.hpp"
#include <cstdio>
using namespace barq;
// kv_len, splits, chunk on stdin: the splits of rows that see v positions cover 0 .. v - 1 once, whatever v (-ftrapv:
// an int that overflows ends the program)
int main() {
    long long kv, ns, chunk;
    while (scanf("%lld %lld %lld", &kv, &ns, &chunk) == 3) {
        const long long seen[] = {kv, kv - 1, kv / 2, kv / 3 + 1, chunk, chunk + 1, 1};
        for (long long v : seen) {
            if (v < 1 || v > kv) continue;
            long long at = 0;
            for (int s = 0; s < ns; s++) {
                const int start = s * (int)chunk, end = q4_range_end(start, (int)chunk, (int)v);
                if (start < v ? start != at || end <= start || end - start > chunk : end > start) return printf("%lld %lld: %d %d\n", kv, v, start, end), 1;
                if (start < v) at = end;
            }
            if (at != v) return printf("%lld %lld: ends at %lld\n", kv, v, at), 1;
        }
    }
}
"""


def compiled(tmp, text):
    src, exe = tmp / "main.cpp", tmp / "main"
    src.write_text(text)
    subprocess.run(["g++", "-O2", "-ftrapv", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    return str(exe)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = compiled(tmp_path_factory.mktemp("plan"), MAIN)

    def run(shapes):
        text = "".join(" ".join(map(str, s)) + "\n" for s in shapes)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        return [dict(zip(("prompt", "G", "groups", "tiles", "n_split", "chunk", "fits"), map(int, o.split()))) for o in out]
    return run


def test_fetches_begin_within_the_range(tmp_path):
    subprocess.run([compiled(tmp_path, WALK)], check=True)


def test_calls_meant_for_the_prompt_kernel_take_it(plan):
    calls = sorted(PROMPT_CALLS)
    assert calls and all(p["prompt"] for p in plan(calls))


LONGEST = 2 ** 31 - 4096   # the entry points take no more


def test_splits_of_every_length(plan, tmp_path):
    """No more splits than the merge takes, none longer than 32-bit offsets allow, all positions in one of them."""
    r = random.Random(5)
    lengths = [1, 31, 128, 129, 4096, 2 ** 20, 2 ** 20 + 1, 2 ** 21, 2 ** 21 + 1, 2 ** 30, 2 ** 30 + 1, 2 ** 30 + 5,
               1_600_000_000, LONGEST - 1, LONGEST] + [int(2 ** r.uniform(0, 31)) for _ in range(200)]
    shapes = [(*r.choice([(1, 1, 64), (32, 8, 128), (16, 16, 256), (14, 2, 64), (5, 2, 128)]), r.choice([1, 1, 5, 200, 2048]),
               min(n, LONGEST)) for n in lengths] + [(1, 1, 64, 1, n) for n in lengths if n <= LONGEST]
    plans = plan(shapes)
    for s, p in zip(shapes, plans):
        assert 1 <= p["n_split"] <= 1024, s
        assert 0 < p["chunk"] <= 2 ** 21 and p["chunk"] % 128 == 0, s
        assert (p["n_split"] - 1) * p["chunk"] < s[4] <= p["n_split"] * p["chunk"], s
    text = "".join(f"{s[4]} {p['n_split']} {p['chunk']}\n" for s, p in zip(shapes, plans))
    subprocess.run([compiled(tmp_path, ENDS)], input=text, text=True, check=True)


def test_a_piece_may_be_longer_than_a_million(plan):
    """(the call of test_gpu_kv_edges.py's test of it)"""
    assert [(p["n_split"], p["chunk"] > 2 ** 20) for p in plan([(4, 1, 64, 6150, 2 ** 20 + 5000)])] == [(1, True)]


def test_calls_whose_launches_fit(plan):
    """Fewer than 2^32 threads each: the kernel's workgroups have 256, the merge's four waves of 256 values."""
    shapes = [(32, 8, 128, 2048, 2048), (2 ** 24 - 1, 2 ** 24 + 16, 64, 1, 1), (2 ** 24, 2 ** 24 + 16, 64, 1, 1),
              (16, 1, 64, 65535, LONGEST), (16, 1, 64, 60000, LONGEST), (65535, 1, 64, 1, LONGEST), (32, 8, 128, 65535, 100000)]
    plans = plan(shapes)
    for (heads, _, hd, rows, _), p in zip(shapes, plans):
        grids = [p["n_split"] * p["tiles"] * p["groups"]] + [((heads * hd + 255) // 256 * rows + 3) // 4] * (p["n_split"] > 1)
        assert p["fits"] == (max(grids) * 256 < 2 ** 32)
    assert [p["fits"] for p in plans] == [1, 1, 0, 0, 1, 1, 1]
