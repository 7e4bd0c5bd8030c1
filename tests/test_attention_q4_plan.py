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
// shapes on stdin -> prompt, G, groups, tiles, n_split, chunk
int main() {
    long long nh, nkv, hd, q, kv;
    while (scanf("%lld %lld %lld %lld %lld", &nh, &nkv, &hd, &q, &kv) == 5) {
        const Q4Plan p = q4_plan(nh, nkv, hd, q, kv, 256);
        printf("%d %d %d %d %d %d\n", (int)p.prompt, p.G, p.groups, p.tiles, p.n_split, p.chunk);
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


def compiled(tmp, text):
    src, exe = tmp / "main.cpp", tmp / "main"
    src.write_text(text)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    return str(exe)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = compiled(tmp_path_factory.mktemp("plan"), MAIN)

    def run(shapes):
        text = "".join(" ".join(map(str, s)) + "\n" for s in shapes)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        return [dict(zip(("prompt", "G", "groups", "tiles", "n_split", "chunk"), map(int, o.split()))) for o in out]
    return run


def test_fetches_begin_within_the_range(tmp_path):
    subprocess.run([compiled(tmp_path, WALK)], check=True)


def test_calls_meant_for_the_prompt_kernel_take_it(plan):
    calls = sorted(PROMPT_CALLS)
    assert calls and all(p["prompt"] for p in plan(calls))
