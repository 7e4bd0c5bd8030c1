"""How an eviction's rows are shared out over launches (csrc/kv_evict_plan.hpp),
compiled on its own."""
import os
import random
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "barq-inference_amd", "csrc")

MAIN = r"""
#include "kv_evict_plan.hpp"
#include <cstdio>
int main() {
    unsigned long long q4, heads, m, hd;
    while (scanf("%llu %llu %llu %llu", &q4, &heads, &m, &hd) == 4) printf("%zu\n", barq::evict_heads(q4 != 0, heads, m, hd));
}
"""


def threads(q4, heads, m, hd):
    """What the launches of kv_evict.hip ask for, whole workgroups of 256."""
    def up(n):
        return (n + 255) // 256 * 256
    if not q4:
        return up(2 * heads * m * (hd // 4 if hd % 4 == 0 else hd))
    tiles, nb = (m + 7) // 8, hd // 32
    return up(heads * tiles * 16) + up(heads * m * nb) + up(heads * tiles * 2 * nb)


def test_launches_have_fewer_than_2_to_32_threads(tmp_path):
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text(MAIN)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = random.Random(1)
    shapes = [(0, 8, 2048, 128), (1, 8, 4096, 128), (0, 32768, 65535, 1), (0, 32768, 65537, 1), (0, 1, 2 ** 31 - 4096, 1),
              (0, 1, 2 ** 31 - 4096, 2), (0, 3, 2 ** 26, 127), (1, 1, 2 ** 31 - 4096, 64), (1, 2, 2 ** 29, 256)]
    shapes += [(r.randint(0, 1), int(2 ** r.uniform(0, 16)), int(2 ** r.uniform(0, 31)), r.choice([64, 128, 256])) for _ in range(500)]
    text = "".join(" ".join(map(str, s)) + "\n" for s in shapes)
    per = [int(x) for x in subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split()]
    for s, p in zip(shapes, per):
        q4, heads, m, hd = s
        assert 0 <= p <= heads, s
        if p:
            assert threads(q4, p, m, hd) < 2 ** 32, s
        if p < heads:   # one more would be too many, or as good as
            assert threads(q4, p + 1, m, hd) > 2 ** 32 - 2048, s
    assert per[0] == 8 and per[1] == 8 and per[2] == 32768 and 0 < per[3] < 32768 and per[5] == 0
