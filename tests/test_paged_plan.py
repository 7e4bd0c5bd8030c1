"""The host side of the paged cache (csrc/paged_plan.hpp), compiled on its own:
what a step's arrays are refused for, and that its plan covers every row and
every position that the row sees once."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "barq-inference_amd", "csrc")

MAIN = r"""
#include "paged_plan.hpp"
#include <cinttypes>
#include <cstring>
using namespace barq;
static int check() {
    PagedLimits lim;
    size_t n, stride;
    if (scanf("%zu %zu %zu %zu %zu %zu %zu", &lim.max_seqs, &lim.max_tokens, &lim.max_pages, &lim.n_pages, &lim.page_size, &n, &stride) != 7) return 1;
    std::vector<int32_t> q(n), kv(n), pages(n * stride);
    for (auto* v : {&q, &kv, &pages}) for (auto& x : *v) if (scanf("%d", &x) != 1) return 1;
    std::vector<uint32_t> stamp(lim.n_pages, 0);
    size_t tokens, entries;
    char msg[160] = "";
    const PagedFault f = paged_check(lim, n, q.data(), kv.data(), pages.data(), stride, stamp.data(), 1, tokens, entries, msg, sizeof msg);
    printf("%d %s\n", (int)f, msg);
    return 0;
}
static int plan() {
    PagedShape sh;
    int f16, hd;
    size_t n, max_tokens;
    if (scanf("%d %d %" SCNd64 " %" SCNd64 " %d %d %zu %zu", &sh.G, &sh.n_kv, &sh.window, &sh.n_sink, &f16, &hd, &max_tokens, &n) != 8) return 1;
    paged_shape_for(sh, f16, hd);
    sh.part_rows = paged_part_rows(sh, max_tokens);
    std::vector<PagedSeq> seqs(n);
    for (auto& s : seqs) if (scanf("%" SCNd64 " %" SCNd64, &s.q_len, &s.kv_len) != 2) return 1;
    PagedPlan p;
    paged_plan(sh, seqs, p);
    printf("%d %d %zu %zu %zu %zu\n", sh.few_step, sh.many_step, sh.part_rows, p.few.size(), p.many.size(), p.merges.size());
    printf("%zu %d", p.n_few, (int)p.once);
    for (auto& i : p.few) printf(" %d", i.next);
    printf("\n");
    for (auto* v : {&p.few, &p.many})
        for (auto& i : *v) printf("%d %d %d %d %d %d %d %d %d %d\n", i.q0, i.past, i.kv_len, i.row0, i.rows, i.a, i.b, i.v0, i.v1, i.part);
    for (auto& m : p.merges) printf("%d %d %d %d %d\n", m.q0, m.row0, m.rows, m.part, m.n_split);
    printf("%zu %zu\n", paged_max_tiles(n, max_tokens, sh.G), (size_t)(2 * (sh.few_target + sh.many_target)));
    return 0;
}
static int groups() {
    int t0, q, kv, log_page;
    size_t n;
    if (scanf("%d %d %d %d %zu", &t0, &q, &kv, &log_page, &n) != 5) return 1;
    std::vector<int32_t> ids(n);
    for (auto& x : ids) if (scanf("%d", &x) != 1) return 1;
    std::vector<PagedGroup> g(paged_max_groups(1, q) + 1);
    const PagedGroup* end = paged_groups(t0, q, kv, ids.data(), log_page, g.data());
    for (const PagedGroup* p = g.data(); p < end; p++) printf("%d %d %d %d\n", p->t0, p->n, p->row, p->pos);
    return 0;
}
int main(int, char** v) {
    if (!strcmp(v[1], "groups")) return groups();
    return strcmp(v[1], "check") ? plan() : check(); }
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-D_GLIBCXX_ASSERTIONS", "-I", CSRC, str(d / "main.cpp"), "-o",
                    str(d / "main")], check=True)

    def run(what, *numbers):
        return subprocess.run([str(d / "main"), what], input=" ".join(map(str, numbers)), capture_output=True, text=True, check=True).stdout
    return run


LIM = (3, 20, 4, 10, 16)   # sequences, tokens, pages of a sequence, of the pool, positions of a page


@pytest.mark.parametrize("q,kv,pages,fault,word", [
    ([], [], [], 0, ""),
    ([1], [1], [[0]], 0, ""),
    ([0, 5], [0, 40], [[-1, -1, -1], [3, -1, 9]], 0, ""),
    ([0, 5], [20, 21], [[1, 2], [1, 5]], 0, ""),                    # a shared prefix
    ([5, 0], [21, 20], [[1, 2], [1, 2]], 0, ""),                    # read while it grows
    ([1] * 4, [1] * 4, [[i] for i in range(4)], 1, "room for 3"),
    ([-1], [5], [[0]], 1, "new tokens"),
    ([6], [5], [[0]], 1, "kv_len 5"),
    ([1], [0x7ffff001], [[0]], 1, "2^31"),
    ([1], [65], [[0, 1, 2, 3, 4]], 1, "needs 5 pages"),
    ([1], [17], [[0]], 1, "the table has 1"),
    ([21], [21], [[0, 1]], 1, "room for 20"),
    ([1], [17], [[0, 10]], 2, "is 10"),
    ([1], [17], [[-2, 1]], 2, "is -2"),
    ([3, 3], [20, 20], [[1, 2], [3, 2]], 2, "two places"),
    ([20], [20], [[4, 4]], 2, "two places"),
])
def test_what_a_step_is_refused_for(program, q, kv, pages, fault, word):
    stride = max((len(p) for p in pages), default=0)
    out = program("check", *LIM, len(q), stride, *q, *kv, *(x for p in pages for x in p))
    got, msg = out.split(" ", 1)
    assert int(got) == fault and word in msg, out


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q,kv", [(1, 1), (1, 16), (1, 17), (0, 5), (16, 16), (16, 40), (33, 64), (100, 259), (2, 33), (31, 47)])
def test_tokens_in_groups_of_a_block(program, page, q, kv):
    rng = random.Random(q + kv)
    ids = rng.sample(range(40), -(-kv // page))
    ids[rng.randrange(len(ids))] = -1
    lines = [list(map(int, l.split())) for l in program("groups", 7, q, kv, page.bit_length() - 1, len(ids), *ids).splitlines()]
    got = [(t + i, row + i if row >= 0 else -1, pos + i) for t, n, row, pos in lines for i in range(n)]
    want = [(7 + i, ids[p // page] * page + p % page if ids[p // page] >= 0 else -1, p) for i, p in enumerate(range(kv - q, kv))]
    assert got == want and len(lines) <= min(q, q // 16 + 2)
    assert all(pos // 16 == (pos + n - 1) // 16 for _, n, _, pos in lines)


def cover(program, G, n_kv, window, n_sink, f16, hd, seqs):
    tokens = max(sum(q for q, _ in seqs), 1)
    lines = [list(map(int, l.split())) for l in program(
        "plan", G, n_kv, window, n_sink, int(f16), hd, tokens, len(seqs), *(x for s in seqs for x in s)).splitlines()]
    few_step, many_step, part_rows, n_few, n_many, n_merges = lines[0]
    n_groups, once, *nexts = lines.pop(1)
    few, many = lines[1:1 + n_few], lines[1 + n_few:1 + n_few + n_many]
    merges = lines[1 + n_few + n_many:1 + n_few + n_many + n_merges]
    # every item of few rows belongs to one workgroup, and its chain ends
    taken = []
    for i in range(n_groups):
        while i >= 0:
            taken.append(i)
            i = nexts[i]
    assert sorted(taken) == list(range(n_few))
    q_of = {sum(q for q, _ in seqs[:s]): q for s, (q, _) in enumerate(seqs) if q}
    assert once == (sum(i[8] - i[7] for i in few) * n_kv * 128 * hd >= 160 << 20 and all(q_of[i[0]] * G <= 16 for i in few))
    tiles, extra = lines[-1]
    assert n_merges <= tiles and max(n_few, n_many) <= tiles + extra   # what batch_create has room for
    starts = [sum(q for q, _ in seqs[:s]) for s in range(len(seqs))]
    seen, parts, states = {}, {}, set()
    for items, step, tile in ((few, few_step, 16), (many, many_step, 128)):
        for q0, past, kv, row0, rows, a, b, v0, v1, part in items:
            assert 0 < rows <= tile and v0 < v1
            s = max(i for i, q in enumerate(starts) if q == q0 and seqs[i][0])
            assert (seqs[s][1], seqs[s][1] - seqs[s][0]) == (kv, past)
            steps = [v if v < a else v - a + b for v in range(v0, v1)]
            assert all(0 <= x * step < kv for x in steps)
            for r in {row0, row0 + rows - 1}:   # (the rows between see less than these two together)
                seen.setdefault((s, r), []).extend((x * step, step) for x in steps)
            for r in range(row0, row0 + rows):
                parts.setdefault((s, r), []).append(part)
            if part >= 0:
                mine = set(range(part, part + rows))
                assert not mine & states and part + rows <= part_rows
                states |= mine
    for s, (q, kv) in enumerate(seqs):
        for r in range(q * G):
            at = parts.pop((s, r))
            assert (at == [-1]) or (len(at) > 1 and -1 not in at)
            if len(at) > 1:
                m = [x for x in merges if x[0] == starts[s] and x[1] <= r < x[1] + x[2]]
                assert len(m) == 1 and sorted(at) == [m[0][3] + i * m[0][2] for i in range(m[0][4])]
            if (s, r) in seen:
                p = kv - q + r // G
                want = {j for j in range(p + 1) if not window or j > p - window or j < n_sink}
                got = [j for base, step in seen[s, r] for j in range(base, base + step)]
                assert len(got) == len(set(got)) and want <= set(got)
    assert not parts


@pytest.mark.parametrize("seqs", [
    [(1, 1)], [(1, 4096)], [(1, 50000)], [(0, 0), (0, 7)], [(0, 100), (1, 100), (0, 0), (3, 3)],
    [(5, 3000), (1, 17), (40, 40), (200, 1000)], [(1, 100 + 97 * i) for i in range(40)], [(1000, 1000)], [(300, 20000)]])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (100, 4), (1000, 200), (5, 64), (100000, 7)])
def test_every_row_sees_its_positions_once(program, seqs, window, n_sink):
    rng = random.Random(len(seqs) + window)
    G, n_kv = rng.choice([(1, 8), (4, 8), (7, 2), (20, 1), (2, 64)])
    for f16, hd in ((True, 128), (False, 64), (True, 256)):
        cover(program, G, n_kv, window, n_sink, f16, hd, seqs)


@pytest.mark.parametrize("lens", [(700, 650, 600, 720, 690), tuple(900 + 17 * i for i in range(8)), (1500,) * 3])
def test_shares_go_on_from_one_sequence_to_the_next(program, lens):
    """Some workgroup has two sequences, all have about the same work, and tiles that read the same keys are not cut so."""
    goes_on = 0
    for hd, slots in ((64, 12), (128, 8), (256, 4)):
        for new in (1, 17):
            cover(program, 1, 64, 0, 0, True, hd, [(new, n) for n in lens])
            out = program("plan", 1, 64, 0, 0, 1, hd, new * len(lens), len(lens), *(x for n in lens for x in (new, n))).splitlines()
            n_few, (groups, _, *nexts) = int(out[0].split()[3]), map(int, out[1].split())
            items = [list(map(int, l.split())) for l in out[2:2 + n_few]]
            if new == 17:
                assert groups == n_few
            elif groups < n_few:
                goes_on += 1
                assert groups <= slots
                load = []
                for i in range(groups):
                    load.append(0)
                    while i >= 0:
                        load[-1] += items[i][8] - items[i][7] + 4
                        i = nexts[i]
                # a share and what a tile's end adds to it, less than four steps; the last may be short
                assert max(load) <= min(load[:-1]) + 11 + max(load) / 16
    assert goes_on


def test_drawn_steps(program):
    rng = random.Random(5)
    for _ in range(150):
        seqs = []
        for _ in range(rng.choice([1, 2, 5, 30])):
            q = rng.choice([0, 1, 1, rng.randint(1, 20), rng.randint(1, 300)])
            seqs.append((q, q + rng.choice([0, rng.randint(0, 50), rng.randint(0, 3000)])))
        w = rng.choice([0, 0, rng.randint(1, 2000)])
        cover(program, rng.choice([1, 2, 4, 7, 20]), rng.choice([1, 2, 8, 32]), w, rng.choice([0, 4, 300]) if w else 0,
              rng.random() < 0.7, rng.choice([64, 128, 256]), seqs)


@pytest.mark.parametrize("n_kv", [1, 8, 100, 512, 513, 700, 5000, 65535])
def test_partial_states_have_a_bound(program, n_kv):
    """64 MiB with 128 dims, whatever the number of kv heads."""
    for hd in (64, 128, 256):
        for seqs in ([(1, 5000)], [(40, 900), (1, 3)], [(300, 3000)]):
            out = program("plan", 2, n_kv, 0, 0, 1, hd, 1000, len(seqs), *(x for s in seqs for x in s)).splitlines()
            assert int(out[0].split()[2]) * n_kv * hd * 4 <= (64 << 20) * hd // 128
            cover(program, 2, n_kv, 0, 0, True, hd, seqs)
