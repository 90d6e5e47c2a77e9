"""The chunk attention's division of a call into units and shares, on the CPU.

tinybrain_b200/csrc/tb_chunk_walk.h is plain arithmetic on the lengths.  Compiled
with the host's compiler here, the shares of a call are walked as the kernels walk
them and compared with the units written down one by one: every tile belongs to
exactly one share, every unit has the rows and positions of its definition, and no
walk leaves the batch (which on the GPU would read beyond the caller's arrays).
"""
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinybrain_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "tb_chunk_walk.h"
using namespace tb;

struct Place { int s, tile, head, limit, tiles; long long begin; };
#define FAIL(...) { printf(__VA_ARGS__); printf("\n"); return; }

template <int NT, int ROWS>
void check(const ChunkParams& p, long long ctas) {
    const int G = p.H / p.Hkv, per = ROWS / G;
    std::vector<Place> all;  // by definition
    long long total = 0, counted = 0;
    for (int s = 0; s < p.batch; ++s) {
        const long long n = p.row_offsets[s + 1] - p.row_offsets[s], len = p.total_lens[s];
        for (long long t0 = 0; t0 < n; t0 += per)
            for (int h = 0; h < p.Hkv; ++h) {
                const long long seen = len - n + (t0 + per < n ? t0 + per : n);
                const long long limit = seen < 0 ? 0 : seen < p.stride * 16ll ? seen : p.stride * 16ll;
                const long long tiles = limit ? (limit + NT - 1) / NT : 1;
                all.push_back({s, (int)(t0 / per), h, (int)limit, (int)tiles, total});
                total += tiles;
            }
        counted += tiles_of_sequence<NT, ROWS>(p, s);
    }
    if (counted != total) FAIL("counted %lld tiles of %lld", counted, total);
    const long long shares = std::min(ctas, total);
    size_t at = 0;
    for (long long c = 0; c < shares; ++c) {
        Share share{total, shares, c, total * (c + 1) / shares, 0};
        const long long begin = total * c / shares;
        while (begin >= all[at].begin + all[at].tiles) ++at;
        Unit u;
        u.s = all[at].s, u.tile = all[at].tile, u.head = all[at].head;
        set_sequence(p, u);
        set_tile<NT, ROWS>(p, u);
        size_t i = at;
        for (long long g = begin; g < share.end;) {
            const Place& w = all[i];
            if (u.s != w.s || u.tile != w.tile || u.head != w.head || u.limit != w.limit || u.tiles != w.tiles)
                FAIL("share %lld of %lld: sequence %d tile %d head %d, not %d %d %d", c, shares, u.s, u.tile, u.head, w.s,
                     w.tile, w.head);
            const long long end = w.begin + w.tiles;
            if (end > share.end && w.begin >= begin) {  // it goes on: in how many shares
                int more = 0;
                while (total * (c + more + 1) / shares < end) ++more;
                if (share.followers((int)(end - share.end)) != more) FAIL("share %lld: followers, not %d", c, more);
            }
            g = end;
            if (g < share.end) {
                next_unit<NT, ROWS>(p, u);
                if (u.s < 0 || u.s >= p.batch) FAIL("share %lld of %lld leaves the batch", c, shares);
                ++i;
            }
        }
    }
    // a walk that goes on past the last unit stays where the arrays are
    if (!all.empty()) {
        Unit u;
        u.s = all.back().s, u.tile = all.back().tile, u.head = all.back().head;
        set_sequence(p, u);
        set_tile<NT, ROWS>(p, u);
        for (int k = 0; k < 3 * p.Hkv; ++k) {
            next_unit<NT, ROWS>(p, u);
            if (u.s < 0 || u.s >= p.batch) FAIL("the walk leaves the batch after the last unit");
        }
    }
    printf("ok\n");
}

int main() {
    int nt, rows, G, kv, stride, batch;
    long long ctas;
    while (scanf("%d %d %d %d %lld %d %d", &nt, &rows, &G, &kv, &ctas, &stride, &batch) == 7) {
        std::vector<int> offsets(batch + 64, 0), lens(batch + 64, 0);  // (room: a walk that fails is seen, not felt)
        for (int s = 0; s < batch; ++s) {
            int n;
            if (scanf("%d %d", &n, &lens[s]) != 2) return 1;
            offsets[s + 1] = offsets[s] + n;
        }
        ChunkParams p{};
        p.row_offsets = offsets.data(), p.total_lens = lens.data();
        p.batch = batch, p.rows = offsets[batch], p.stride = stride;
        p.H = G * kv, p.Hkv = kv, p.rows_above = 0, p.rows_upto = 1 << 30;
        if (nt == 64 && rows == 128) check<64, 128>(p, ctas);
        else if (nt == 128 && rows == 128) check<128, 128>(p, ctas);
        else if (nt == 16 && rows == 8) check<16, 8>(p, ctas);
        else return 1;
    }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", CSRC, "-o", str(d / "walk"), str(d / "walk.cpp")])

    def run(cases):
        """cases: (positions of a tile, rows of a unit, G, KV heads, shares, [(new, length), ...])."""
        lines = []
        for nt, rows, G, kv, ctas, seqs in cases:
            stride = max(1, max(-(-t // 16) for _, t in seqs))
            lines.append(" ".join(map(str, [nt, rows, G, kv, ctas, stride, len(seqs)] + [x for s in seqs for x in s])))
        r = subprocess.run([str(d / "walk")], input="\n".join(lines), capture_output=True, text=True, check=True)
        got = r.stdout.splitlines()
        assert len(got) == len(cases)
        bad = [(c[:5], c[5][:3], g) for c, g in zip(cases, got) if g != "ok"]
        assert not bad, (len(bad), bad[:5])

    return run


@pytest.mark.parametrize("nt,rows,most", [(64, 128, 128), (128, 128, 128), (16, 8, 8)])
@pytest.mark.parametrize("batch", [1, 16])
def test_shares_hold_every_tile_once_for_any_head_group(walk, nt, rows, most, batch):
    cases = []
    for G in range(1, most + 1):
        per = rows // G
        for k in (1, 2, 3, 5, 8, 17):
            for n in (k * per - 1, k * per, k * per + 1):  # about a row tile's end
                if n > 0:
                    cases += [(nt, rows, G, kv, ctas, [(n, n + held)] * batch)
                              for kv, ctas, held in ((1, 148, 0), (4, 148, 700), (2, 7, 33), (3, 1, 0))]
    walk(cases)


def test_shares_of_long_prompts_at_every_length(walk):
    walk([(64, 128, G, kv, 148, [(n, n)]) for G, kv in ((7, 4), (5, 8), (3, 8), (6, 2)) for n in range(20, 2049, 7)])
    walk([(64, 128, 7, 4, 148, [(n, 8192)]) for n in (512, 1291, 2048)])


def test_shares_of_ragged_batches(walk):
    g = np.random.default_rng(0)
    cases = []
    for _ in range(300):
        nt, rows = [(64, 128), (128, 128), (16, 8)][g.integers(3)]
        G, batch = int(g.integers(1, min(rows, 40) + 1)), int(g.integers(1, 30))
        total = g.integers(0, 900, batch)
        new = np.where(g.random(batch) < 0.3, 0, g.integers(0, 300, batch))  # some idle, some with more rows than tokens
        if new.any():
            cases.append((nt, rows, G, int(g.integers(1, 9)), int(g.integers(1, 149)), list(zip(new.tolist(), total.tolist()))))
    walk(cases)
