"""Linear attention: where workgroups and states of segments are counted (csrc/linear_plan.h), compiled for the host, and what a
batch of one prompt and many single tokens asks for (no GPU)."""
import os
import random
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")
from test_linear_attention import args  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# lines: heads in_type most_q total seqs, seqs + 1 starts; answers: what goes wrong, 0 for nothing, then places of workgroups,
# of states, and of launches that join
PLACES = """
#include "linear_plan.h"
#include <iostream>
#include <set>
#include <vector>
using namespace iq4xs;
int main() {
    iq4xs_linear_attention_args g = {};
    while (std::cin >> g.heads >> g.in_type >> g.most_q >> g.total >> g.seqs) {
        std::vector<int> starts(g.seqs + 1);
        for (int& s : starts) std::cin >> s;
        g.dk = g.dv = 128;
        LinearPlan p;
        if (!linear_plan(g, 256, p) || p.steps) return 1;
        const int64_t units = g.heads * (g.dv / linear_chunk_columns(g.dk, g.dv));
        const int64_t runs = places_in(p.runs, g.total, g.seqs), kept = places_in(p.kept, g.total, g.seqs);
        const int64_t joins = p.join_rows ? joining_rows(g.total, p.length) : g.seqs;
        std::set<int64_t> run, state, joined;
        int wrong = p.grid != runs * units;
        for (int64_t j = 0; j < joins && p.join_rows; ++j) {
            const int64_t row = 2 * j * p.length;
            int seq = -1;
            for (int i = 0; i < g.seqs; ++i) if (starts[i] <= row) seq = i;
            if (seq >= 0 && row - starts[seq] < 2 * (int64_t)p.length) wrong += !joined.insert(seq).second;
        }
        for (int i = 0; i < g.seqs; ++i) {
            int64_t n = starts[i + 1] - starts[i];
            if (n > g.most_q) n = g.most_q;
            const int64_t parts = (n + p.length - 1) / p.length;
            for (int64_t part = 0; part < parts; ++part) {
                const int64_t at = p.runs.of(starts[i], i) + part;
                wrong += at < 0 || at >= runs || !run.insert(at).second;
                int seq = -1;  // as the kernel finds it
                for (int s = 0; s < g.seqs; ++s) if (p.runs.of(starts[s], s) <= at) seq = s;
                wrong += seq != i;
                if (parts > 1) {
                    const int64_t to = p.kept.of(starts[i], i) + part;
                    wrong += to < 0 || to >= kept || !state.insert(to).second;
                }
            }
            wrong += parts > p.segments || (parts > 2 && p.join_rows && !joined.count(i));
        }
        if (p.segments > 1) {
            wrong += kept > 2 * g.total / p.length || kept > g.seqs * p.segments || kept > g.total / p.length + g.seqs;
            wrong += runs > g.total / p.length + g.seqs || joins > g.total / (2 * p.length) + 1;
        }
        std::cout << wrong << " " << runs << " " << kept << " " << joins << "\\n";
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")
    d = tmp_path_factory.mktemp("places")
    (d / "s.cpp").write_text(PLACES)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "qwen_3.8_27b_optimizations_amd", "csrc"), str(d / "s.cpp"), "-o",
                    str(d / "s")], check=True)

    def run(batches):
        lines = []
        for heads, kind, most, before, after, lens in batches:
            starts = [before + sum(lens[:i]) for i in range(len(lens) + 1)]
            lines.append(" ".join(map(str, [heads, kind, most, starts[-1] + after, len(lens), *starts])))
        r = subprocess.run([str(d / "s")], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True)
        out = [tuple(map(int, x.split())) for x in r.stdout.splitlines()]
        assert len(out) == len(batches)
        return out

    return run


def test_every_segment_has_a_place_of_its_own(ask):
    rng = random.Random(1)
    spread = lambda n: int(n ** rng.random())  # noqa: E731
    batches = [(2, 2, 1500, 0, 0, [1500] + [1] * 63), (2, 2, 1500, 7, 0, [1] * 63 + [1500]), (2, 2, 513, 0, 0, [513, 0, 0, 513]),
               (1, 2, 257, 0, 3, [257] * 20), (64, 2, 4096, 0, 0, [4096]), (1, 0, 10**9, 5, 0, [10**9, 1, 0, 10**9 - 1])]
    for _ in range(400):
        lens = [rng.choice([0, 1, 1, spread(40), spread(3000), spread(9000)]) for _ in range(rng.choice([1, 2, 5, 30, 90]))]
        lens[rng.randrange(len(lens))] = 300 + spread(6000)
        batches.append((rng.choice([1, 2, 16, 64]), rng.randrange(3), max(max(lens) - rng.choice([0, 0, 100]), 17),
                        rng.choice([0, 3, 700]), rng.choice([0, 5]), lens))
    bad = [(b, w) for b, w in zip(batches, ask(batches)) if w[0]]
    assert not bad


def test_a_prompt_among_many_single_tokens(pkg, ask):
    """States of segments for the prompt alone, and workgroups for no more than all sequences."""
    L = pkg.lib()
    for seqs, runs in ((64, 72), (256, 264), (1024, 1034)):
        total = 4096 + seqs - 1
        need = L.iq4xs_linear_attention_workspace_bytes(args(pkg, it=2, heads=64, hk=64, qs=8192, ks=8192, vs=8192, seqs=seqs,
                                                             total=total, most_q=4096))
        assert 0 < need < 100e6, (seqs, need)
        wrong, places, kept, joins = ask([(64, 2, 4096, 0, 0, [4096] + [1] * (seqs - 1))])[0]
        assert not wrong and places <= runs and kept <= 20 and joins <= 6, (seqs, places, kept, joins)
