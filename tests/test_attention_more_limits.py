"""Lengths at the ends of their ranges in calls with first tokens and with shared prefixes, and the blocks that the Python side
passes (no GPU)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = """
#include "attention_plan.h"
#include <cstdio>
#include <initializer_list>
using namespace iq4xs;
static bool fine(const AttentionPlan& p, int64_t most_kv) {
    const int64_t keys = most_kv < KEYS_END ? most_kv : KEYS_END;
    return p.chunk > 0 && p.chunk % 128 == 0 && p.splits > 0 && p.grid > 0 && p.grid % p.splits == 0 &&
           (int64_t)p.chunk * p.splits >= keys && (int64_t)p.chunk * (p.splits - 1) < keys;
}
int main() {
    const int64_t most = 0x7FFFFFFF;
    for (int type : {1, 3}) for (int d : {64, 128, 256}) for (int heads : {1, 8}) for (int64_t group : {1, 8})
        for (int64_t seqs : {1, 3, 64, 528, 1000, 5000}) for (int64_t groups : {1, 2, 300})
            for (int64_t len : {(int64_t)1, (int64_t)8187, most / 2, (int64_t)KEYS_END - 1, (int64_t)KEYS_END, most - 128,
                                most - 127, most})
                for (int64_t own : {(int64_t)1, (int64_t)9001, (int64_t)KEYS_END, most - 127, most}) for (int path : {0, 1, 2}) {
                    iq4xs_kv_cache cache = {};
                    cache.heads = heads, cache.head_dim = d, cache.type = type;
                    iq4xs_paged_attention_args g = {};
                    g.cache = &cache, g.q_heads = (int)(heads * group), g.out_type = 1, g.causal = 1;
                    g.seqs = g.total = seqs, g.most_q = 1, g.most_kv = own;
                    iq4xs_shared_prefix x = {};
                    x.groups = groups, x.most_len = len, x.most_rows = seqs, x.path = path;
                    SharedPlan p;
                    bool ok = shared_plan_fits(g, x, 256, p);
                    if (ok && p.once) ok = fine(p.prefix, len) && fine(p.own, own) && p.parts() == p.prefix.splits + p.own.splits;
                    else if (ok) ok = fine(p.own, len + own);
                    if (!ok) std::printf("%d %d %d %d %d %d %lld %lld %d\\n", type, d, heads, (int)group, (int)seqs, (int)groups,
                                         (long long)len, (long long)own, path);
                }
}
"""


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")

    def run(text):
        d = tmp_path_factory.mktemp("host")
        (d / "s.cpp").write_text(text)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        "-I" + os.path.join(ROOT, "include"),
                        "-I" + os.path.join(ROOT, "qwen_3.8_27b_optimizations_amd", "csrc"), str(d / "s.cpp"), "-o",
                        str(d / "s")], check=True)
        return subprocess.run([str(d / "s")], capture_output=True, text=True, check=True).stdout

    return run


def test_plans_of_the_longest_lengths(compiled):
    """`At least` so many tokens, up to the largest number: splits hold every key that counts, and none is empty."""
    assert compiled(PLAN) == ""


def test_blocks_are_whole_structs(pkg, compiled):
    """What the Python side passes is as long as the struct, padding and all: the library copies it."""
    sizes = compiled('#include "iq4xs_mi355x.h"\n#include <cstdio>\nint main() { std::printf("%zu %zu %zu", '
                     "sizeof(iq4xs_paged_attention_args), sizeof(iq4xs_shared_prefix), sizeof(iq4xs_linear_attention_args)); }")
    layouts = (pkg._ATTENTION, pkg._SHARED, pkg._LINEAR)
    blocks = [pkg._block(x, *x.unpack(bytes(x.size))) for x in layouts]
    assert [len(b) for b in blocks] == [int(n) for n in sizes.split()]
    source = open(pkg.__file__).read()
    assert all(f"_{name}.pack(" not in source for name in ("ATTENTION", "SHARED", "LINEAR"))
