"""Attention with first tokens beside a window and with shared prefixes: the keys of the workgroups, their steps and the
parts that are joined (csrc/attention_plan.h), compiled for the host and asked about many calls: every key that a row sees
reaches it exactly once, and the parts that are joined are those that were written."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = os.environ.get("CXX", "g++")


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which(CXX) is None:
        pytest.skip("needs a host C++ compiler")
    exe = str(tmp_path_factory.mktemp("plan") / "attention_more")
    subprocess.run([CXX, "-std=c++17", "-O2", "-Wall",
                    "-I" + os.path.join(ROOT, "qwen_3.8_27b_optimizations_amd", "csrc"),
                    "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "arith", "attention_more.cpp"),
                    "-o", exe], check=True)

    def wrong(calls):
        r = subprocess.run([exe], input="\n".join(calls) + "\n", capture_output=True, text=True, check=True)
        out = [int(x) for x in r.stdout.split()]
        assert len(out) == len(calls)
        return [(c, n) for c, n in zip(calls, out) if n]

    return wrong


def words(*x):
    return " ".join(str(int(y)) for y in x)


def starts_of(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def sinks_call(new, kv, window, sinks, causal=True, heads=1, group=1, d=128, kind=1, lse=0, most_q=None, most_kv=None):
    return "sinks " + words(sum(new), max(new) if most_q is None else most_q, max(kv + [1]) if most_kv is None else most_kv,
                            window, causal, heads, group, d, kind, lse, 4, sinks, len(kv), *starts_of(new), *kv)


def shared_call(new, kv, firsts, lens, most_own, most_len, most_rows, causal=True, heads=1, group=1, d=128, kind=1, lse=0,
                most_q=None):
    return "shared " + words(sum(new), max(new) if most_q is None else most_q, most_own, causal, heads, group, d, kind, lse,
                             4, len(lens), firsts is not None, most_len, most_rows, len(kv), *starts_of(new), *kv,
                             *(firsts or []), *lens)


def test_first_tokens_and_windows(ask):
    """Windows that end within the first tokens, before them and far behind; rows that see nothing; lengths off the truth."""
    fixed = [sinks_call([1], [n], w, s, causal=c) for n in (0, 1, 2, 31, 33, 64, 65, 400) for w in (1, 2, 31, 32, 33, 200)
             for s in (1, 4, 31, 32, 33, 64, 65, 300, 500) for c in (True, False)]
    fixed += [sinks_call([300], [5000], 700, 4, heads=2, group=8), sinks_call([1], [9000], 4096, 4, heads=8, group=8)]
    assert not ask(fixed)
    rng = random.Random(3)
    spread = lambda n: int(n ** rng.random())  # noqa: E731
    calls = []
    for _ in range(700):
        seqs = rng.choice([1, 1, 2, 5])
        new = [spread(300) for _ in range(seqs)]
        kv = [max(0, rng.choice([n, n + spread(6000), n + spread(300), n - spread(50)])) for n in new]
        over = rng.random() < 0.3
        calls.append(sinks_call(new, kv, max(1, spread(3000)), spread(400), rng.random() < 0.7, rng.choice([1, 2, 8]),
                                rng.choice([1, 3, 8]), rng.choice([64, 128, 256]), rng.choice([1, 3]), rng.random() < 0.5,
                                max(1, spread(max(new))) if over else None,
                                max(1, max(kv) - spread(max(kv) + 1)) if over else max(1, max(kv))))
    assert not ask(calls)


def test_shared_prefixes(ask):
    """Groups of one and several sequences, sequences of no group, empty ones, lengths off the truth, groups that are not in
    the call."""
    fixed = [shared_call([1, 1], [70, 80], None, [64], 16, 64, 2), shared_call([0, 3], [40, 80], None, [40], 40, 40, 3),
             shared_call([2, 2, 2], [90, 91, 92], [1, 3], [64], 92, 64, 4),
             shared_call([2, 2, 2], [90, 91, 92], [0, 9], [64], 92, 64, 6),
             shared_call([2, 2, 2], [90, 91, 92], [-1, 2], [64], 92, 64, 6),
             shared_call([2, 2], [90, 91], [0, 1, 1, 2], [64, 10, 0], 92, 64, 4)]
    assert not ask(fixed)
    rng = random.Random(4)
    spread = lambda n: int(n ** rng.random())  # noqa: E731
    calls = []
    for _ in range(500):
        seqs = rng.choice([1, 2, 3, 7])
        new = [rng.choice([0, 1, spread(5), spread(150)]) for _ in range(seqs)]
        if not sum(new):
            new[0] = 1
        groups = rng.choice([1, 1, 2, 3])
        cuts = sorted(rng.randrange(0, seqs + 1) for _ in range(groups - 1))
        firsts = [rng.choice([0, 0, min(1, cuts[0] if cuts else seqs)])] + cuts + [rng.choice([seqs, seqs, max(cuts + [0])])]
        lens = [spread(5000) - 1 for _ in range(groups)]
        if groups == 1 and rng.random() < 0.5:
            firsts = None
        of = lambda i: next((g for g in range(groups) if firsts[g] <= i < firsts[g + 1]), -1) if firsts else 0  # noqa: E731
        own = [n + spread(1500) - 1 for n in new]
        kv = [o + (lens[of(i)] if of(i) >= 0 else 0) for i, o in enumerate(own)]
        off = rng.random() < 0.3
        calls.append(shared_call(new, kv, firsts, lens, max(1, spread(max(own) + 2) if off else max(own)),
                                 max(1, spread(max(lens) + 2) if off else max(lens)),
                                 max(1, spread(sum(new)) if off else sum(new)), rng.random() < 0.8, rng.choice([1, 2, 8]),
                                 rng.choice([1, 3, 8]), rng.choice([64, 128, 256]), rng.choice([1, 3]),
                                 rng.random() < 0.5, max(1, spread(max(new))) if off else None))
    assert not ask(calls)
