"""Attention with first tokens and with shared prefixes: the 64-bit form against the row-by-row one, and refusals before
anything is launched (no GPU)."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")
import attention_more_reference as more  # noqa: E402
import attention_reference as ref  # noqa: E402
from test_attention_reference import BAD_ATTENTION, BAD_CACHES, FAKE, attention_args, cache_of  # noqa: E402
from test_gpu_attention import Problem  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 7), (False, 5), (False, 0)])
def test_the_reference_without_first_tokens_is_the_plain_one(cache, causal, window):
    p = Problem([20, 3, 0, 33], [5, 3, 2, 1], 2, 3, 64, 16, cache)
    p.table[0, 1] = -1
    want = ref.attention(p.q, p.k, p.v, p.ks, p.vs, p.table, p.starts, p.kv_len, causal, window, p.scale)
    got = more.attention(p, more.window_and_sinks(causal, window, 0))
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_first_tokens_are_keys_before_the_window():
    sees = more.window_and_sinks(True, 3, 2)(0, torch.tensor([[0], [1], [4], [9]]), torch.arange(10)[None])
    assert [[j for j in range(10) if r[j]] for r in sees.tolist()] == [[0], [0, 1], [0, 1, 2, 3, 4], [0, 1, 7, 8, 9]]


def shared_of(pkg, **over):
    f = dict(first=0, len=FAKE, groups=1, most_len=16, most_rows=3, path=pkg.SHARED_ONCE)
    f.update(over)
    return pkg._SHARED.pack(*f.values()) + bytes(4)


def test_the_struct_matches_the_header(pkg, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")
    src = tmp_path / "s.cpp"
    src.write_text('#include "iq4xs_mi355x.h"\n#include <cstdio>\nint main() { std::printf("%zu %zu", '
                   'sizeof(iq4xs_shared_prefix), offsetof(iq4xs_shared_prefix, path)); }')
    subprocess.run(["g++", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    size, last = map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split())
    assert last + 4 == pkg._SHARED.size and size >= pkg._SHARED.size


BAD_SHARED = [dict(len=0), dict(groups=0), dict(groups=-1), dict(groups=2), dict(groups=1 << 31, first=FAKE),
              dict(most_len=0), dict(most_len=1 << 31), dict(most_rows=0), dict(most_rows=-1), dict(path=3),
              dict(path=-1)]


def test_refusals_before_launch(pkg):
    L, E, N, C = pkg.lib(), pkg.ERROR_INVALID_VALUE, pkg.ERROR_NOT_SUPPORTED, pkg.ERROR_INVALID_CONFIG
    good = cache_of(pkg)

    def both(args, prefix=None):
        prefix = shared_of(pkg) if prefix is None else prefix
        assert L.iq4xs_shared_attention_workspace_bytes(args, prefix) == 0
        return (L.iq4xs_paged_attention_sinks(args, 4, FAKE, 1 << 40, None),
                L.iq4xs_shared_attention(args, prefix, FAKE, 1 << 40, None))

    for over in BAD_CACHES:
        cache = cache_of(pkg, **over)
        assert both(attention_args(pkg, cache)) == (E, E), over
    cache = cache_of(pkg, d=96)
    assert both(attention_args(pkg, cache)) == (N, N)
    for over in BAD_ATTENTION:
        assert both(attention_args(pkg, good, **over)) == (E, E), over
    assert both(None) == (E, E)
    args = attention_args(pkg, good)
    for sinks in (-1, -2**63):
        assert L.iq4xs_paged_attention_sinks(args, sinks, FAKE, 1 << 40, None) == E
    for over in BAD_SHARED:
        bad = shared_of(pkg, **over)
        assert L.iq4xs_shared_attention_workspace_bytes(args, bad) == 0, over
        assert L.iq4xs_shared_attention(args, bad, FAKE, 1 << 40, None) == E, over
    assert L.iq4xs_shared_attention(args, None, FAKE, 1 << 40, None) == E
    # a window with a shared prefix is another call's work
    assert L.iq4xs_shared_attention(attention_args(pkg, good, window=8), shared_of(pkg), FAKE, 1 << 40, None) == N
    # launches too large for a grid, workspaces too small or not aligned
    cache = cache_of(pkg, heads=1)
    wide = attention_args(pkg, cache, hq=1 << 16, qs=(1 << 16) * 128, total=1 << 16, most_q=1 << 16)
    assert both(wide) == (C, C)
    need = L.iq4xs_shared_attention_workspace_bytes(args, shared_of(pkg))
    assert need > 0
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 16, need)):
        assert L.iq4xs_shared_attention(args, shared_of(pkg), ws, size, None) == E, (ws, size)
    long = attention_args(pkg, good, most_kv=100000, window=50000, width=8000)
    need = L.iq4xs_paged_attention_workspace_bytes(long)
    assert need > 0
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 16, need)):
        assert L.iq4xs_paged_attention_sinks(long, 4, ws, size, None) == E, (ws, size)


def test_nothing_to_do_launches_nothing(pkg):
    L, good = pkg.lib(), cache_of(pkg)
    for over in (dict(total=0), dict(seqs=0)):
        args = attention_args(pkg, good, **over)
        assert L.iq4xs_paged_attention_sinks(args, 4, None, 0, None) == 0
        assert L.iq4xs_shared_attention_workspace_bytes(args, shared_of(pkg, len=0, most_len=0)) == 0
        assert L.iq4xs_shared_attention(args, shared_of(pkg, len=0), None, 0, None) == 0


def test_each_sequence_by_itself_is_the_plain_call(pkg):
    """And taken for little that is shared, for one sequence of a group, and for full tiles of rows."""
    L, good = pkg.lib(), cache_of(pkg, heads=8)
    ask = lambda f, *a: L.iq4xs_shared_attention_workspace_bytes(f, *a)  # noqa: E731
    for seqs, new, most_len, once in ((64, 1, 16384, True), (2, 1, 100, False), (1, 1, 1 << 20, False), (3, 1, 1 << 20, True),
                                      (64, 40, 16384, False)):
        f = dict(hq=64, qs=64 * 128, total=seqs * new, most_q=new, seqs=seqs)
        args = attention_args(pkg, good, most_kv=1000, **f)
        sizes = [ask(args, shared_of(pkg, most_len=most_len, most_rows=seqs * new, path=p))
                 for p in (pkg.SHARED_AUTO, pkg.SHARED_ONCE, pkg.SHARED_EACH)]
        assert sizes[0] == sizes[1 if once else 2] and sizes[1] > 0, (seqs, new, most_len)
        whole = attention_args(pkg, good, most_kv=1000 + most_len, **f)
        assert sizes[2] == L.iq4xs_paged_attention_workspace_bytes(whole)


def test_workspaces_hold_both_launches(pkg):
    """Parts of the prefix's launch and of the sequences': sums and four statistics each for every row and head."""
    L, good = pkg.lib(), cache_of(pkg)
    for total, most_rows, most_len, most_kv in ((3, 3, 16, 20), (64, 64, 16384, 1024), (500, 200, 5000, 5000)):
        args = attention_args(pkg, good, total=total, most_q=max(1, total // 8), seqs=min(8, total), most_kv=most_kv)
        need = L.iq4xs_shared_attention_workspace_bytes(args, shared_of(pkg, most_len=most_len, most_rows=most_rows))
        part = total * 4 * (128 + 4) * 4
        assert need % part == 0 and need // part >= 2
    assert math.isfinite(need) and ctypes.sizeof(ctypes.c_size_t) == 8
