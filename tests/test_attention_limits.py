"""Arguments of attention at the ends of their types' ranges: what the host computes from them before anything runs."""
import sys

import pytest

torch = pytest.importorskip("torch")
from test_attention_reference import FAKE, attention_args, cache_of  # noqa: E402

BIG = [2**31 - 1, 2**31, 2**32, 2**62, 2**63 - 100, 2**63 - 41, 2**63 - 32, sys.maxsize]


@pytest.mark.parametrize("window", BIG)
@pytest.mark.parametrize("kind", [1, 3])
def test_a_window_past_every_key_is_none(pkg, window, kind):
    """As much workspace as without a window: one token and prompts, one sequence and many, long caches and short."""
    scales = FAKE if kind == 3 else 0
    for d in (64, 128, 256):
        cache = cache_of(pkg, heads=8, d=d, type=kind, ks=scales, vs=scales)
        for seqs, new in ((1, 1), (1, 700), (8, 5), (300, 1)):
            for most_kv in (20, 4096, 131072, 2**31 - 1):
                ask = lambda w: pkg.lib().iq4xs_paged_attention_workspace_bytes(  # noqa: E731
                    attention_args(pkg, cache, hq=64, qs=64 * d, total=seqs * new, most_q=new, seqs=seqs, most_kv=most_kv,
                                   window=w))
                assert ask(window) == ask(0), (d, seqs, new, most_kv)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_results_with_a_window_past_every_key(pkg, new, cache):
    from test_gpu_attention import Problem

    p = Problem([new + 900, new], [new] * 2, 2, 4, 128, 16, cache)
    for causal in (True, False):
        want = p.run(pkg, torch.device("cuda:0"), causal)
        for window in (2**31 - 2, 2**31, sys.maxsize):
            got = p.run(pkg, torch.device("cuda:0"), causal, window)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 900])
@pytest.mark.parametrize("most_q,d", [(1, 128), (3, 256), (40, 64), (40, 128)])
def test_sequences_of_more_new_tokens_than_most_q(pkg, most_q, d, window, causal):
    """Their first most_q rows against a call that is told how many there are."""
    import test_gpu_attention as t

    dev, new, kv = torch.device("cuda:0"), [1200, 2, 50], [2600, 30, 700]
    print(f"[more than most_q] {most_q} {d} {window} {causal}", flush=True)
    p = t.Problem(kv, new, 2, 4, d, 16, "f16", seed=d)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    at = [s + i for s, n in zip((0, 1200, 1202), new) for i in range(min(n, most_q))]
    want, want_lse = p.run(pkg, dev, causal, window)
    got, lse = pkg.paged_attention(q, c, table, starts, kv_len, most_q, 2600, causal=causal, window=window, lse=True,
                                   scale=p.scale)
    # two ways to split the same sums, each within weights' and output's half steps (2^-11) of values below 6
    assert bool(((got[at].double() - want[at].double()).abs() <= 2 * 2 * 2.0 ** -11 * 6).all())
    assert bool(((lse[at] - want_lse[at]).abs() <= 2.0 ** -14).all())


def rising(starts, rows):
    """For each row the sequence whose start is the last at or below it, counted as the kernels count."""
    return [sum(s <= r for s in starts) - 1 for r in rows]


FALLING = [[100, 200, 300, 5], [700, 900, 1000, 0], [0, 50, 20, 60]]


def test_starts_that_fall_put_rows_before_their_sequence():
    """The count of starts at or below a row then names a sequence that begins after it: what the kernels must look for."""
    for starts in FALLING[:2]:
        seq = rising(starts, range(60))
        assert any(0 <= s < 3 and starts[s] > r and starts[s + 1] > starts[s] for r, s in enumerate(seq))


@pytest.mark.gpu
@pytest.mark.parametrize("starts", FALLING)
def test_starts_that_fall_stay_in_bounds(pkg, starts):
    """Not a call that has an answer: rows of no sequence are zero where the cache is read back, and nothing else is read
    than tables and pages."""
    import test_gpu_attention as t

    dev = torch.device("cuda:0")
    print(f"[falling starts] {starts}", flush=True)
    p = t.Problem([3000, 2000, 1000], [20] * 3, 2, 4, 128, 16, "f16")
    q, c, table, _, kv_len = p.on(pkg, dev)
    fall = torch.tensor(starts, dtype=torch.int32, device=dev)
    k, v = pkg.kv_gather(c, table, fall, 60)
    seq = rising(starts, range(60))
    for r, s in enumerate(seq):
        if not (0 <= s < 3) or starts[s] > r:
            assert not bool(k[r].any()) and not bool(v[r].any())
    out, lse = pkg.paged_attention(q, c, table, fall, kv_len, 20, 3000, window=1500, lse=True)
    torch.cuda.synchronize()
    assert out.shape == q.shape


@pytest.mark.parametrize("over,heads,code", [
    (dict(seqs=2**30, total=2**30, most_q=2**30, hq=2**20, qs=2**27), 2**20, 9),  # the plan's products wrap to zero
    (dict(seqs=2**30, total=2**30, most_q=2**30, hq=2**20, qs=2**27), 1, 9),
    (dict(total=2**28, most_q=2**28, hq=8, qs=1024), 8, 9),                       # a workgroup for each row and head
    (dict(seqs=2**30, total=100, most_q=100, hq=8, qs=1024), 8, 9),               # for each sequence and head
    (dict(seqs=2**31 - 64), 2, 1), (dict(seqs=2**31 - 1), 2, 1)])
def test_calls_too_large_to_launch_are_refused(pkg, over, heads, code):
    cache = cache_of(pkg, heads=heads)
    args = attention_args(pkg, cache, **over)
    assert pkg.lib().iq4xs_paged_attention_workspace_bytes(args) == 0
    assert pkg.lib().iq4xs_paged_attention(args, FAKE, 1 << 62, None) == code


def test_the_stride_between_the_heads_of_one_head_says_nothing(pkg):
    x = torch.zeros(3, 7, 128).transpose(0, 1)  # [tokens, heads, head], a head's tokens one after another
    assert pkg._rows(x[:, :1], "q") == (7, 1, 128, 128)
    assert pkg._rows(torch.zeros(7, 3, 128)[:, 1:2], "q") == (7, 1, 128, 384)
    for bad in (x, x[:, :2], torch.zeros(7, 1, 256)[..., ::2]):
        with pytest.raises(ValueError):
            pkg._rows(bad, "q")


@pytest.mark.gpu
def test_one_head_of_another_layout(pkg):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(4, 9, 128, generator=g, device=dev).half().transpose(0, 1)  # [9 tokens, 4 heads, 128]
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    views, copies = [x[:, i:i + 1] for i in range(3)], [x[:, i:i + 1].contiguous() for i in range(3)]
    assert all(torch.equal(a, b) for a, b in zip(pkg.qk_norm_rope(*views[:2], pos), pkg.qk_norm_rope(*copies[:2], pos)))
    results = []
    for q, k, v in (views, copies):
        cache = pkg.KVCache(*(torch.zeros(1, 1, 16, 128, dtype=torch.float16, device=dev) for _ in range(2)))
        q = pkg.qk_norm_rope_append(q, k, v, pos, pos.long(), cache)
        results.append((q, cache.k_pages, cache.v_pages))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    i32 = lambda *n: torch.tensor(n, dtype=torch.int32, device=dev)  # noqa: E731
    out = [pkg.paged_attention(q, cache, i32(0)[None], i32(0, 9), i32(9), 9, 9) for q in (views[0], copies[0])]
    assert torch.equal(*out)


@pytest.mark.gpu
@pytest.mark.parametrize("new,d", [(1, 128), (5, 256), (60, 64)])
def test_most_kv_off_the_truth(pkg, new, d):
    """Below it the first keys count, as if the sequences were that long; above it the splits change and nothing else."""
    import test_gpu_attention as t

    dev = torch.device("cuda:0")
    print(f"[most_kv] {new} {d}", flush=True)
    p = t.Problem([3000, new + 100, 700], [new] * 3, 2, 4, d, 16, "f16", seed=d)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    ask = lambda lens, most: pkg.paged_attention(q, c, table, starts, lens, new, most, lse=True)  # noqa: E731
    cut = ask(kv_len, 1000)
    assert all(torch.equal(a, b) for a, b in zip(cut, ask(kv_len.clamp(max=1000), 1000)))
    for most in (3001, 100000, 2**31 - 1):
        out, lse = ask(kv_len, most)
        want, want_lse = ask(kv_len, 3000)
        # two ways to split the same sums, each within weights' and output's half steps (2^-11) of values below 6
        assert bool(((out.double() - want.double()).abs() <= 2 * 2 * 2.0 ** -11 * 6).all())
        assert bool(((lse - want_lse).abs() <= 2.0 ** -14).all())
