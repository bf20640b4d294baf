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
