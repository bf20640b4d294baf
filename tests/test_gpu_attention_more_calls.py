"""Calls with first tokens and with shared prefixes that callers make now and then: batches that share nothing this step,
lengths that are only bounds, outputs without their log-sum-exp."""
import pytest

torch = pytest.importorskip("torch")
import attention_more_reference as more  # noqa: E402
from test_gpu_attention import Problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


@pytest.mark.parametrize("new", [1, 40])
def test_a_batch_that_shares_nothing(pkg, dev, new):
    p = Problem([new + 60, new + 75], [new] * 2, 2, 4, 128, 16, "f16")
    q, c, table, starts, kv_len = p.on(pkg, dev)
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    for path in (pkg.SHARED_AUTO, pkg.SHARED_ONCE, pkg.SHARED_EACH):
        out, lse = pkg.shared_attention(q, c, table, starts, kv_len, none, new, new + 75, 0, lse=True, scale=p.scale,
                                        path=path)
        more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(True, 0, 0))
    with pytest.raises(pkg.Iq4xsError):
        pkg.shared_attention(q, c, table, starts, kv_len, none, new, new + 75, -1)


# ------------------------------------------------------------------ outputs alone
def sinks_out(pkg, dev, p, window, sinks, lse=False, causal=True, **kw):
    q, c, table, starts, kv_len = p.on(pkg, dev)
    return pkg.paged_attention(q, c, table, starts, kv_len, max(p.new), max(p.kv + [1]), causal=causal, window=window,
                               lse=lse, scale=p.scale, sinks=sinks, **kw)


def shared_out(pkg, dev, p, shared, lse=False, causal=True, path=1, **kw):
    q, c, table, starts, kv_len = p.on(pkg, dev)
    n = torch.tensor([shared], dtype=torch.int32, device=dev)
    return pkg.shared_attention(q, c, table, starts, kv_len, n, max(p.new), max(p.kv) - shared, shared, causal=causal,
                                lse=lse, scale=p.scale, path=path, **kw)


def check(p, got, sees):
    """Outputs of a call without a log-sum-exp, held to the same bounds."""
    more.compare(p, got.cpu(), more.attention(p, sees)[1], sees)


@pytest.mark.parametrize("cache,q_type", [("f16", None), ("bf16", None), ("q8", "f16")])
@pytest.mark.parametrize("new,group", [([1, 1, 1], 8), ([2, 1, 5], 8), ([70, 3, 131], 2), ([400, 380, 300], 16)])
def test_outputs_alone_keep_their_bits(pkg, dev, cache, q_type, new, group):
    """What a row's statistics are wanted for says nothing about its output."""
    for d in (64, 128, 256):
        p = Problem([n + 900 + 100 * i for i, n in enumerate(new)], new, 1, group, d, 16, cache, q_type, seed=d)
        assert torch.equal(sinks_out(pkg, dev, p, 300, 40), sinks_out(pkg, dev, p, 300, 40, lse=True)[0])
        more.share(p, [0, 3], [777])
        for path in (pkg.SHARED_ONCE, pkg.SHARED_EACH):
            assert torch.equal(shared_out(pkg, dev, p, 777, path=path), shared_out(pkg, dev, p, 777, lse=True, path=path)[0])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group,window,sinks", [([2, 1, 5, 3], 8, 16, 4), ([70, 1, 131, 64], 2, 17, 4),
                                                    ([33, 40, 17, 100], 8, 64, 64), ([129, 64, 65, 63], 1, 1, 65),
                                                    ([40, 50, 31, 23], 3, 130, 3), ([75, 75, 75, 75], 4, 15, 130),
                                                    ([12, 1, 9, 5], 4, 100, 300), ([1, 1, 1, 1], 40, 33, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_first_tokens_over_rounded_codes(pkg, dev, d, new, group, window, sinks, causal):
    """An 8-bit cache, bf16 outputs and no log-sum-exp: the kernel whose keys are fp16, tiles of first tokens before it."""
    kv = [new[0], new[1] + 250, new[2], new[3] + 129]
    p = Problem(kv, new, 1, group, d, 16, "q8", "bf16", seed=d + group)
    check(p, sinks_out(pkg, dev, p, window, sinks, causal=causal), more.window_and_sinks(causal, window, sinks))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [5, 100])
def test_splits_over_rounded_codes(pkg, dev, d, new):
    p = Problem([9000, 5, 2600, 1030], [new, min(new, 5), new, new], 2, 8, d, 64, "q8", "bf16", seed=3)
    check(p, sinks_out(pkg, dev, p, 2500, 70), more.window_and_sinks(True, 2500, 70))
    # more new tokens than cached ones, empty sequences, pages of first tokens that are not in the cache
    p = Problem([new - 1, 0, 1, new], [new, new, new, 1], 2, 8, d, 16, "q8", "bf16")
    check(p, sinks_out(pkg, dev, p, 2, 4), more.window_and_sinks(True, 2, 4))
    p = Problem([new + 100, new + 20], [new] * 2, 2, 8, d, 16, "q8", "bf16")
    p.table[0, 0], p.table[1, 1] = -1, 1 << 30
    check(p, sinks_out(pkg, dev, p, 10, 20), more.window_and_sinks(True, 10, 20))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group", [([1] * 6, 8), ([2, 1, 5, 3], 8), ([70, 1, 131, 64], 2), ([33, 40, 17, 100], 5)])
def test_prefixes_over_rounded_codes(pkg, dev, d, new, group):
    """More than 32 rows of a group, of which a sequence has fewer or more."""
    for shared in (1, 37, 100, 700):
        p = Problem([shared + n + 40 * i for i, n in enumerate(new)], new, 2, group, d, 16, "q8", "bf16", seed=d + shared)
        more.share(p, [0, len(new)], [shared])
        check(p, shared_out(pkg, dev, p, shared), more.window_and_sinks(True, 0, 0))
    p = Problem([6000 + n for n in (3, 700, 2100)], [2, 1, 3], 2, 8, d, 64, "q8", "bf16", seed=5)
    more.share(p, [0, 3], [5990])
    check(p, shared_out(pkg, dev, p, 5990), more.window_and_sinks(True, 0, 0))


@pytest.mark.parametrize("cache,q_type", [("f16", None), ("bf16", None), ("q8", "f16"), ("q8", "bf16")])
@pytest.mark.parametrize("new", [1, 9, 70])
def test_hidden_and_infinite_keys_without_a_log_sum_exp(pkg, dev, new, cache, q_type):
    """NaN and infinities where no row sees them: not a bit changes.  A first or shared token's value that is not finite
    reaches the rows that see it, in its channels alone."""
    bad = [float("nan"), float("inf"), float("-inf")]
    for shared in (0, 50):
        p = Problem([new + 137, new + 95], [new] * 2, 2, 4, 128, 16, cache, q_type, seed=new)
        if shared:
            more.share(p, [0, 2], [shared])
        run = lambda: shared_out(pkg, dev, p, shared) if shared else sinks_out(pkg, dev, p, 20, 5)  # noqa: E731,B023
        clean = run()
        check(p, clean, more.window_and_sinks(True, 0 if shared else 20, 5))

        def spoil(page, off, i):
            for x, s in ((p.k, p.ks), (p.v, p.vs)):  # noqa: B023
                if s is None:
                    x[page, :, off] = bad[i % 3]
                else:
                    x[page, :, off], s[page, :, off] = 127, bad[i % 3]

        for page in set(range(p.k.shape[0])) - set(p.table[p.table >= 0].tolist()):
            for off in range(16):
                spoil(page, off, off)
        for s, n in enumerate(p.kv):
            for j in [*([] if shared else range(5, n - new + 1 - 20)), *range(n, -(-n // 16) * 16)]:
                spoil(int(p.table[s, j // 16]), j % 16, j)
        assert torch.equal(run(), clean)
        page, hit = int(p.table[0, 0]), torch.zeros_like(clean, dtype=torch.bool)
        rows = slice(None) if shared else slice(0, new)  # the prefix is everyone's
        if cache == "q8":
            p.v[page, 1, 3, 32:64], p.vs[page, 1, 3, 1] = 127, float("inf")
            hit[rows, 4:, 32:64] = True
        else:
            p.v[page, 1, 3, 37] = float("inf")
            hit[rows, 4:, 37] = True
        got = run()
        assert bool((got[hit] == float("inf")).all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_bounds_of_the_longest_lengths(pkg, dev, new, cache):
    """Callers that know no better bound than the largest number."""
    p = more.share(Problem([new + 460, new + 475], [new] * 2, 2, 4, 128, 16, cache), [0, 2], [400])
    q, c, table, starts, kv_len = p.on(pkg, dev)
    n, most = torch.tensor([400], dtype=torch.int32, device=dev), 2**31 - 1
    for path in (pkg.SHARED_ONCE, pkg.SHARED_EACH):
        out, lse = pkg.shared_attention(q, c, table, starts, kv_len, n, new, most, most, lse=True, scale=p.scale, path=path)
        more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(True, 0, 0))
    out, lse = pkg.paged_attention(q, c, table, starts, kv_len, new, most, window=most - 1, sinks=5, lse=True, scale=p.scale)
    more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(True, 0, 0))
