"""Attention with first tokens beside a window, and of batches that share prefixes, on the GPU against 64 bits: at the
lengths, windows, pages and groups where it can go wrong.  Tolerances: attention_more_reference.compare."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_more_reference as more  # noqa: E402
from test_gpu_attention import CACHES, Problem, vars_of  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


def sinks_run(pkg, dev, p, window, sinks, causal=True, **kw):
    q, c, table, starts, kv_len = p.on(pkg, dev)
    return pkg.paged_attention(q, c, table, starts, kv_len, max(p.new), max(p.kv + [1]), causal=causal, window=window,
                               lse=True, scale=p.scale, sinks=sinks, **kw)


def sinks_check(pkg, dev, p, window, sinks, causal=True):
    print(f"[sinks] {vars_of(p)} causal={causal} window={window} sinks={sinks}", flush=True)
    out, lse = sinks_run(pkg, dev, p, window, sinks, causal)
    torch.cuda.synchronize()
    more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(causal, window, sinks))
    return out, lse


def shared_run(pkg, dev, p, firsts, lens, causal=True, most_own=None, most_shared=None, most_group=None, path=1, **kw):
    q, c, table, starts, kv_len = p.on(pkg, dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    groups = firsts if firsts is not None else [0, len(p.kv)]
    own = list(p.kv)
    for g, n in enumerate(lens):
        for i in range(groups[g], groups[g + 1]):
            own[i] -= n
    return pkg.shared_attention(q, c, table, starts, kv_len, i32(lens), max(p.new), max(own + [1]) if most_own is None else
                                most_own, max(list(lens) + [1]) if most_shared is None else most_shared,
                                groups=None if firsts is None else i32(firsts), most_group=most_group, causal=causal,
                                lse=True, scale=p.scale, path=path, **kw)


def shared_check(pkg, dev, p, firsts, lens, causal=True, **kw):
    print(f"[shared] {vars_of(p)} causal={causal} groups={firsts} lens={lens}", flush=True)
    more.share(p, firsts if firsts is not None else [0, len(p.kv)], lens)
    out, lse = shared_run(pkg, dev, p, firsts, lens, causal, **kw)
    torch.cuda.synchronize()
    more.compare(p, out.cpu(), lse.cpu(), more.window_and_sinks(causal, 0, 0))
    return out, lse


# ------------------------------------------------------------------ first tokens beside a window
@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group,window,sinks", [(1, 1, 20, 4), (2, 8, 33, 33), (3, 5, 64, 1), (1, 20, 1, 70)])
def test_single_tokens(pkg, dev, cache, q_type, d, heads, group, window, sinks):
    """Lengths below the first tokens, between them and the window, and far behind."""
    kv = [1, 2, 4, 5, 16, 24, 25, 33, 66, 67, 130, 700]
    sinks_check(pkg, dev, Problem(kv, [1] * 12, heads, group, d, 16, cache, q_type, seed=d + group), window, sinks)


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group,window,sinks", [([2, 1, 5], 8, 16, 4), ([16, 3, 9], 4, 5, 40), ([13, 16, 2], 16, 100, 7)])
def test_a_few_tokens(pkg, dev, cache, q_type, d, new, group, window, sinks):
    sinks_check(pkg, dev, Problem([40, 300, 77], new, 2, group, d, 32, cache, q_type, seed=d + group), window, sinks)


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group,window,sinks", [([70, 1, 131, 64], 2, 17, 4), ([33, 40, 17, 100], 8, 64, 64),
                                                    ([129, 64, 65, 63], 1, 1, 65), ([40, 50, 31, 23], 3, 130, 3)])
def test_prompts(pkg, dev, cache, q_type, d, new, group, window, sinks):
    kv = [new[0], new[1] + 250, new[2], new[3] + 129]
    sinks_check(pkg, dev, Problem(kv, new, 1, group, d, 16, cache, q_type, seed=d + group), window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 300), (15, 16), (17, 31), (64, 128), (100, 5), (10000, 4), (0, 4)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [1, 3, 75])
def test_windows_and_first_tokens(pkg, dev, window, sinks, causal, new):
    for cache in ("bf16", "q8"):
        p = Problem([new + 290, new, new + 31], [new] * 3, 2, 4, 128, 16, cache, seed=window + sinks)
        sinks_check(pkg, dev, p, window, sinks, causal)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("cache,q_type", CACHES)
def test_many_splits(pkg, dev, new, cache, q_type):
    """Windows over several workgroups, of which one has the first tokens too; sequences shorter than the window."""
    p = Problem([9000, 5, 2600, 1030], [new, min(new, 5), new, new], 2, 8, 128, 64, cache, q_type, seed=3)
    sinks_check(pkg, dev, p, 2500, 40)


@pytest.mark.parametrize("new", [3, 100])
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_rows_that_see_nothing(pkg, dev, new, cache):
    """More new tokens than cached ones, and empty sequences; pages of first tokens that are not in the cache."""
    sinks_check(pkg, dev, Problem([new - 1, 0, 1, new], [new, new, new, 1], 2, 4, 128, 16, cache), 2, 4)
    p = Problem([new + 100, new + 20], [new] * 2, 2, 4, 128, 16, cache)
    p.table[0, 0], p.table[1, 1] = -1, 1 << 30
    sinks_check(pkg, dev, p, 10, 20)


@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("cache,q_type", CACHES)
def test_hidden_keys_and_values_do_not_matter(pkg, dev, new, cache, q_type):
    """NaN, infinities between the first tokens and the window, past the end and in pages of nobody: not a bit changes.  A
    first token's value that is not finite reaches the rows that see it, in its channel alone."""
    p = Problem([new + 137, new + 95], [new] * 2, 2, 4, 128, 16, cache, q_type, seed=new)
    clean, lse = sinks_check(pkg, dev, p, 20, 5)
    bad = [math.nan, math.inf, -math.inf]

    def spoil(page, off, i):
        for x, s in ((p.k, p.ks), (p.v, p.vs)):
            if s is None:
                x[page, :, off] = bad[i % 3]
            else:
                x[page, :, off] = 127
                s[page, :, off] = bad[i % 3]

    for page in set(range(p.k.shape[0])) - set(p.table[p.table >= 0].tolist()):
        for off in range(16):
            spoil(page, off, off)
    for s, n in enumerate(p.kv):
        for j in [*range(5, n - new + 1 - 20), *range(n, -(-n // 16) * 16)]:
            spoil(int(p.table[s, j // 16]), j % 16, j)
    again, lse2 = sinks_run(pkg, dev, p, 20, 5)
    assert torch.equal(clean, again) and torch.equal(lse, lse2)
    if cache == "q8":
        return
    p.v[int(p.table[0, 0]), 1, 3, 37] = math.inf
    got, _ = sinks_run(pkg, dev, p, 20, 5)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:new, 4:, 37] = True
    assert bool((got[hit] == math.inf).all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("new", [1, 60])
def test_without_effect_first_tokens_are_the_plain_call(pkg, dev, new):
    p = Problem([new + 900, new], [new] * 2, 2, 4, 128, 16, "f16")
    for window in (0, new + 900, 2**40):
        want, got = p.run(pkg, dev, True, window), sinks_run(pkg, dev, p, window, 7)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), window
    for sinks in (new + 900, 2**31, 2**62):  # every key: as without a window
        more.compare(p, *(x.cpu() for x in sinks_run(pkg, dev, p, 5, sinks)), more.window_and_sinks(True, 0, 0))
    with pytest.raises(pkg.Iq4xsError):
        sinks_run(pkg, dev, p, 5, -1)


# ------------------------------------------------------------------ shared prefixes
@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 8), (1, 20)])
def test_shared_single_tokens(pkg, dev, cache, q_type, d, heads, group):
    """The next token of each sequence, behind prefixes that end with a page and inside one."""
    for shared in (1, 16, 37, 200):
        kv = [shared + n for n in (1, 2, 17, 64, 130, 300)]
        shared_check(pkg, dev, Problem(kv, [1] * 6, heads, group, d, 16, cache, q_type, seed=d + shared), None, [shared])


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("new,group", [([2, 1, 5, 3], 8), ([70, 1, 131, 64], 2), ([33, 40, 17, 100], 5)])
def test_shared_prompts(pkg, dev, cache, q_type, new, group):
    for d, shared in ((64, 100), (128, 64), (256, 33)):
        kv = [shared + new[0], shared + new[1] + 50, shared + new[2], shared + new[3] + 129]
        shared_check(pkg, dev, Problem(kv, new, 2, group, d, 32, cache, q_type, seed=d), None, [shared])


@pytest.mark.parametrize("firsts,lens", [([0, 2, 5], [90, 31]), ([1, 3], [64]), ([0, 0, 3, 5], [7, 100, 0]),
                                         ([0, 1, 2, 3, 4, 5], [5, 16, 40, 0, 1])])
@pytest.mark.parametrize("new", [[1] * 5, [3, 0, 2, 40, 1]])
@pytest.mark.parametrize("causal", [True, False])
def test_groups(pkg, dev, firsts, lens, new, causal):
    """Sequences of no group, groups of one and of none, and sequences without new tokens."""
    for cache in ("f16", "q8"):
        p = Problem([n + 101 + 30 * i for i, n in enumerate(new)], new, 2, 4, 128, 16, cache, seed=len(lens))
        shared_check(pkg, dev, p, firsts, lens, causal)


@pytest.mark.parametrize("cache,q_type", CACHES)
def test_long_prefixes(pkg, dev, cache, q_type):
    """Many splits of both launches, and enough rows for the second way of joining."""
    p = Problem([6000 + n for n in (3, 700, 2100)], [2, 1, 3], 2, 8, 128, 64, cache, q_type, seed=5)
    shared_check(pkg, dev, p, None, [5990])
    p = Problem([1200, 1100, 1090], [400, 380, 300], 1, 16, 64, 64, cache, q_type, seed=6)
    shared_check(pkg, dev, p, None, [700])


def test_lengths_that_differ_from_what_the_call_was_told(pkg, dev):
    """More shared tokens than most_shared: a sequence's own part goes on where they end.  Rows past most_group are not
    written; sequences past most_q have their first rows computed."""
    p = more.share(Problem([300, 310, 290], [2, 3, 2], 2, 4, 128, 16, "f16"), [0, 3], [250])
    sees = more.window_and_sinks(True, 0, 0)
    out, lse = shared_run(pkg, dev, p, None, [250], most_shared=100, most_own=250)
    more.compare(p, out.cpu(), lse.cpu(), sees)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    want, want_lse = out.clone(), lse.clone()
    out, lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    one = torch.tensor([250], dtype=torch.int32, device=dev)
    for most_q, most_rows, written in ((3, 4, [0, 1, 2, 3]), (2, 7, [0, 1, 2, 3, 5, 6]), (2, 4, [0, 1, 2, 3])):
        out.fill_(7.0)
        lse.fill_(7.0)
        args = pkg._ATTENTION.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr(), c._address, table.data_ptr(),
                                   starts.data_ptr(), kv_len.data_ptr(), 8 * 128, table.shape[1], 3, 7, most_q, 60, 0, 8,
                                   pkg.TYPE_F16, pkg.TYPE_F16, 1, p.scale)
        prefix = pkg._SHARED.pack(0, one.data_ptr(), 1, 250, most_rows, pkg.SHARED_ONCE) + bytes(4)
        ws = torch.empty(pkg.lib().iq4xs_shared_attention_workspace_bytes(args, prefix), dtype=torch.uint8, device=dev)
        pkg.lib().check("iq4xs_shared_attention", args, prefix, ws.data_ptr(), ws.numel(),
                        torch.cuda.current_stream().cuda_stream)
        left = [i for i in range(7) if i not in written]
        assert bool((out[left] == 7).all()) and bool((lse[left] == 7).all()), (most_q, most_rows)
        # the same sums split otherwise: half a step of fp16 weights and outputs each, of values below 6
        assert bool(((out[written] - want[written]).abs() <= 2 * 2 * 2.0 ** -11 * 6).all())
        assert bool(((lse[written] - want_lse[written]).abs() <= 2.0 ** -14).all())


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("cache,q_type", CACHES)
def test_what_shared_calls_do_not_see_does_not_matter(pkg, dev, new, cache, q_type):
    """Past every sequence's end and in pages of nobody."""
    p = more.share(Problem([new + 60, new + 75, new + 51], [new] * 3, 2, 4, 128, 16, cache, q_type), [0, 3], [50])
    for path in (pkg.SHARED_ONCE, pkg.SHARED_EACH):
        clean, lse = shared_run(pkg, dev, p, None, [50], path=path)
        more.compare(p, clean.cpu(), lse.cpu(), more.window_and_sinks(True, 0, 0))
        kept = [None if t is None else t.clone() for t in (p.k, p.v, p.ks, p.vs)]
        mine = {(int(p.table[s, j // 16]), j % 16) for s, n in enumerate(p.kv) for j in range(n)}
        for page in range(p.k.shape[0]):
            for off in range(16):
                if (page, off) in mine:
                    continue
                for x, s in ((p.k, p.ks), (p.v, p.vs)):
                    if s is None:
                        x[page, :, off] = math.nan if off % 2 else math.inf
                    else:
                        x[page, :, off], s[page, :, off] = 127, math.nan if off % 2 else math.inf
        again, lse2 = shared_run(pkg, dev, p, None, [50], path=path)
        assert torch.equal(clean, again) and torch.equal(lse, lse2)
        p.k, p.v, p.ks, p.vs = kept


@pytest.mark.parametrize("new", [1, 30])
def test_each_sequence_by_itself_is_the_plain_call(pkg, dev, new):
    p = more.share(Problem([new + 400, new + 275, new + 351], [new] * 3, 2, 4, 128, 16, "f16"), [0, 3], [250])
    want = p.run(pkg, dev)
    for path in (pkg.SHARED_AUTO, pkg.SHARED_EACH):
        got = shared_run(pkg, dev, p, None, [250], path=path, most_own=max(p.kv) - 250, most_shared=250)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new", [1, 50])
def test_a_value_of_the_prefix_that_is_not_finite(pkg, dev, new):
    p = more.share(Problem([new + 60, new + 75], [new] * 2, 2, 4, 128, 16, "f16"), [0, 2], [48])
    clean, _ = shared_run(pkg, dev, p, None, [48])
    p.v[int(p.table[0, 1]), 1, 3, 37] = -math.inf
    got, _ = shared_run(pkg, dev, p, None, [48])
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:, 4:, 37] = True
    assert bool((got[hit] == -math.inf).all()) and torch.equal(got[~hit], clean[~hit])


def test_graphs_streams_and_repeats(pkg, dev):
    """Both calls, captured on a side stream and replayed with other lengths and inputs in place; repeats give the same
    bits."""
    p = more.share(Problem([300, 341, 500], [1] * 3, 2, 8, 128, 16, "f16"), [0, 3], [280])
    q, cache, table, starts, kv_len = p.on(pkg, dev)
    shared = torch.tensor([280], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(4)

    def step():
        a = pkg.paged_attention(q, cache, table, starts, kv_len, 1, 500, window=100, sinks=4, lse=True)
        b = pkg.shared_attention(q, cache, table, starts, kv_len, shared, 1, 220, 280, lse=True, path=pkg.SHARED_ONCE)
        return [*a, *b]

    first = step()
    for x, y in zip(first, step()):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, y in zip(first, step()):
            assert torch.equal(x, y)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
        for rep in range(4):
            q.copy_(torch.randn(q.shape, device=dev, generator=g))
            kv_len.copy_(torch.tensor([281 + rep, 300 + 7 * rep, 500 - 50 * rep], dtype=torch.int32))
            for t in outs:
                t.fill_(float("nan"))
            graph.replay()
            side.synchronize()
            kept = [t.clone() for t in outs]
            for a, e in zip(kept, step()):
                assert torch.equal(a, e), rep
    torch.cuda.current_stream().wait_stream(side)


def test_refused_tensors(pkg, dev):
    p = Problem([20, 20], [1, 1], 2, 4, 128, 16, "f16")
    q, c, table, starts, kv_len = p.on(pkg, dev)
    n = torch.tensor([16], dtype=torch.int32, device=dev)
    run = lambda n=n, **kw: pkg.shared_attention(q, c, table, starts, kv_len, n, 1, 4, 16, **kw)  # noqa: E731
    run()
    run(groups=torch.tensor([0, 2], dtype=torch.int32, device=dev))
    for bad in (dict(n=n.long()), dict(n=n.cpu()), dict(n=torch.cat([n, n])), dict(groups=n.new_tensor([0, 1, 2])),
                dict(groups=torch.tensor([0, 2])), dict(groups=torch.tensor([0, 2], device=dev))):
        with pytest.raises(ValueError):
            run(**bad)
    for bad in (dict(most_group=0), dict(scale=math.nan), dict(path=7)):
        with pytest.raises(pkg.Iq4xsError):
            run(**bad)
