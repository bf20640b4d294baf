"""Paged attention on the GPU against the row-by-row form in 64 bits, at the sizes, masks and pages where it can go wrong.

Tolerance of an output, derived: weights are rounded to 16 bits for their product with the values (half a step u of
bf16 or fp16 each, relative to sum w |v| / sum w =: size), values of an 8-bit cache to fp16 as well; a score is a sum of
head terms in fp32, off by at most (head + 8) 2^-24 of the sum of the terms' magnitudes, which moves a weight and the
sum of weights by as much; fp16 weights below its normal range are off by 2^-25 of the largest weight each; hardware exp2
and log2 add 2^-20; and the output is rounded once."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


class Problem:
    """Pages in random order, sequences of the given cached and new tokens, on the CPU."""

    def __init__(self, kv, new, heads, group, d, page, cache="f16", q_type=None, seed=1, extra=2, scale=None):
        g = torch.Generator().manual_seed(seed)
        self.q_type = TYPES[q_type or ("f16" if cache == "q8" else cache)]
        self.kv, self.new, self.cache = list(kv), list(new), cache
        per = [-(-n // page) for n in kv]
        count = sum(per) + extra
        pool = torch.randn(2, count, heads, page, d, generator=g)
        if cache == "q8":
            (self.k, self.ks), (self.v, self.vs) = ref.codes(pool[0]), ref.codes(pool[1])
        else:
            self.k, self.v, self.ks, self.vs = pool[0].to(TYPES[cache]), pool[1].to(TYPES[cache]), None, None
        order = torch.randperm(count, generator=g).to(torch.int32)
        self.table = torch.full((len(kv), max(per + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32)
        self.q = (1.7 * torch.randn(sum(new), heads * group, d, generator=g)).to(self.q_type)
        self.scale = d ** -0.5 if scale is None else scale

    def on(self, pkg, dev):
        up = lambda t: None if t is None else t.to(dev)  # noqa: E731
        c = pkg.KVCache(up(self.k), up(self.v), up(self.ks), up(self.vs))
        return up(self.q), c, up(self.table), up(self.starts), up(self.kv_len)

    def run(self, pkg, dev, causal=True, window=0, **kw):
        q, c, table, starts, kv_len = self.on(pkg, dev)
        return pkg.paged_attention(q, c, table, starts, kv_len, max(self.new), max(self.kv + [1]), causal=causal,
                                   window=window, lse=True, scale=self.scale, **kw)

    def check(self, pkg, dev, causal=True, window=0, out_type=None):
        print(f"[attention] {vars_of(self)} causal={causal} window={window}", flush=True)
        got, lse = self.run(pkg, dev, causal, window, out_type=out_type)
        torch.cuda.synchronize()
        self.compare(got.cpu(), lse.cpu(), causal, window)
        return got

    def compare(self, got, lse, causal, window):
        want, want_lse, size, terms = ref.attention(self.q, self.k, self.v, self.ks, self.vs, self.table, self.starts,
                                                    self.kv_len, causal, window, self.scale)
        d = self.q.shape[-1]
        u = 2.0 ** -8 if self.q_type == torch.bfloat16 and self.cache != "q8" else 2.0 ** -11
        score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20
        values = u + (2.0 ** -11 + 127 * 2.0 ** -25 if self.cache == "q8" else 0)
        # fp16 keys of an 8-bit cache that are rounded (prompts): half a step in every term of a score
        if self.cache == "q8":
            score = score + 2.0 ** -11 * terms
        tail = max(self.kv + [1]) * 2.0 ** -25 * ref.stored(self.v, self.vs).abs().nan_to_num(posinf=0).max()
        tol = size * (values + 2 * score[..., None]) + tail + torch.finfo(got.dtype).eps / 2 * want.abs()
        if got.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        err = (got.double() - want).abs()
        assert bool(torch.isfinite(got).all())
        assert bool((err <= tol).all()), ((err - tol).max().item(), (err / tol).max().item())
        none = want_lse == -math.inf
        assert bool((lse[none] == -math.inf).all()) and bool((got[none] == 0).all())
        e = (lse.double() - want_lse)[~none].abs()
        assert bool((e <= score[~none] + 2.0 ** -22 * want_lse[~none].abs()).all()), e.max().item()


def vars_of(p):
    return dict(kv=p.kv[:6], new=p.new[:6], q=tuple(p.q.shape), pages=tuple(p.k.shape), cache=p.cache, q_type=p.q_type)


CACHES = [("f16", None), ("bf16", None), ("q8", "f16"), ("q8", "bf16")]


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 8), (3, 5), (1, 16), (1, 20)])
def test_single_tokens(pkg, dev, cache, q_type, d, heads, group):
    """Decoding: lengths of one, around a tile's and a page's end, and long enough to be split."""
    Problem([1, 2, 15, 16, 17, 31, 33, 64, 65, 130, 700], [1] * 11, heads, group, d, 16, cache, q_type,
            seed=d + group).check(pkg, dev)


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group", [([2, 1, 5], 8), ([16, 3, 9], 4), ([7, 7, 1], 1), ([13, 16, 2], 16)])
def test_a_few_tokens(pkg, dev, cache, q_type, d, new, group):
    """Drafts being verified: every row has its own last key."""
    Problem([40, 300, 77], new, 2, group, d, 32, cache, q_type, seed=d + group).check(pkg, dev)


@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group", [([70, 1, 131, 64], 2), ([33, 40, 17, 100], 8), ([129, 64, 65, 63], 1),
                                       ([40, 50, 31, 23], 3)])
def test_prompts(pkg, dev, cache, q_type, d, new, group):
    """Whole prompts of different lengths, some behind earlier tokens."""
    kv = [new[0], new[1] + 50, new[2], new[3] + 129]
    Problem(kv, new, 1, group, d, 16, cache, q_type, seed=d + group).check(pkg, dev)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_page_sizes(pkg, dev, page, new):
    Problem([new, new + 100, new + 301], [new] * 3, 2, 4, 128, page, "f16", seed=page).check(pkg, dev)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 100, 10000])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [1, 3, 75])
def test_windows(pkg, dev, window, causal, new):
    for cache in ("bf16", "q8"):
        Problem([new + 290, new, new + 31], [new] * 3, 2, 4, 128, 16, cache, seed=window).check(pkg, dev, causal, window)


@pytest.mark.parametrize("new", [1, 5, 80])
def test_every_key(pkg, dev, new):
    Problem([new + 200, new], [new] * 2, 2, 8, 64, 16, "f16").check(pkg, dev, causal=False)


@pytest.mark.parametrize("new", [3, 100])
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_rows_that_see_nothing(pkg, dev, new, cache):
    """More new tokens than cached ones, empty sequences, and windows that lie before every key."""
    Problem([new - 1, 0, 1, new], [new, new, new, 1], 2, 4, 128, 16, cache).check(pkg, dev)
    Problem([2, 0, 1], [new] * 3, 1, 1, 64, 16, cache).check(pkg, dev, window=1)


@pytest.mark.parametrize("new", [1, 4, 100])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_output_types(pkg, dev, new, out_type):
    for cache, q_type in CACHES:
        got = Problem([new + 77], [new], 2, 4, 128, 16, cache, q_type).check(pkg, dev, out_type=TYPES[out_type])
        assert got.dtype == TYPES[out_type]


@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("cache,q_type", CACHES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_hidden_keys_and_values_do_not_matter(pkg, dev, new, cache, q_type, d):
    """NaN, infinities and the type's limits past a sequence's end, in pages of nobody, and (causal, window) in tokens
    that the other rows may see: every row is what the keys it sees make it, bit for bit."""
    p = Problem([new + 37, new + 5], [new] * 2, 2, 4, d, 16, cache, q_type, seed=new)
    clean, lse = p.run(pkg, dev, True, 20)
    p.compare(clean.cpu(), lse.cpu(), True, 20)
    bad = [math.nan, math.inf, -math.inf]

    def spoil(page, off, i):
        for x, s in ((p.k, p.ks), (p.v, p.vs)):
            if s is None:
                x[page, :, off] = bad[i % 3]
            else:
                x[page, :, off] = 127
                s[page, :, off] = bad[i % 3]

    used = set(p.table[p.table >= 0].tolist())
    for page in set(range(p.k.shape[0])) - used:
        for off in range(16):
            spoil(page, off, off)
    for s, n in enumerate(p.kv):
        for j in range(n, -(-n // 16) * 16):
            spoil(int(p.table[s, j // 16]), j % 16, j)
        for j in range(max(0, n - new + 1 - 20)):  # before every row's window
            spoil(int(p.table[s, j // 16]), j % 16, j)
    again, lse2 = p.run(pkg, dev, True, 20)
    assert torch.equal(clean, again) and torch.equal(lse, lse2)
    if new < 3:
        return
    # one token of NaN that the rows before it do not see, and those 20 and more after it no longer
    for s, n in enumerate(p.kv):
        j = n - new + 1
        spoil(int(p.table[s, j // 16]), j % 16, 0)
    last, lse3 = p.run(pkg, dev, True, 20)
    last, clean, lse3, lse = last.cpu(), clean.cpu(), lse3.cpu(), lse.cpu()
    for s in range(2):
        for i in range(new):
            row = s * new + i
            if 1 <= i < 21:
                assert bool(torch.isnan(last[row]).all()), (s, i)
                assert bool(torch.isnan(lse3[row]).all()), (s, i)
            else:
                assert torch.equal(last[row], clean[row]) and torch.equal(lse3[row], lse[row]), (s, i)


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
def test_a_value_that_is_not_finite_stays_in_its_rows_and_channels(pkg, dev, new, value, cache):
    """One channel of one token's value: rows that see it have it there, nothing else changes (channels of its scale's
    group with an 8-bit cache)."""
    p = Problem([new + 37], [new], 2, 4, 128, 16, cache, seed=new)
    clean, lse = p.run(pkg, dev)
    j = new + 37 - new + 1  # seen from row 1 on
    page, off = int(p.table[0, j // 16]), j % 16
    if cache == "q8":
        p.v[page, 1, off, 32:64] = 5
        p.vs[page, 1, off, 1] = value
    else:
        p.v[page, 1, off, 37] = value
    got, lse2 = p.run(pkg, dev)
    got, clean = got.cpu(), clean.cpu()
    assert torch.equal(lse, lse2)
    hit = slice(32, 64) if cache == "q8" else slice(37, 38)
    part = got[1:, 4:, hit]
    assert bool((torch.isnan(part) if math.isnan(value) else part == value).all())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1:, 4:, hit] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("new", [1, 4, 70])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_pages_outside_the_cache_are_masked(pkg, dev, new, cache):
    p = Problem([new + 100, new + 20], [new] * 2, 2, 4, 128, 16, cache)
    p.table[0, 1], p.table[0, 3], p.table[1, 0] = -1, p.k.shape[0], 1 << 30
    p.check(pkg, dev)


def test_lengths_past_the_table_are_cut(pkg, dev):
    p = Problem([64], [1], 1, 4, 64, 16, "f16")
    want, lse = p.run(pkg, dev, causal=False)
    p.kv_len[0] = 200  # the table holds 64 tokens
    got, lse2 = p.run(pkg, dev, causal=False)
    assert torch.equal(got, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("new", [1, 40])
def test_strided_queries(pkg, dev, new):
    """q as a view of a fused projection's rows."""
    p = Problem([new + 90] * 2, [new] * 2, 2, 4, 128, 16, "bf16")
    want, _ = p.run(pkg, dev)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    wide = torch.full((q.shape[0], 12, 128), math.nan, dtype=q.dtype, device=dev)
    wide[:, :8] = q
    got = pkg.paged_attention(wide[:, :8], c, table, starts, kv_len, new, new + 90)
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [30.0, 1e-3, -0.1, 0.0])
@pytest.mark.parametrize("new", [1, 50])
def test_peaked_and_flat_weights(pkg, dev, scale, new):
    Problem([new + 150], [new], 2, 4, 128, 16, "f16", scale=scale).check(pkg, dev)


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("cache,q_type", CACHES)
def test_rising_scores(pkg, dev, new, cache, q_type):
    """Every tile raises the maximum: keys along the query's direction, longer and longer."""
    p = Problem([new + 400], [new], 1, 2, 64, 16, cache, q_type)
    n, pool = new + 400, torch.zeros(2, p.k.shape[0], 1, 16, 64)
    p.q = torch.ones_like(p.q)
    for j in range(n):
        pool[0, p.table[0, j // 16], 0, j % 16] = j / 40
        pool[1, p.table[0, j // 16], 0, j % 16] = math.sin(j)
    if cache == "q8":
        (p.k, p.ks), (p.v, p.vs) = ref.codes(pool[0]), ref.codes(pool[1])
    else:
        p.k, p.v = pool[0].to(TYPES[cache]), pool[1].to(TYPES[cache])
    p.check(pkg, dev)


@pytest.mark.parametrize("cache,q_type", CACHES)
def test_long_context(pkg, dev, cache, q_type):
    """A context of many splits against the same in 64 bits on the GPU, page by page in order."""
    n, heads, group, d = 40009, 2, 8, 128
    g = torch.Generator(device=dev).manual_seed(9)
    count = -(-n // 64)
    pool = torch.randn(2, count, heads, 64, d, device=dev, generator=g)
    if cache == "q8":
        (k, ks), (v, vs) = ref.codes(pool[0]), ref.codes(pool[1])
    else:
        (k, v), ks, vs = pool.to(TYPES[cache]).unbind(0), None, None
        k, v = k.contiguous(), v.contiguous()
    kind = TYPES[q_type or cache]
    q = (1.7 * torch.randn(3, heads * group, d, device=dev, generator=g)).to(kind)
    table = torch.arange(count, dtype=torch.int32, device=dev)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = pkg.paged_attention(q, pkg.KVCache(k, v, ks, vs), table, i32(0, 3), i32(n), 3, n, lse=True)
    flat = lambda p, s: ref.stored(p, s).transpose(0, 1).reshape(heads, -1, d)[:, :n]  # noqa: E731
    K, V = flat(k, ks), flat(v, vs)
    u = 2.0 ** -8 if kind == torch.bfloat16 else 2.0 ** -11
    for i in range(3):
        for h in range(heads):
            m = n - 2 + i
            z = q[i, h * group:(h + 1) * group].double() @ K[h, :m].t() / math.sqrt(d)
            w = torch.softmax(z, -1)
            o, size = w @ V[h, :m], w @ V[h, :m].abs()
            # 2^-8 or 2^-11 for weights, output and 8-bit values, scores within 2^-11 of their terms' size (about 30 here
            # at most: 1.7 * 128 * 0.64 * 3 / sqrt(128)) where keys are rounded; errors of 40000 terms mostly cancel
            tol = size * (2 * u + 2.0 ** -11 + 2.0 ** -6) + u * o.abs() + n * 2.0 ** -25 / w.amax(-1, True).reciprocal()
            assert bool(((out[i, h * group:(h + 1) * group].double() - o).abs() <= tol).all())
            e = (lse[i, h * group:(h + 1) * group].double() - torch.logsumexp(z, -1)).abs().max().item()
            assert e <= 2.0 ** -11 * 30, e


def test_the_same_call_gives_the_same_bits(pkg, dev):
    for new, kv in ((1, 5000), (60, 900)):
        p = Problem([kv, kv // 3], [new] * 2, 2, 8, 128, 16, "f16")
        first, lse = p.run(pkg, dev)
        for _ in range(3):
            again, lse2 = p.run(pkg, dev)
            assert torch.equal(first, again) and torch.equal(lse, lse2)


def test_pool_past_32_bits(pkg, dev):
    """A cache of 2^32 + elements a tensor: tokens of the last pages are their own."""
    pages, page, heads, d = 4100, 1024, 8, 128  # 4.3e9 elements, 8.6 GB each
    k = torch.zeros(pages, heads, page, d, dtype=torch.float16, device=dev)
    v = torch.zeros_like(k)
    p = Problem([2000], [1], heads, 2, d, 1024, "f16")
    for s, (i, j) in enumerate(((0, pages - 1), (1, pages - 3))):
        k[j], v[j] = p.k[p.table[0, i]].to(dev), p.v[p.table[0, i]].to(dev)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=dev)
    want, lse = p.run(pkg, dev)
    cache = pkg.KVCache(k, v)
    got = pkg.paged_attention(p.q.to(dev), cache, table, p.starts.to(dev), p.kv_len.to(dev), 1, 2000)
    assert torch.equal(got, want)
    rows = pkg.kv_gather(cache, table, torch.tensor([0, 2000], dtype=torch.int32, device=dev), 2000)
    for x, pool in zip(rows, (p.k, p.v)):
        flat = torch.cat([pool[p.table[0, 0]], pool[p.table[0, 1]]], 1).transpose(0, 1)[:2000]
        assert torch.equal(x.cpu(), flat)


def test_graph_replays_and_side_streams(pkg, dev):
    """The three calls of a step, captured once and replayed with other inputs in place, against eager calls."""
    hq, hk, d, b = 16, 2, 128, 3
    p = Problem([300, 41, 500], [1] * b, hk, hq // hk, d, 16, "f16")
    q0, cache, table, starts, kv_len = p.on(pkg, dev)
    g = torch.Generator(device=dev).manual_seed(4)
    new = lambda h: torch.randn(b, h, d, device=dev, generator=g)  # noqa: E731
    q, k, v = new(hq), new(hk), new(hk)
    pos = kv_len - 1
    slots = torch.stack([table[s, (n - 1) // 16].long() * 16 + (n - 1) % 16 for s, n in enumerate(p.kv)])
    f = ref.frequencies(d).to(dev)

    def step():
        x = pkg.qk_norm_rope_append(q, k, v, pos, slots, cache, f, out_type=torch.float16)
        o = pkg.paged_attention(x, cache, table, starts, kv_len, 1, 500, lse=True)
        return [*o, *pkg.kv_gather(cache, table[:1], starts.new_tensor([0, 300]), 300)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        one = starts.new_tensor([0, 300])
        side.synchronize()
        graph = torch.cuda.CUDAGraph()

        def captured():
            x = pkg.qk_norm_rope_append(q, k, v, pos, slots, cache, f, out_type=torch.float16)
            o = pkg.paged_attention(x, cache, table, starts, kv_len, 1, 500, lse=True)
            return [*o, *pkg.kv_gather(cache, table[:1], one, 300)]

        with torch.cuda.graph(graph, stream=side):
            outs = captured()
        for rep in range(4):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device=dev, generator=g))
            for t in outs:
                t.fill_(float("nan"))
            graph.replay()
            side.synchronize()
            kept = [t.clone() for t in outs]
            for a, e in zip(kept, step()):
                assert torch.equal(a, e), rep
    torch.cuda.current_stream().wait_stream(side)


def test_refused_tensors(pkg, dev):
    p = Problem([20], [1], 2, 4, 128, 16, "f16")
    q, c, table, starts, kv_len = p.on(pkg, dev)
    run = lambda q=q, table=table, starts=starts, kv_len=kv_len, c=c, **kw: pkg.paged_attention(  # noqa: E731
        q, c, table, starts, kv_len, 1, 20, **kw)
    run()
    for bad in (dict(q=q.bfloat16()), dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(q=q.cpu()),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(table=table.long()), dict(table=table[0]),
                dict(starts=starts[:1]), dict(starts=starts.long()), dict(kv_len=kv_len.cpu()), dict(kv_len=kv_len.long()),
                dict(out_type=torch.int8)):
        with pytest.raises(ValueError):
            run(**bad)
    with pytest.raises(pkg.Iq4xsError):
        run(window=-1)
    k = c.k_pages
    for bad in ((k, k[:, :1]), (k, k.bfloat16()), (k.int(), k.int()), (k.to(torch.int8), k.to(torch.int8)),
                (k, k, k, k), (k[:, :, :12].contiguous(),) * 2, (k[..., :96].contiguous(),) * 2, (k.cpu(), k.cpu()),
                (k.transpose(1, 2), k.transpose(1, 2)), (k[0], k[0])):
        with pytest.raises(ValueError):
            pkg.KVCache(*bad)
