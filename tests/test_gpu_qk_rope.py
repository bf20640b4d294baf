"""Norm and rotation of queries and keys, the paged cache they are written to and its read-back, against 64 bits.

Tolerance, derived: the sum of squares of a head in fp32 is off by at most head * 2^-24 relative (half of that reaches
its root), the norm, the gain, the turn's products and sum round six times (2^-24 each, relative to the pair's length),
rsqrt, sine and cosine are within 2^-22; the angle is formed in 64 bits; the result is rounded once to its type."""
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


def rows(t, heads, d, kind, seed, wide=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, heads, d, generator=g) * torch.exp(wide * torch.randn(1, heads, d, generator=g))).to(kind)


def tolerance(x64, want, rot, d, kind, half):
    """Elementwise: fp32 errors are relative to the length of the pair that turns."""
    size = x64.abs().clone()
    a, b = (size[..., :rot // 2], size[..., rot // 2:rot]) if half else (size[..., 0:rot:2], size[..., 1:rot:2])
    both = a + b
    turned = torch.cat([both, both], -1) if half else torch.stack([both, both], -1).flatten(-2)
    size = torch.cat([turned, size[..., rot:]], -1)
    tol = size * (d * 2.0 ** -25 + 6 * 2.0 ** -24 + 3 * 2.0 ** -22) + torch.finfo(kind).eps / 2 * want.abs()
    return tol + (2.0 ** -25 if kind == torch.float16 else 1e-37)


def close(got, want, tol):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()


CASES = [(1, 8, 2, 128, 128), (3, 5, 1, 64, 64), (7, 3, 3, 64, 16), (2, 16, 1, 256, 64), (65, 4, 4, 128, 0),
         (130, 64, 8, 128, 64), (33, 7, 2, 256, 256), (2, 1, 1, 128, 32), (5, 9, 3, 64, 48)]


@pytest.mark.parametrize("t,hq,hk,d,rot", CASES)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("half", [True, False])
def test_dense(pkg, dev, t, hq, hk, d, rot, kind, out, half):
    print(f"[qk] {t} {hq} {hk} {d} {rot} {kind} {out} {half}", flush=True)
    q, k = rows(t, hq, d, TYPES[kind], 1), rows(t, hk, d, TYPES[kind], 2)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 1 << 20, (t,), generator=g, dtype=torch.int32)
    gq, gk = 1 + 0.2 * torch.randn(d, generator=g), None if t == 3 else 1 + 0.2 * torch.randn(d, generator=g)
    f = ref.frequencies(rot) if rot else None
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    got = pkg.qk_norm_rope(up(q), up(k), up(pos), up(f), up(gq), up(gk), rope=pkg.ROPE_HALF if half else
                           pkg.ROPE_INTERLEAVED, out_type=TYPES[out])
    for x, gain, y in ((q, gq, got[0]), (k, gk, got[1])):
        want = ref.norm_rope(x, pos, f, gain, 1e-6, half)
        close(y, want, tolerance(ref.norm_rope(x, pos, None, gain, 1e-6, half), want, rot, d, TYPES[out], half))


@pytest.mark.parametrize("pos", [0, 1, -5, (1 << 31) - 1, -(1 << 31)])
def test_far_positions(pkg, dev, pos):
    q, k = rows(2, 2, 128, torch.float32, 5), rows(2, 1, 128, torch.float32, 6)
    p, f = torch.full((2,), pos, dtype=torch.int32), ref.frequencies(128)
    got = pkg.qk_norm_rope(q.to(dev), k.to(dev), p.to(dev), f.to(dev))
    want = ref.norm_rope(q, p, f, None, 1e-6, True)
    # the angle's own rounding in 64 bits: 2^31 * 2^-52 radians
    tol = tolerance(ref.norm_rope(q, p, None, None, 1e-6, True), want, 128, 128, torch.float32, True)
    close(got[0], want, tol + 2.0 ** -20 * want.abs().max())


def test_strided_rows(pkg, dev):
    """q, k and v as views of one fused projection."""
    x = rows(9, 12, 128, torch.bfloat16, 7).to(dev)
    pos, f = torch.arange(9, dtype=torch.int32, device=dev), ref.frequencies(128).to(dev)
    a = pkg.qk_norm_rope(x[:, :8], x[:, 8:10], pos, f)
    b = pkg.qk_norm_rope(x[:, :8].contiguous(), x[:, 8:10].contiguous(), pos, f)
    assert all(torch.equal(i, j) for i, j in zip(a, b))


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e30, math.inf, math.nan])
def test_extreme_heads_stay_in_their_head(pkg, dev, value):
    q, k = rows(2, 4, 128, torch.float32, 8, 0.0), rows(2, 1, 128, torch.float32, 9, 0.0)
    pos, f = torch.tensor([3, 70], dtype=torch.int32), ref.frequencies(128)
    clean = pkg.qk_norm_rope(q.to(dev), k.to(dev), pos.to(dev), f.to(dev))[0]
    q[1, 2] = value
    got = pkg.qk_norm_rope(q.to(dev), k.to(dev), pos.to(dev), f.to(dev))[0]
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(got[keep.to(dev)], clean[keep.to(dev)])
    if value in (0.0, 1e-30):
        assert bool((got[1, 2].abs() <= value * 2000).all())
    elif math.isfinite(value):  # the squares pass fp32's range: 1 / inf
        assert bool((got[1, 2] == 0).all())
    else:
        assert bool(torch.isnan(got[1, 2]).all())


@pytest.mark.parametrize("cache_type", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("t,hq,hk,d,rot,half", [(1, 8, 2, 128, 128, True), (50, 6, 3, 64, 16, True),
                                                (37, 4, 4, 256, 64, False), (20, 5, 1, 128, 0, True),
                                                (700, 8, 8, 64, 48, False)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_append_and_read_back(pkg, dev, cache_type, t, hq, hk, d, rot, half, kind):
    print(f"[append] {cache_type} {t} {hq} {hk} {d} {rot} {half} {kind}", flush=True)
    page, pages = 16, t // 16 + 3
    g = torch.Generator().manual_seed(t)
    q, k, v = (rows(t, h, d, TYPES[kind], i) for i, h in enumerate((hq, hk, hk)))
    v[0, 0, :32] = 0
    pos = torch.randint(0, 1 << 17, (t,), generator=g, dtype=torch.int32)
    slots = torch.randperm(page * pages, generator=g)[:t].contiguous()
    if t > 5:
        slots[3], slots[4] = -1, page * pages  # not stored
    shape = (pages, hk, page, d)
    if cache_type == "q8":
        pools = [torch.randint(-127, 128, shape, generator=g).to(torch.int8).to(dev) for _ in range(2)]
        pools += [torch.rand((pages, hk, page, d // 32), generator=g).half().to(dev) for _ in range(2)]
    else:
        pools = [torch.randn(shape, generator=g).to(TYPES[cache_type]).to(dev) for _ in range(2)]
    before = [x.cpu().clone() for x in pools]
    cache = pkg.KVCache(*pools)
    f = ref.frequencies(rot).to(dev) if rot else None
    rope = pkg.ROPE_HALF if half else pkg.ROPE_INTERLEAVED
    up = lambda x: x.to(dev)  # noqa: E731
    out = pkg.qk_norm_rope_append(up(q), up(k), up(v), up(pos), up(slots), cache, f, rope=rope, out_type=torch.float16)
    dense = pkg.qk_norm_rope(up(q), up(k), up(pos), f, rope=rope, out_type=torch.float32)
    assert torch.equal(out, pkg.qk_norm_rope(up(q), up(k), up(pos), f, rope=rope, out_type=torch.float16)[0])
    keep = (slots >= 0) & (slots < page * pages)
    at = slots[keep]
    want = [x.clone() for x in before]
    # the cache holds the dense fp32 keys and the values, rounded or as codes of their own
    for i, x in ((0, dense[1].cpu()), (1, v)):
        if cache_type == "q8":
            c, s = ref.codes(x[keep])
            want[i][at // page, :, at % page] = c
            want[i + 2][at // page, :, at % page] = s
        else:
            want[i][at // page, :, at % page] = x[keep].to(TYPES[cache_type])
    for a, b in zip(pools, want):
        assert torch.equal(a.cpu(), b)
    # read back: every page in order as one sequence, in each type
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    starts = torch.tensor([0, pages * page], dtype=torch.int32, device=dev)
    for kind_out in TYPES.values():
        got = pkg.kv_gather(cache, table, starts, pages * page, out_type=kind_out)
        for i, x in enumerate(got):
            full = want[i].float()
            if cache_type == "q8":
                full = full * want[i + 2].float().repeat_interleave(32, -1)
            assert torch.equal(x.cpu(), full.to(kind_out).transpose(1, 2).reshape(-1, hk, d))


def test_codes_of_extreme_groups(pkg, dev):
    """A NaN makes its group's scale NaN, an infinity its largest; zeros and tiny values have no scale."""
    v = torch.ones(5, 1, 64)
    v[0, 0, 3], v[1, 0, 40], v[2, 0, :32], v[3, 0] = math.nan, -math.inf, 0.0, 1e-9
    v[4, 0, 0] = 1e30
    pools = [torch.zeros(1, 1, 16, 64, dtype=torch.int8, device=dev) for _ in range(2)]
    pools += [torch.zeros(1, 1, 16, 2, dtype=torch.float16, device=dev) for _ in range(2)]
    z = torch.arange(5, device=dev)
    pkg.qk_norm_rope_append(v.to(dev), v.to(dev), v.to(dev), z.int(), z, pkg.KVCache(*pools))
    c, s = pools[1][0, 0, :5].cpu(), pools[3][0, 0, :5].cpu()
    want_c, want_s = ref.codes(v[:, 0].nan_to_num(posinf=3e38, neginf=-3e38))
    assert bool(torch.isnan(s[0, 0])) and bool((c[0, :32] == 0).all())
    s[0, 0], want_s[0, 0], c[0, :32], want_c[0, :32] = 0, 0, 0, 0
    assert torch.equal(s, want_s) and torch.equal(c, want_c)


@pytest.mark.parametrize("cache_type", ["bf16", "q8"])
@pytest.mark.parametrize("hk,d", [(1, 64), (3, 128), (8, 256)])
def test_gather_of_ragged_sequences(pkg, dev, cache_type, hk, d):
    """Empty sequences, pages that end inside a sequence, rows outside every sequence, pages not in the cache, and more
    sequences than a wave counts at once."""
    g = torch.Generator().manual_seed(hk)
    lens = [0, 1, 16, 17, 0, 40] + [int(x) for x in torch.randint(0, 9, (150,), generator=g)]
    pages = sum(-(-n // 16) for n in lens) + 1
    pool = torch.randn(2, pages, hk, 16, d, generator=g)
    if cache_type == "q8":
        (k, ks), (v, vs) = ref.codes(pool[0]), ref.codes(pool[1])
    else:
        (k, v), ks, vs = pool.bfloat16().unbind(0), None, None
        k, v = k.contiguous(), v.contiguous()
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), 3), -1, dtype=torch.int32)
    n = 0
    for s, m in enumerate(lens):
        for j in range(-(-m // 16)):
            table[s, j] = order[n]
            n += 1
    table[5, 1] = pages  # not in the cache
    lead, total = 2, sum(lens) + 7
    starts = torch.tensor([lead + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    got = pkg.kv_gather(pkg.KVCache(up(k), up(v), up(ks), up(vs)), up(table), up(starts), total, out_type=torch.float32)
    for x, p, sc in ((got[0], k, ks), (got[1], v, vs)):
        want = torch.zeros(total, hk, d, dtype=torch.float64)
        for s, m in enumerate(lens):
            r, ok = ref.sequence_rows(p, sc, table[s], m)
            want[starts[s]:starts[s] + m] = torch.where(ok[:, None, None], r, torch.zeros_like(r))
        assert torch.equal(x.cpu().double(), want)


def test_no_tokens(pkg, dev):
    z = torch.zeros(0, 4, 128, device=dev)
    q, k = pkg.qk_norm_rope(z, z[:, :1], torch.zeros(0, dtype=torch.int32, device=dev))
    assert q.shape == (0, 4, 128) and k.shape == (0, 1, 128)


def test_refused_tensors(pkg, dev):
    q, k = torch.randn(4, 8, 128, device=dev), torch.randn(4, 2, 128, device=dev)
    pos, f = torch.arange(4, dtype=torch.int32, device=dev), ref.frequencies(128).to(dev)
    pages = torch.zeros(2, 2, 16, 128, dtype=torch.float16, device=dev)
    cache, slots = pkg.KVCache(pages, pages.clone()), torch.arange(4, device=dev)
    pkg.qk_norm_rope(q, k, pos, f)
    pkg.qk_norm_rope_append(q, k, k, pos, slots, cache, f)
    for bad in (dict(q=q.half()), dict(q=q.double(), k=k.double()), dict(k=k[:3]), dict(k=k[..., :64]), dict(pos=pos.long()),
                dict(pos=pos[:3]), dict(freqs=f.float()), dict(freqs=f[:7]), dict(freqs=torch.cat([f, f])),
                dict(q_gamma=torch.ones(64, device=dev)), dict(rope=2), dict(out_type=torch.int8), dict(q=q.cpu()),
                dict(pos=pos.cpu()), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            pkg.qk_norm_rope(**{**dict(q=q, k=k, pos=pos, freqs=f), **bad})
    for bad in (dict(v=k[:3]), dict(v=k.half()), dict(slots=slots.int()), dict(slots=slots[:3]), dict(k=k[:, :1], v=k[:, :1])):
        with pytest.raises(ValueError):
            pkg.qk_norm_rope_append(**{**dict(q=q, k=k, v=k, pos=pos, slots=slots, cache=cache, freqs=f), **bad})
    for bad in (dict(total=-1), dict(out_type=torch.int8), dict(table=pos), dict(starts=pos.long())):
        with pytest.raises(ValueError):
            pkg.kv_gather(**{**dict(cache=cache, table=pos[None], starts=pos[:2], total=4), **bad})
