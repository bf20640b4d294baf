"""What attention does to single keys, to large scales and to infinities of an 8-bit cache.

A row that sees one key has that key's value, as the weight and the sum it is divided by are the same number: the fp32
quotient is within 2^-23 of the stored number (fp16 of code times scale), which rounds back to it."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402
from test_gpu_attention import Problem, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 40, 150])
def test_one_key_is_its_value(pkg, dev, new, d, cache):  # noqa: F811
    print(f"[one key] {new} {d} {cache}", flush=True)
    p = Problem([new + 700, new], [new, new], 2, 4, d, 16, cache, seed=new + d)
    got, _ = p.run(pkg, dev, window=1)
    for s in range(2):
        v, _ = ref.sequence_rows(p.v, p.vs, p.table[s], p.kv[s])
        v = v[p.kv[s] - new:].to(torch.float16 if cache == "q8" else p.v.dtype)
        want = v.repeat_interleave(4, 1)
        assert torch.equal(got[s * new:(s + 1) * new].cpu(), want.to(got.dtype)), s


@pytest.mark.parametrize("q_type", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_large_finite_scales(pkg, dev, new, q_type):  # noqa: F811
    """Scales past 65504 / 127 whose codes keep the values within fp16."""
    p = Problem([new + 300], [new], 2, 4, 128, 16, "q8", q_type, seed=new)
    p.v //= 2  # -64 to 63
    p.vs[int(p.table[0, 3]), :, 5] = 900
    p.check(pkg, dev, out_type=torch.float32)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_infinite_scales_among_keys_that_all_see(pkg, dev, new, d, value):  # noqa: F811
    p = Problem([new + 300], [new], 2, 4, d, 16, "q8", seed=new)
    clean, lse = p.run(pkg, dev)
    page, off = int(p.table[0, 3]), 5
    p.v[page, 1, off, 32:64] = 5
    p.vs[page, 1, off, 1] = value
    got, lse2 = p.run(pkg, dev)
    got, clean = got.cpu(), clean.cpu()
    assert torch.equal(lse, lse2)
    part = got[:, 4:, 32:64]
    assert bool((torch.isnan(part) if math.isnan(value) else part == value).all())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[:, 4:, 32:64] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("d,heads", [(64, 16), (128, 8), (256, 4)])
@pytest.mark.parametrize("kv,new", [([1500, 40, 2100], [130, 40, 120]), ([1400], [300])])
def test_many_rows_in_several_splits(pkg, dev, d, heads, kv, new):  # noqa: F811
    """Enough rows that a wave joins several: equal to the sequences on their own, where fewer are joined another way."""
    print(f"[many rows] {d} {kv} {new}", flush=True)
    p = Problem(kv, new, heads, 8, d, 16, "f16", seed=d)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    for window in (0, 700):
        out, lse = pkg.paged_attention(q, c, table, starts, kv_len, max(new), max(kv), window=window, lse=True)
        for s in range(len(kv)):
            for lo in range(0, new[s], 16):  # rows of 16 tokens at a time, as drafts at the end of what they see
                n = min(16, new[s] - lo)
                first, end = int(starts[s]) + lo, kv[s] - new[s] + lo + n
                one, l1 = pkg.paged_attention(q[first:first + n], c, table[s:s + 1],
                                              torch.tensor([0, n], dtype=torch.int32, device=dev),
                                              torch.tensor([end], dtype=torch.int32, device=dev), n, end, window=window,
                                              lse=True)
                # both are within two half steps of fp16 (weights, output) of the same sum, of values below 6
                assert bool(((one - out[first:first + n]).abs() <= 2 * 2 * 2.0 ** -11 * 6).all()), (s, lo)
                assert bool(((l1 - lse[first:first + n]).abs() <= 2.0 ** -14).all()), (s, lo)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("new", [1, 3, 30])
def test_calls_repeat_bit_for_bit(pkg, dev, new, cache, d):  # noqa: F811
    """Lengths of one step, of several and of several splits, the call again and again: nothing is read unfinished."""
    p = Problem([1, 33, 64, 65, 130, 700, 1500, 9000], [1] * 5 + [new] * 3, 1, 8, d, 16, cache, seed=d)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    first = None
    for _ in range(12):
        got = pkg.paged_attention(q, c, table, starts, kv_len, max(p.new), max(p.kv), lse=True)
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
