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
