"""8-bit values that fp16 does not hold: a finite scale times a code above 65504.  They are infinities in attention, of
the rows and channels that see them and of nothing else."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_attention import Problem, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [3, 8, 15, 70])
@pytest.mark.parametrize("late", [True, False])
@pytest.mark.parametrize("scale,code", [(900, 127), (516, 127), (900, -127), (3e4, 3), (65504, -2)])
def test_codes_past_fp16_stay_in_their_rows_and_channels(pkg, dev, scale, code, late, new, d):  # noqa: F811
    """A key that the first new token does not see (late), and one that all see.  With and without log-sum-exp, as which
    an 8-bit cache takes other kernels."""
    print(f"[past fp16] {scale} {code} {late} {new} {d}", flush=True)
    p = Problem([new + 300], [new], 2, 4, d, 16, "q8", "bf16", seed=new)
    j = 301 if late else 77
    page, off = int(p.table[0, j // 16]), j % 16
    p.v[page, 1, off, 32:64] = 0
    p.v[page, 1, off, 40] = 1
    p.vs[page, 1, off, 1] = scale

    def run():
        q, c, table, starts, kv_len = p.on(pkg, dev)
        for out_type, lse in ((torch.float32, True), (torch.bfloat16, False)):
            got = pkg.paged_attention(q, c, table, starts, kv_len, new, new + 300, lse=lse, out_type=out_type)
            yield (got[0].cpu(), got[1].cpu()) if lse else (got.cpu(), torch.zeros(1))

    clean = list(run())
    p.v[page, 1, off, 37] = code
    first = 1 if late else 0
    for (out, lse), (got, lse2) in zip(clean, run()):
        assert bool(torch.isfinite(out).all()) and torch.equal(lse, lse2)
        assert bool((got[first:, 4:, 37] == math.copysign(math.inf, code)).all())
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[first:, 4:, 37] = False
        assert torch.equal(got[keep], out[keep])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_the_largest_values_that_fp16_holds_come_back_finite(pkg, dev, d, kind):  # noqa: F811
    """Appended, read back in fp16 and attended to.  Half a code's step (515.5 / 2), the last code standing for up to 51
    less than 65520, and half of fp16's own step there (16); past fp16 what comes back is an infinity in fp16 and 127 * 516
    in fp32."""
    held = [65504.0, -65504.0, 65500.0, 65501.0, 65490.0, 65519.0, 40000.0]
    past = [65536.0, 1e5, -1e30, math.inf]
    values = torch.tensor(held + past)
    n = len(values)
    g = torch.Generator().manual_seed(d)
    x = (torch.randn(n, 1, d, generator=g) * 3e4).clamp(-6e4, 6e4)
    x[:, 0, 37] = values
    x = x.to(kind)
    if kind == torch.bfloat16:
        held = held[6:]  # the others round to 65536
    count = len(held)
    first = n - len(past) - count
    cache = pkg.KVCache(*(torch.zeros(1, 1, 16, w, dtype=t, device=dev)
                          for w, t in ((d, torch.int8), (d, torch.int8), (d // 32, torch.float16), (d // 32, torch.float16))))
    at = torch.arange(n, device=dev)
    q = torch.randn(n, 4, d, generator=g).to(kind).to(dev)
    pkg.qk_norm_rope_append(q, torch.zeros_like(x).to(dev), x.to(dev), at.int(), at, cache, out_type=torch.float16)
    table, starts = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([0, n], dtype=torch.int32, device=dev)
    _, v16 = pkg.kv_gather(cache, table, starts, n, out_type=torch.float16)
    _, v32 = pkg.kv_gather(cache, table, starts, n, out_type=torch.float32)
    v16, v32 = v16.cpu(), v32.cpu()
    rows = slice(first, first + count)
    assert bool(torch.isfinite(v16[rows]).all())
    err = (v16[rows].double() - x[rows].double()).abs()
    assert bool((err <= 515.5 / 2 + 51 + 16).all()), err.max().item()
    over = x[first + count:, 0, 37].double()
    assert bool((v16[first + count:, 0, 37] == over.sign() * math.inf).all())
    assert bool((v32[first + count:, 0, 37].double() == over.sign() * 127 * 516).all())
    # a row that sees only values that fp16 holds, as a single token and among many
    for new in (1, 20):
        one = lambda *i: torch.tensor(i, dtype=torch.int32, device=dev)  # noqa: E731
        out = pkg.paged_attention(q[:1].half().expand(new, -1, -1).contiguous(), cache, table, one(0, new),
                                  one(first + count), new, n, causal=False, window=0, out_type=torch.float32)
        if first == 0:  # keys of zero: equal weights
            want = v16[rows].double().mean(0)
            # values in fp16, half a step of 32 at the most, and their mean once more
            assert bool(((out.cpu().double() - want).abs() <= 32).all())
