"""Long 16-bit contexts of many splits, single tokens and many rows, in 64 bits on the GPU.

Tolerance, derived: weights and the sum they are divided by are rounded alike (a half step u each, moving the quotient by
at most 2 u of the weighted mean of |v|), scores and log-sum-exp as sums in fp32 ((head + 8) 2^-24 of the terms, 2^-20 for
exp2 and log2), fp16 weights below its normal range 2^-31 of the largest for each key; outputs in fp32."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_attention import TYPES, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_long_context(pkg, dev, cache, d, new):  # noqa: F811
    print(f"[long] {cache} {d} {new}", flush=True)
    n, heads, group, kind = 20011, 2, 4, TYPES[cache]
    g = torch.Generator(device=dev).manual_seed(d)
    count = -(-n // 64)
    k, v = (torch.randn(count, heads, 64, d, device=dev, generator=g).to(kind) for _ in range(2))
    q = (1.7 * torch.randn(new, heads * group, d, device=dev, generator=g)).to(kind)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(count, dtype=torch.int32, device=dev)[None]
    out, lse = pkg.paged_attention(q, pkg.KVCache(k, v), table, i32(0, new), i32(n), new, n, lse=True,
                                   out_type=torch.float32)
    K, V = (x.double().transpose(0, 1).reshape(heads, -1, d)[:, :n] for x in (k, v))
    u = torch.finfo(kind).eps / 2
    for i in range(new):
        m = n - new + 1 + i
        for h in range(heads):
            x = q[i, h * group:(h + 1) * group].double()
            z = x @ K[h, :m].t() / math.sqrt(d)
            terms = (x.abs() @ K[h, :m].abs().t()).amax(-1) / math.sqrt(d)
            w = torch.softmax(z, -1)
            o, size = w @ V[h, :m], w @ V[h, :m].abs()
            score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20
            tail = n * 2.0 ** -31 * V.abs().max() if cache == "f16" else 0
            tol = size * (2 * u + 2 * score[:, None]) + 2.0 ** -24 * o.abs() + tail
            err = (out[i, h * group:(h + 1) * group].double() - o).abs()
            assert bool((err <= tol).all()), (i, h, (err / tol).max().item())
            want = torch.logsumexp(z, -1)
            e = (lse[i, h * group:(h + 1) * group].double() - want).abs()
            assert bool((e <= score + 2.0 ** -22 * want.abs()).all()), (i, h, e.max().item(), score.max().item())
