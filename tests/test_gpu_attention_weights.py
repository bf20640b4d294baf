"""Weights far below a row's largest, as the first token of a context leaves them in many models: one key takes nearly all
of the weight, its value is nothing, and the output is what the others make.

Tolerance, derived: that of test_gpu_attention.py, but for weights in fp16 below its normal range.  A row's weights are
scaled so that the largest of a wave is 2^6 at the least when it comes: half a step there, 2^-25, is 2^-31 of the
largest weight for each key.  bf16 has fp32's range.  Outputs in fp32, or bf16 with a half step of 2^-8 or so."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402
from test_gpu_attention import TYPES, Problem, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def sink(n, new, gap, spread, cache, q_type, d):
    """Key `where` lies `gap` above the others' mean score, whose deviation is `spread`; its value is zero."""
    p = Problem([n], [new], 1, 4, d, 16, cache, q_type, seed=7)
    g = torch.Generator().manual_seed(n)
    pool = torch.zeros(2, p.k.shape[0], 1, 16, d)
    p.q = torch.ones_like(p.q)
    score = spread * torch.randn(n, generator=g)
    value = 1 + 0.25 * torch.randn(n, d, generator=g)
    where = 3
    score[where], value[where] = gap, 0
    for j in range(n):
        pool[0, p.table[0, j // 16], 0, j % 16] = score[j] / (d * p.scale)
        pool[1, p.table[0, j // 16], 0, j % 16] = value[j]
    if cache == "q8":
        (p.k, p.ks), (p.v, p.vs) = ref.codes(pool[0]), ref.codes(pool[1])
    else:
        p.k, p.v = pool[0].to(TYPES[cache]), pool[1].to(TYPES[cache])
    return p


@pytest.mark.parametrize("cache,q_type", [("f16", None), ("bf16", None), ("q8", "f16"), ("q8", "bf16")])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,new", [(128, 1), (120, 6), (3000, 1), (700, 40)])
@pytest.mark.parametrize("gap", [10, 15, 17, 18])
@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_small_weights_beside_a_large_one(pkg, dev, gap, spread, n, new, d, cache, q_type):  # noqa: F811
    print(f"[sink] {gap} {spread} {n} {new} {d} {cache} {q_type}", flush=True)
    p = sink(n, new, gap, spread, cache, q_type, d)
    want, want_lse, size, terms = ref.attention(p.q, p.k, p.v, p.ks, p.vs, p.table, p.starts, p.kv_len, True, 0, p.scale)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    for out_type, lse in ((torch.float32, True), (torch.float32, False), (torch.bfloat16, False)):
        got = pkg.paged_attention(q, c, table, starts, kv_len, new, n, lse=lse, scale=p.scale, out_type=out_type)
        got, sums = got if lse else (got, None)
        exact = cache != "q8" or out_type != torch.bfloat16
        u = 2.0 ** -8 if cache == "bf16" else 2.0 ** -11
        score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20 + (0 if exact else 2.0 ** -11 * terms)
        values = u + (2.0 ** -11 + 127 * 2.0 ** -25 if cache == "q8" else 0)
        tail = 0 if cache == "bf16" else n * 2.0 ** -31 * ref.stored(p.v, p.vs).abs().max().item()
        # sum of weights at least the largest, so that a tail's share is at most itself
        tol = size * (values + 2 * score[..., None]) + tail + torch.finfo(out_type).eps / 2 * want.abs()
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), (out_type, (err / tol).max().item(), (err / want.abs().clamp(min=1e-30)).max().item())
        if lse:
            e = (sums.cpu().double() - want_lse).abs()
            assert bool((e <= score + 2.0 ** -22 * want_lse.abs()).all()), e.max().item()


@pytest.mark.parametrize("cache,q_type", [("f16", None), ("q8", "f16"), ("q8", "bf16")])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("n,new,where", [(128, 1, 100), (120, 6, 113), (700, 40, 650), (700, 40, 672), (700, 40, 699)])
def test_the_large_one_comes_late(pkg, dev, n, new, where, d, cache, q_type):  # noqa: F811
    """Sums and weights that are already there are scaled down when it comes."""
    p = sink(n, new, 16, 0.5, cache, q_type, d)
    (page, off), (last, end) = [(int(p.table[0, j // 16]), j % 16) for j in (3, where)]
    for x in (p.k, p.v, p.ks, p.vs):
        if x is not None:
            x[page, :, off], x[last, :, end] = x[last, :, end].clone(), x[page, :, off].clone()
    want, want_lse, size, terms = ref.attention(p.q, p.k, p.v, p.ks, p.vs, p.table, p.starts, p.kv_len, True, 0, p.scale)
    got, lse = p.run(pkg, dev, out_type=torch.float32)
    score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20
    values = 2.0 ** -11 + (2.0 ** -11 + 127 * 2.0 ** -25 if cache == "q8" else 0)
    # as above, and half a step once more for the weights that are scaled as they are
    tol = size * (values + 2 * score[..., None]) + n * 2.0 ** -30 * ref.stored(p.v, p.vs).abs().max().item()
    tol = tol + 2.0 ** -24 * want.abs()
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()
    assert bool(((lse.cpu().double() - want_lse).abs() <= score + 2.0 ** -22 * want_lse.abs()).all())
