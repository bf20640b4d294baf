"""Attention over an 8-bit cache, held to what each kernel rounds.

Which keys are exact and which are rounded follows the outputs: bf16 outputs alone, of more than 32 rows of a cache head,
go through keys rounded to fp16 and one fp16 number for each weight; all others through exact keys and two numbers.

Tolerance, derived.  Scores: a sum of head terms in fp32, (head + 8) 2^-24 of the terms' magnitudes, and 2^-20 for exp2
and log2; 2^-11 of the terms more where keys are rounded.  A weight moves by as much, and so does their sum.  Values: half
a step of fp16, 2^-11, and 2^-25 below its normal range.  One number for a weight: 2^-11 of it, which moves the sum too;
two: 2^-21.  Either way no less than 2^-31 of the row's largest weight for each key.  The output is rounded once."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402
from test_gpu_attention import Problem, dev, vars_of  # noqa: E402,F401

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rounds_keys(p, out_type, lse):
    return out_type == BF16 and not lse and max(p.new) * (p.q.shape[1] // p.k.shape[1]) > 32


def run(p, pkg, dev, out_type, lse=False, causal=True, window=0):  # noqa: F811
    q, c, table, starts, kv_len = p.on(pkg, dev)
    got = pkg.paged_attention(q, c, table, starts, kv_len, max(p.new), max(p.kv + [1]), causal=causal, window=window,
                              lse=lse, scale=p.scale, out_type=out_type)
    got, sums = got if lse else (got, None)
    return got.cpu(), None if sums is None else sums.cpu()


def compare(p, got, sums, want, causal=True, window=0):
    out, lse, size, terms = want
    d, rounded = p.q.shape[-1], rounds_keys(p, got.dtype, sums is not None)
    score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20 + (2.0 ** -11 * terms if rounded else 0)
    weights = 2 * 2.0 ** -11 if rounded else 2.0 ** -20
    tail = max(p.kv + [1]) * 2.0 ** -31 * ref.stored(p.v, p.vs).abs().nan_to_num(posinf=0).max()
    tol = size * (weights + 2.0 ** -11 + 2 * torch.expm1(score)[..., None]) + 2.0 ** -25 + tail
    tol = tol + torch.finfo(got.dtype).eps / 2 * out.abs() + (2.0 ** -25 if got.dtype == F16 else 0)
    err = (got.double() - out).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol).all()), (rounded, (err / tol).max().item())
    none = lse == -math.inf
    assert bool((got[none] == 0).all())
    if sums is not None:
        assert bool((sums[none] == -math.inf).all())
        e = (sums.double() - lse)[~none].abs()
        assert bool((e <= score[~none] + 2.0 ** -22 * lse[~none].abs()).all()), e.max().item()


def check(p, pkg, dev, causal=True, window=0, kinds=((BF16, False), (F32, True), (F16, False))):  # noqa: F811
    want = ref.attention(p.q, p.k, p.v, p.ks, p.vs, p.table, p.starts, p.kv_len, causal, window, p.scale)
    for out_type, lse in kinds:
        print(f"[8 bits] {vars_of(p)} causal={causal} window={window} {out_type} {lse}", flush=True)
        compare(p, *run(p, pkg, dev, out_type, lse, causal, window), want)


@pytest.mark.parametrize("q_type", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group", [([31, 7], 1), ([32, 32], 1), ([33, 1], 1), ([8, 4], 4), ([11, 4], 3), ([7, 9], 5),
                                       ([70, 1, 131, 64], 2), ([40, 31, 100], 8), ([129, 64, 65, 63], 1)])
def test_both_sides_of_the_rule(pkg, dev, new, group, d, q_type):  # noqa: F811
    kv = [n + (0, 50, 129, 700)[i] for i, n in enumerate(new)]
    check(Problem(kv, new, 2, group, d, 16, "q8", q_type, seed=d + group), pkg, dev)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 17, 63, 64, 100, 10000])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(pkg, dev, window, causal, d):  # noqa: F811
    check(Problem([75 + 290, 75, 75 + 31], [75] * 3, 2, 2, d, 16, "q8", "bf16", seed=window), pkg, dev, causal, window)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_page_sizes(pkg, dev, d, page):  # noqa: F811
    check(Problem([90, 190, 391], [90, 40, 3], 2, 2, d, page, "q8", "f16", seed=page), pkg, dev)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_every_key(pkg, dev, d):  # noqa: F811
    check(Problem([280, 80, 20], [80, 80, 9], 2, 8, d, 16, "q8", "bf16"), pkg, dev, causal=False)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_several_splits(pkg, dev, d):  # noqa: F811
    check(Problem([3000, 1100], [40, 35], 1, 2, d, 64, "q8", "bf16", seed=d), pkg, dev)
    check(Problem([3000, 1100], [40, 35], 1, 2, d, 64, "q8", "f16", seed=d), pkg, dev, window=1500)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_see_nothing(pkg, dev, d):  # noqa: F811
    check(Problem([59, 0, 1, 60], [60, 60, 60, 1], 2, 2, d, 16, "q8", "bf16"), pkg, dev)
    check(Problem([2, 0, 1], [60] * 3, 1, 1, d, 16, "q8", "f16"), pkg, dev, window=1)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_outside_the_cache(pkg, dev, d):  # noqa: F811
    p = Problem([160, 80], [60] * 2, 2, 2, d, 16, "q8", "bf16")
    p.table[0, 1], p.table[0, 3], p.table[1, 0] = -1, p.k.shape[0], 1 << 30
    check(p, pkg, dev)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_hidden_keys_and_values_do_not_matter(pkg, dev, d, bad):  # noqa: F811
    """Past a sequence's end, in pages of nobody, before every window, and (NaN) in a token that the first rows do not
    see."""
    new = 70
    p = Problem([new + 37, new + 5], [new] * 2, 2, 4, d, 16, "q8", "bf16", seed=new)
    clean, _ = run(p, pkg, dev, BF16, window=20)

    def spoil(page, off):
        for x, s in ((p.k, p.ks), (p.v, p.vs)):
            x[page, :, off], s[page, :, off] = 127, bad

    for page in set(range(p.k.shape[0])) - set(p.table[p.table >= 0].tolist()):
        for off in range(16):
            spoil(page, off)
    for s, n in enumerate(p.kv):
        for j in (*range(n, -(-n // 16) * 16), *range(max(0, n - new + 1 - 20))):
            spoil(int(p.table[s, j // 16]), j % 16)
    again, _ = run(p, pkg, dev, BF16, window=20)
    assert torch.equal(clean, again)
    if math.isnan(bad):
        for s, n in enumerate(p.kv):
            j = n - new + 1
            spoil(int(p.table[s, j // 16]), j % 16)
        last, _ = run(p, pkg, dev, BF16, window=20)
        for s in range(2):
            for i in range(new):
                row = s * new + i
                assert bool(torch.isnan(last[row]).all()) if 1 <= i < 21 else torch.equal(last[row], clean[row]), (s, i)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_calls_repeat_bit_for_bit(pkg, dev, d):  # noqa: F811
    p = Problem([33, 130, 1500, 9000], [33, 40, 100, 64], 1, 8, d, 16, "q8", "bf16", seed=d)
    q, c, table, starts, kv_len = p.on(pkg, dev)
    first = None
    for _ in range(12):
        got = pkg.paged_attention(q, c, table, starts, kv_len, 100, 9000, out_type=BF16)
        first = got if first is None else first
        assert torch.equal(got, first)


@pytest.mark.parametrize("new", [1, 5, 40, 90])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_exact_keys_of_a_long_context(pkg, dev, new, d):  # noqa: F811
    """Log-sum-exp and fp32 outputs over many splits, in 64 bits on the GPU: what rounded keys (2^-11 of the terms) would
    not pass."""
    n, heads, group = 20011, 2, 4
    g = torch.Generator(device=dev).manual_seed(d)
    count = -(-n // 64)
    pool = torch.randn(2, count, heads, 64, d, device=dev, generator=g)
    (k, ks), (v, vs) = ref.codes(pool[0]), ref.codes(pool[1])
    q = (1.7 * torch.randn(new, heads * group, d, device=dev, generator=g)).half()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(count, dtype=torch.int32, device=dev)[None]
    out, lse = pkg.paged_attention(q, pkg.KVCache(k, v, ks, vs), table, i32(0, new), i32(n), new, n, lse=True,
                                   out_type=F32)
    flat = lambda c, s: ref.stored(c, s).transpose(0, 1).reshape(heads, -1, d)[:, :n]  # noqa: E731
    K, V = flat(k, ks), flat(v, vs)
    for i in range(new):
        m = n - new + 1 + i
        for h in range(heads):
            x = q[i, h * group:(h + 1) * group].double()
            z = x @ K[h, :m].t() / math.sqrt(d)
            terms = (x.abs() @ K[h, :m].abs().t()).amax(-1) / math.sqrt(d)
            w = torch.softmax(z, -1)
            o, size = w @ V[h, :m], w @ V[h, :m].abs()
            score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20
            tol = size * (2.0 ** -11 + 2.0 ** -20 + 2 * score[:, None]) + 2.0 ** -25 + n * 2.0 ** -31 * V.abs().max()
            err = (out[i, h * group:(h + 1) * group].double() - o).abs()
            assert bool((err <= tol).all()), (i, h, (err / tol).max().item())
            want = torch.logsumexp(z, -1)
            e = (lse[i, h * group:(h + 1) * group].double() - want).abs()
            assert bool((e <= score + 2.0 ** -22 * want.abs()).all()), (i, h, e.max().item(), score.max().item())
