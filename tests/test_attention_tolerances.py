"""What the tolerances of tests/test_gpu_attention_8bit.py let through, on the CPU: the form in 64 bits, rounded once,
passes; with keys rounded to fp16 it does not where keys are exact, and does where the kernels round them."""
import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402
from test_gpu_attention import Problem  # noqa: E402
from test_gpu_attention_8bit import compare  # noqa: E402


def attention(p, keys, scales=None):
    values = (p.v, p.vs) if scales is not None else (ref.stored(p.v, p.vs), None)
    return ref.attention(p.q, keys, values[0], scales, values[1], p.table, p.starts, p.kv_len, True, 0, p.scale)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [8, 40])
def test_rounded_keys_pass_where_they_are_rounded_only(d, new):
    p = Problem([new + 300, new + 40], [new] * 2, 2, 4, d, 16, "q8", "f16", seed=d)
    want = attention(p, p.k, p.ks)
    out, lse = want[0], want[1]
    compare(p, out.float(), lse.float(), want)
    compare(p, out.half(), None, want)
    compare(p, out.bfloat16(), None, want)
    out, lse, _, _ = attention(p, ref.stored(p.k, p.ks).half())
    with pytest.raises(AssertionError):
        compare(p, out.float(), lse.float(), want)
    if new > 8:
        compare(p, out.bfloat16(), None, want)
