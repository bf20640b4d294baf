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
