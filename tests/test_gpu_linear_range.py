"""Linear attention over the range of fp32: large keys, values, queries and states beside decays that take most of them away,
states that grow, and decays that are not finite.  Tolerances: linear_reference."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_linear_attention import Problem, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# tokens of one step, of a chunk, of several and of segments; decays of 2^-39 in 32 tokens are just below those after which
# scales go into the accumulators
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 20, 70, 300, 1100])
@pytest.mark.parametrize("q,k,v,state", [(1, 1, 1e27, 0), (1, 1e20, 1e13, 0), (1, 1e14, 1e23, 1), (1e-3, 1, 1e37, 1e36),
                                         (1e30, 1, 1, 1), (1e20, 1e-20, 1e25, 1e5), (1, 1, 1, 1e36), (1e-30, 1e36, 1e-2, 0)])
def test_large_numbers(pkg, dev, kind, n, q, k, v, state):  # noqa: F811
    g = torch.Generator().manual_seed(n)
    decay = -39 * math.log(2) / 32 * (1 + 0.1 * torch.rand(n, 3, generator=g) - 0.1)
    decay[:, 1] *= 0.02
    p = Problem(dev, [n], 3, 1, 64, 64, kind, decay=decay)
    p.q, p.k, p.v = ((x.float() * by).to(x.dtype) for x, by in ((p.q, q), (p.k, k), (p.v, v)))
    p.states *= state
    p.check(pkg)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [70, 300, 1100])
def test_large_numbers_that_begin_late(pkg, dev, kind, n):  # noqa: F811
    """In the middle of a batch of chunks, in one channel of one head."""
    decay = torch.full((n, 4), -39 * math.log(2) / 32)
    p = Problem(dev, [n], 4, 2, 128, 128, kind, decay=decay)
    at = n // 2 + 20
    p.v[at:, 1, 77] = 1e32
    p.check(pkg)
    p.k[at + 1, 1, 100] = 1e35
    p.v[:, 2:] *= 1e-3
    p.check(pkg)
    p.q[-2:, 0, 5] = 1e33
    p.v[at:, 1, 77] = 1.0
    p.check(pkg)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("state", [1e37, 1e-30])
@pytest.mark.parametrize("n", [5, 100, 900])
def test_states_of_any_size(pkg, dev, kind, state, n):  # noqa: F811
    """Large ones that have gone by the time that large queries come; small ones and small values."""
    decay = torch.full((n + 3, 2), -39 * math.log(2) / 32)
    decay[:, 1] /= 2
    p = Problem(dev, [n, 3], 2, 1, 64, 128, kind, decay=decay)
    p.states *= state
    p.v *= min(state, 1)
    if n >= 100:
        p.q[n // 2:n] *= 1e4
    p.check(pkg, torch.float32)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_states_that_grow(pkg, dev, kind):  # noqa: F811
    """By more than fp32 holds, while there is nothing or next to nothing that grows."""
    n = 1100
    p = Problem(dev, [n], 2, 1, 64, 64, kind, decay=torch.full((n, 2), 0.5))
    p.states.zero_()
    p.v[:-20] = 0
    p.check(pkg)
    n = 768
    p = Problem(dev, [n], 2, 1, 64, 64, kind, decay=torch.full((n, 2), 0.4))
    p.states.zero_()
    p.v[:-9] = 0
    p.v[240:256] = (1e-30 * torch.randn(16, 2, 64, device=dev)).to(p.v.dtype)
    p.decay[512:] = 0.05
    p.check(pkg)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("n,at", [(3, 1), (31, 9), (150, 70), (150, 127), (300, 0), (900, 500), (900, 899)])
def test_decays_that_are_not_finite(pkg, dev, kind, value, n, at):  # noqa: F811
    """The head, from that token on; other heads, earlier tokens and other sequences keep their bits."""
    p = Problem(dev, [n, n], 4, 2, 64, 64, kind)
    clean, states = p.run(pkg)
    p.decay[at, 1] = value
    out, s = p.run(pkg)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[at:n, 1] = True
    assert torch.equal(out[~hit], clean[~hit]) and not bool(torch.isfinite(out[hit]).any())
    rest = torch.zeros_like(states, dtype=torch.bool)
    rest[p.dst[0], 1] = True
    assert torch.equal(s[~rest], states[~rest]) and not bool(torch.isfinite(s[rest]).any())
