"""Linear attention on the GPU against the token-by-token form in 64 bits: types, heads, lengths, decays, slots and the
edges of its chunks and segments.  Tolerances: linear_reference."""
import math

import pytest

torch = pytest.importorskip("torch")
import linear_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


class Problem:
    def __init__(self, dev, lens, heads, hk, dk, dv, kind, each=True, seed=1, slots=None, decay=None, before=0, after=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
        total = before + sum(lens) + after
        self.q, self.k = ((rnd(total, hk, dk) * dk ** -0.5 * 1.3).to(TYPES[kind]) for _ in range(2))
        self.v = rnd(total, heads, dv).to(TYPES[kind])
        slow = torch.exp(torch.linspace(math.log(0.5), math.log(1e-3), heads, device=dev))
        self.decay = -slow * torch.nn.functional.softplus(rnd(total, heads)) if each else -slow
        if decay is not None:
            self.decay = decay.to(dev)
        self.lens, self.scale = list(lens), 0.7
        self.starts = torch.tensor([before + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
        n = 2 * len(lens) if slots is None else slots
        self.states = 0.3 * rnd(n, heads, dk, dv)
        order = torch.randperm(max(n, 2 * len(lens)), device=dev, generator=g)
        self.src, self.dst = order[:len(lens)].contiguous(), order[len(lens):2 * len(lens)].contiguous()

    def run(self, pkg, states=None, out_type=None, most_q=None):
        s = self.states.clone() if states is None else states
        out = pkg.linear_attention(self.q, self.k, self.v, self.decay, self.starts, max(self.lens + [1]) if most_q is None
                                   else most_q, s, self.src, self.dst, self.scale, out_type)
        return out, s

    def want(self, most_q=None):
        return (*ref.linear(self.q, self.k, self.v, self.decay, self.starts, most_q, self.states, self.src, self.dst,
                            self.scale), self.q.shape[2])

    def check(self, pkg, out_type=None):
        print(f"[linear] lens={self.lens[:6]} q={tuple(self.q.shape)} v={tuple(self.v.shape)} {self.q.dtype} {out_type}",
              flush=True)
        out, states = self.run(pkg, out_type=out_type)
        torch.cuda.synchronize()
        first, end = int(self.starts[0]), int(self.starts[-1])
        w = self.want()
        ref.compare(out[first:end], states, (w[0][first:end], w[1][first:end], *w[2:]))
        return out, states


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("dv", [64, 128, 256])
@pytest.mark.parametrize("each", [True, False])
def test_lengths(pkg, dev, kind, dk, dv, each):
    """No token, one, and around a chunk's end; a state from a slot and to another."""
    for heads, hk, lens in ((2, 1, [1, 0, 5, 1]), (2, 2, [130, 1, 63, 64, 0, 65, 17]), (3, 1, [200, 33])):
        Problem(dev, lens, heads, hk, dk, dv, kind, each, seed=dk + dv).check(pkg)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[1, 1, 1], [16, 3], [100, 31]])
def test_output_types(pkg, dev, kind, out, lens):
    got, _ = Problem(dev, lens, 4, 2, 128, 128, kind).check(pkg, TYPES[out])
    assert got.dtype == TYPES[out]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 49, 96, 127, 128, 129])
def test_every_way_to_go(pkg, dev, kind, n):
    Problem(dev, [n, max(1, n - 1)], 8, 4, 128, 64, kind, seed=n).check(pkg)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 256), (128, 128), (256, 64)])
def test_long_sequences_in_segments(pkg, dev, kind, dk, dv):
    """Few heads: the sequence is cut, and the states of the segments are joined."""
    Problem(dev, [1500], 2, 1, dk, dv, kind, seed=dk).check(pkg)
    Problem(dev, [900, 64, 1, 0, 513, 640], 2, 2, dk, dv, kind, seed=dk, each=False).check(pkg)


def test_many_heads(pkg, dev):
    Problem(dev, [300, 77], 64, 16, 128, 128, "bf16").check(pkg)
    Problem(dev, [1] * 70, 32, 32, 128, 128, "f32").check(pkg)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 200, 1100])
def test_decays_from_nothing_to_all(pkg, dev, kind, n):
    """Heads that keep everything, forget at once, and now and then forget everything (the rest keeps its bits)."""
    g = torch.Generator().manual_seed(5)
    decay = torch.zeros(n, 6)
    decay[:, 1] = -300.0
    decay[:, 2] = -math.inf
    decay[:, 3] = torch.where(torch.rand(n, generator=g) < 0.1, -1000.0, -0.01)
    decay[:, 4] = torch.where(torch.rand(n, generator=g) < 0.1, -math.inf, -1e-4)
    decay[:, 5] = -torch.exp(6 * torch.randn(n, generator=g))
    Problem(dev, [n], 6, 2, 64, 64, kind, decay=decay).check(pkg)
    Problem(dev, [n], 3, 1, 64, 64, kind, decay=torch.tensor([0.0, -math.inf, 0.01])).check(pkg)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[40, 3, 90], [1, 1, 1], [700, 20, 5]])
def test_slots(pkg, dev, kind, lens):
    """In place, from nothing, to nowhere, past the states, several from one; other slots are left alone."""
    p = Problem(dev, lens, 2, 1, 64, 64, kind, slots=6)
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=dev)  # noqa: E731
    for src, dst in (((4, 1, 0), (4, 1, 0)), ((-1, 6, 2), (0, 1, 3)), ((2, 2, 2), (-1, 1 << 40, 5)),
                     ((-(1 << 40), 5, 0), (1, 2, 3))):
        p.src, p.dst = i64(*src), i64(*dst)
        _, states = p.check(pkg)
        rest = [i for i in range(6) if i not in dst]
        assert torch.equal(states[rest], p.states[rest])
    p.states[3] = math.nan  # a slot that is written, and not read
    p.src, p.dst = i64(1, -1, 2), i64(3, 4, 5)
    out, states = p.run(pkg)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(states).all())
    most = max(lens)
    bare = pkg.linear_attention(p.q, p.k, p.v, p.decay, p.starts, most, scale=p.scale)
    p.src = i64(-1, -1, -1)
    assert torch.equal(bare, p.run(pkg)[0])
    kept = p.states.clone()
    out = pkg.linear_attention(p.q, p.k, p.v, p.decay, p.starts, most, kept, to_slots=p.dst, scale=p.scale)
    assert torch.equal(out, bare) and torch.equal(kept, p.run(pkg)[1])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,at", [(9, 4), (150, 70), (150, 127), (900, 500)])
def test_what_is_not_finite_stays_where_it_belongs(pkg, dev, kind, value, n, at):
    """A value: its channel, from its token on.  A key or a query: its head from there on, or its row."""
    p = Problem(dev, [n, n], 4, 2, 64, 64, kind, each=False)
    clean, states = p.run(pkg)

    def changed():
        out, s = p.run(pkg)
        return out, s, (out != clean) | torch.isnan(out), (s != states) | torch.isnan(s)

    kept = p.v[at, 1, 37].clone()
    p.v[at, 1, 37], p.v[at + 1, 1, 3] = value, value
    out, s, diff, sdiff = changed()
    allowed = torch.zeros_like(diff)
    allowed[at:n, 1, 37] = True
    allowed[at + 1:n, 1, 3] = True
    assert not bool((diff & ~allowed).any()) and not bool(torch.isfinite(out[allowed]).any())
    rest = torch.zeros_like(sdiff)
    rest[p.dst[0], 1, :, 37] = rest[p.dst[0], 1, :, 3] = True
    assert not bool((sdiff & ~rest).any()) and not bool(torch.isfinite(s[rest]).any())
    p.v[at, 1, 37], p.v[at + 1, 1, 3] = kept, 0.5
    clean, states = p.run(pkg)
    kept = p.k[at, 1, 5].clone()
    p.k[at, 1, 5] = value
    out, s, diff, sdiff = changed()
    allowed = torch.zeros_like(diff)
    allowed[at:n, 2:] = True
    assert not bool((diff & ~allowed).any())
    assert bool(torch.isfinite(s[p.dst[1]]).all()) and bool(torch.isfinite(s[p.dst[0], :2]).all())
    assert not bool(torch.isfinite(s[p.dst[0], 2:, 5]).any())
    p.k[at, 1, 5] = kept
    p.q[at, 0, 9] = value
    out, s, diff, sdiff = changed()
    allowed = torch.zeros_like(diff)
    allowed[at, :2] = True
    assert not bool((diff & ~allowed).any()) and not bool(sdiff.any()) and not bool(torch.isfinite(out[at, :2]).any())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [160, 1400])
def test_values_that_are_not_finite_in_chunk_after_chunk(pkg, dev, kind, n):
    """Each in a channel of its own, several in one chunk, in every segment: every channel from its token on."""
    p = Problem(dev, [n], 2, 1, 128, 128, kind, each=False)
    clean, states = p.run(pkg)
    allowed, rest = torch.zeros_like(clean, dtype=torch.bool), torch.zeros_like(states, dtype=torch.bool)
    for c, t in enumerate([3, 31, 32, 33, 63, 64, 70, 95, 97, 128, 130, n // 2, n // 2 + 1, n - 40, n - 2, n - 1]):
        p.v[t, 1, 8 * c + c % 8] = math.nan if c % 2 else math.inf
        allowed[t:, 1, 8 * c + c % 8] = True
        rest[p.dst[0], 1, :, 8 * c + c % 8] = True
    out, s = p.run(pkg)
    assert torch.equal(out[~allowed], clean[~allowed]) and not bool(torch.isfinite(out[allowed]).any())
    assert torch.equal(s[~rest], states[~rest]) and not bool(torch.isfinite(s[rest]).any())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[1, 1], [70, 5], [800, 130]])
def test_rows_of_no_sequence(pkg, dev, kind, lens):
    """NaN before the first and behind the last: not a bit changes, and those outputs are not written."""
    p = Problem(dev, lens, 2, 2, 128, 64, kind, before=3, after=70)
    a, b = 3, 3 + sum(lens)
    want, states = p.check(pkg)
    for x in (p.q, p.k, p.v, p.decay):
        x[:a], x[b:] = math.nan, math.nan
    out = torch.full_like(want, 7.0)
    got = p.states.clone()
    args = pkg._LINEAR.pack(p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), p.decay.data_ptr(), p.starts.data_ptr(),
                            got.data_ptr(), p.src.data_ptr(), p.dst.data_ptr(), out.data_ptr(), 256, 256, 128, 2,
                            got.shape[0], 2, b + 70, max(lens), 2, 2, 128, 64, pkg._types(torch)[p.q.dtype],
                            pkg._types(torch)[out.dtype], p.scale)
    ws = torch.empty(max(1, pkg.lib().iq4xs_linear_attention_workspace_bytes(args)), dtype=torch.uint8, device=dev)
    ws.fill_(255)  # NaN
    pkg.lib().check("iq4xs_linear_attention", args, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out[a:b], want[a:b]) and torch.equal(got, states)
    assert bool((out[:a] == 7).all()) and bool((out[b:] == 7).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("most_q", [1, 5, 40, 300])
def test_sequences_of_more_than_most_q(pkg, dev, kind, most_q):
    """Their first most_q tokens, and the states after those."""
    p = Problem(dev, [700, 3, 41], 2, 1, 64, 64, kind)
    out, states = p.run(pkg, most_q=most_q)
    w = p.want(most_q)
    rows = [s + i for s, n in zip((0, 700, 703), p.lens) for i in range(min(n, most_q))]
    ref.compare(out[rows], states, (w[0][rows], w[1][rows], *w[2:]))


@pytest.mark.parametrize("n", [1, 40, 700])
def test_strides(pkg, dev, n):
    """Views of one projection's rows, and decays as they are."""
    p = Problem(dev, [n, n], 4, 2, 128, 64, "bf16")
    want, states = p.run(pkg)
    wide = torch.full((2 * n, 2 * 128 + 2 * 128 + 4 * 64 + 8), math.nan, dtype=p.q.dtype, device=dev)
    q, k, v = wide[:, :256].view(-1, 2, 128), wide[:, 256:512].view(-1, 2, 128), wide[:, 512:768].view(-1, 4, 64)
    for a, b in ((q, p.q), (k, p.k), (v, p.v)):
        a.copy_(b)
    s = p.states.clone()
    got = pkg.linear_attention(q, k, v, p.decay, p.starts, n, s, p.src, p.dst, p.scale)
    assert torch.equal(got, want) and torch.equal(s, states)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompts_and_then_tokens(pkg, dev, kind):
    """A prompt, a draft and single tokens, each from the state before, against the whole at once."""
    p = Problem(dev, [150], 4, 2, 64, 128, kind)
    w = p.want()
    states = p.states.clone()
    outs, at, slot = [], 0, p.src
    for n in (100, 30, 13, 1, 1, 4, 1):
        starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
        part = slice(at, at + n)
        outs.append(pkg.linear_attention(p.q[part], p.k[part], p.v[part], p.decay[part], starts, n, states, slot, p.dst,
                                         p.scale))
        at, slot = at + n, p.dst
    ref.compare(torch.cat(outs), states, w)


@pytest.mark.parametrize("lens", [[1, 1], [20, 9], [300, 70], [1000]])
def test_graphs_streams_and_repeats(pkg, dev, lens):
    p = Problem(dev, lens, 4, 2, 128, 128, "bf16")
    first, states = p.run(pkg)
    for _ in range(3):
        again, s = p.run(pkg)
        assert torch.equal(first, again) and torch.equal(states, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, s = p.run(pkg)
        assert torch.equal(first, again) and torch.equal(states, s)
        live = p.states.clone()
        p.dst = p.src  # in place: each replay goes on from the one before
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, _ = p.run(pkg, live)
        live.copy_(p.states)
        eager = p.states.clone()
        g = torch.Generator(device=dev).manual_seed(3)
        for rep in range(4):
            p.v.copy_(torch.randn(p.v.shape, device=dev, generator=g))
            out.fill_(float("nan"))
            graph.replay()
            side.synchronize()
            kept = out.clone()
            want, _ = p.run(pkg, eager)
            assert torch.equal(kept, want) and torch.equal(live, eager), rep
    torch.cuda.current_stream().wait_stream(side)


def test_states_past_32_bits(pkg, dev):
    """2^32 elements and more: the last slots are their own."""
    slots, heads = 1030, 64
    p = Problem(dev, [1, 70], heads, 16, 256, 256, "bf16", slots=2)
    states = torch.empty(slots, heads, 256, 256, device=dev)
    for i in range(2):
        states[slots - 2 + i] = p.states[i]
    p.src = torch.tensor([0, 1], device=dev)
    p.dst = p.src
    want, new = p.run(pkg)
    p.src = p.dst = p.src + slots - 2
    got, _ = p.run(pkg, states)
    assert torch.equal(got, want) and torch.equal(states[-2:], new)


def test_refused_tensors(pkg, dev):
    p = Problem(dev, [3, 4], 4, 2, 64, 128, "bf16")

    def run(q=p.q, k=p.k, v=p.v, decay=p.decay, starts=p.starts, most_q=4, states=p.states, src=p.src, dst=p.dst, **kw):
        return pkg.linear_attention(q, k, v, decay, starts, most_q, states, src, dst, **kw)

    run()
    for bad in (dict(q=p.q.float()), dict(k=p.k.half()), dict(v=p.v.float()), dict(q=p.q[:, :1]), dict(k=p.k[:5]),
                dict(v=p.v[:, :3]), dict(q=p.q.cpu()), dict(k=p.k.cpu()), dict(v=p.v.cpu()), dict(q=p.q[0]),
                dict(v=p.v.transpose(1, 2).contiguous().transpose(1, 2)), dict(decay=p.decay.double()),
                dict(decay=p.decay[:, :2]), dict(decay=p.decay[:5]), dict(decay=p.decay[0, :3]), dict(decay=p.decay.cpu()),
                dict(starts=p.starts.long()), dict(starts=p.starts.cpu()), dict(states=None), dict(states=p.states.half()),
                dict(states=p.states[:, :3]), dict(states=p.states.cpu()), dict(src=p.src.int()), dict(dst=p.dst[:1]),
                dict(dst=p.dst.cpu()), dict(out_type=torch.int8)):
        with pytest.raises(ValueError):
            run(**bad)
    for bad in (dict(most_q=0), dict(scale=math.nan), dict(q=p.q[..., :32], k=p.k[..., :32])):
        with pytest.raises((pkg.Iq4xsError, ValueError)):
            run(**bad)
    none = pkg.linear_attention(p.q[:0], p.k[:0], p.v[:0], p.decay[:0], p.starts * 0, 1, p.states, p.src, p.dst)
    assert none.shape == (0, 4, 128)
