"""Linear attention on the GPU over batches of prompts and many single tokens, whose segments are counted compactly: against
64 bits, with nothing written past the workspace and nothing read that was not written.  Tolerances: linear_reference."""
import pytest

torch = pytest.importorskip("torch")
import linear_reference as ref  # noqa: E402
from test_gpu_linear_attention import Problem, dev  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def packed(pkg, p, out, states):
    total, hk, dk = p.q.shape
    heads, dv = p.v.shape[1:]
    kinds = pkg._types(torch)
    return pkg._block(pkg._LINEAR, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), p.decay.data_ptr(), p.starts.data_ptr(),
                      states.data_ptr(), p.src.data_ptr(), p.dst.data_ptr(), out.data_ptr(), hk * dk, hk * dk, heads * dv,
                      heads, states.shape[0], len(p.lens), total, max(p.lens), heads, hk, dk, dv, kinds[p.q.dtype],
                      kinds[out.dtype], p.scale)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,before,after", [([1500] + [1] * 63, 0, 0), ([1] * 63 + [1500], 5, 3),
                                               ([1] * 40 + [0, 1300, 0, 0, 1, 1] + [1] * 60, 0, 2),
                                               ([1] * 130 + [800, 513, 1, 769, 0] + [1] * 70, 9, 0), ([257] * 20, 0, 0),
                                               ([400] * 20, 0, 0),
                                               ([3, 0, 2000, 1999], 300, 40), ([1] * 300 + [1025, 512, 511, 1024], 1, 1)])
def test_prompts_among_single_tokens(pkg, dev, kind, lens, before, after):  # noqa: F811
    p = Problem(dev, lens, 2, 1, 64, 64, kind, before=before, after=after)
    print(f"[batches] {len(lens)} sequences, {sum(lens)} tokens, {kind}", flush=True)
    out, states = torch.full_like(p.v, 7.0), p.states.clone()
    args = packed(pkg, p, out, states)
    need = pkg.lib().iq4xs_linear_attention_workspace_bytes(args)
    assert need < 64 * 2 * 64 * 64 * 4  # none of 257 tokens each: one segment
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device=dev)  # NaN
    stream = torch.cuda.current_stream().cuda_stream
    pkg.lib().check("iq4xs_linear_attention", args, ws.data_ptr(), need, stream)
    torch.cuda.synchronize()
    first, end = before, before + sum(lens)
    assert bool((ws[need:] == 255).all()) and bool((out[:first] == 7).all()) and bool((out[end:] == 7).all())
    w = p.want()
    ref.compare(out[first:end], states, (w[0][first:end], w[1][first:end], *w[2:]))
    again, other = torch.full_like(out, 7.0), p.states.clone()  # over the workspace as it was left
    pkg.lib().check("iq4xs_linear_attention", packed(pkg, p, again, other), ws.data_ptr(), need, stream)
    assert torch.equal(again, out) and torch.equal(other, states)


@pytest.mark.parametrize("most_q", [40, 700])
def test_prompts_cut_short_among_single_tokens(pkg, dev, most_q):  # noqa: F811
    p = Problem(dev, [1] * 30 + [900, 3, 1400, 1, 650] + [1] * 50, 2, 1, 64, 64, "bf16")
    out, states = p.run(pkg, most_q=most_q)
    w = p.want(most_q)
    rows = [int(s) + i for s, n in zip(p.starts, p.lens) for i in range(min(n, most_q))]
    ref.compare(out[rows], states, (w[0][rows], w[1][rows], *w[2:]))


def test_lengths_that_change_under_a_graph(pkg, dev):  # noqa: F811
    """The same rows dealt to sequences otherwise from replay to replay."""
    n = 2000
    p = Problem(dev, [n - 40] + [1] * 40, 2, 1, 64, 64, "bf16")
    live = p.states.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.linear_attention(p.q, p.k, p.v, p.decay, p.starts, n, live, p.src, p.dst, p.scale)
    for lens in ([n - 40] + [1] * 40, [1] * 40 + [n - 40], [1] * 20 + [1000] + [1] * 19 + [961], [n] + [0] * 40,
                 [50] * 39 + [49, 1]):
        p.lens = lens
        p.starts.copy_(torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32))
        live.copy_(p.states)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want, states = p.run(pkg, most_q=n)
        assert torch.equal(out, want) and torch.equal(live, states)
        ref.compare(out, live, p.want())
