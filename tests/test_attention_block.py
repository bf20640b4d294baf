"""The example that runs the attention half of a layer: prompts, then steps from a replayed graph, against 64 bits.

Tolerance, derived: queries and stored keys are rounded (u = 2^-11 or 2^-8 of each term of a score; an 8-bit key by half
a code, and its scale by u), the norm, the turn and the sum in fp32 stay below 2^-16 of the terms; weights are rounded
(u, and 2^-25 of the largest each), values stored with u or half a code."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
import attention_reference as ref  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("attention_block", os.path.join(ROOT, "examples",
                                                                                  "attention_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def attended(block, q, k, v, pos, first):
    """Rows of one sequence over all its tokens in 64 bits; also the means of |v| and of a code's step, and a score's
    terms.  first: position of the first row."""
    d, group = block.head, block.q_heads // block.k_heads
    cpu = lambda t: t.cpu()  # noqa: E731
    q = ref.norm_rope(cpu(q), pos[first:], cpu(block.freqs), cpu(block.q_gain), block.eps, True)
    k = ref.norm_rope(cpu(k), pos, cpu(block.freqs), cpu(block.k_gain), block.eps, True)
    v = cpu(v).double()
    q = q.view(q.shape[0], -1, group, d)
    z = torch.einsum("thgd,nhd->thgn", q, k) * d ** -0.5
    most = torch.einsum("thgd,nhd->thgn", q.abs(), k.abs()).amax(-1) * d ** -0.5
    # terms of a score with every key's channel replaced by its group's code step
    step = k.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(*k.shape[:-1], -1, 32).flatten(-2) / 127
    coded = torch.einsum("thgd,nhd->thgn", q.abs(), step).amax(-1) * d ** -0.5
    seen = torch.arange(k.shape[0])[None] <= pos[first:, None]
    w = torch.softmax(z.masked_fill(~seen[:, None, None], -torch.inf), -1)
    vstep = v.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(*v.shape[:-1], -1, 32).flatten(-2) / 127
    mean = lambda x: torch.einsum("thgn,nhd->thgd", w, x).flatten(1, 2)  # noqa: E731
    return mean(v), mean(v.abs()), mean(vstep), most.flatten(1, 2), coded.flatten(1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("head,q_heads,k_heads", [(64, 8, 2), (128, 6, 1), (256, 4, 2)])
def test_prompts_then_steps_of_a_graph(example, kind, head, q_heads, k_heads):
    print(f"[block] {kind} {head} {q_heads} {k_heads}", flush=True)
    dev, hidden, prompts, steps = torch.device("cuda:0"), 512, [70, 1, 33], 4
    torch.manual_seed(3)
    block = example.synthetic_block(hidden, q_heads, k_heads, head, kind, dev)
    seqs = example.Sequences(len(prompts), max(prompts) + steps, 16, dev)
    cache = example.new_cache(seqs.pages, k_heads, 16, head, kind, dev)

    h = example.pkg.synthetic_activations(sum(prompts) * hidden, 5, device=dev).view(-1, hidden)
    q, k, v = block.project(h)
    rows = block.attend(q, k, v, cache, seqs, seqs.grow(prompts), max(prompts), max(prompts))
    cut = [t.split(prompts) for t in (q, k, v, rows)]
    history = [[(k.clone(), v.clone())] for k, v in zip(cut[1], cut[2])]
    checks = [(cut[0][i], i, 0, prompts[i], cut[3][i]) for i in range(len(prompts))]

    step = torch.empty(len(prompts), hidden, device=dev)
    graph, out = example.decode_graph(block, cache, seqs, step, seqs.room)
    for n in range(steps):
        step.copy_(example.pkg.synthetic_activations(step.numel(), 20 + n, device=dev).view_as(step))
        graph.replay()
        q, k, v = block.project(step)
        # the same step outside the graph gives the same bits: the token's slot is written again
        seqs.kv_len -= 1
        rows = block.attend(q, k, v, cache, seqs, seqs.step(), 1, seqs.room)
        again = example.pkg.mul_mat(block.wo, rows, q_heads * head, hidden, len(prompts))
        assert torch.equal(out, again), n
        for i in range(len(prompts)):
            history[i].append((k[i:i + 1].clone(), v[i:i + 1].clone()))
            checks.append((q[i:i + 1].clone(), i, prompts[i] + n, prompts[i] + n + 1, rows[i:i + 1].clone()))
    assert seqs.kv_len.tolist() == [p + steps for p in prompts]

    u = 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    for q, i, first, end, got in checks:
        k, v = (torch.cat(x)[:end] for x in zip(*history[i]))
        want, size, vstep, most, coded = attended(block, q, k, v, torch.arange(end), first)
        score = 2.0 ** -16 * most + 2 * u * most + (coded / 2 if kind == "q8" else 0)
        # a score that is off by e moves a weight by up to e^e - 1 both ways, the sum as much
        tol = size * (2 * u + 2.0 ** -11 + 2 * torch.expm1(score)[..., None]) + (vstep / 2 if kind == "q8" else 0)
        tol = tol + end * 2.0 ** -25 * v.abs().max().item()
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), (i, first, (err / tol).max().item())


def test_slots_of_sequences(example):
    """Positions and slots of prompts, then of steps, each slot once and in its sequence's pages."""
    seqs, used = example.Sequences(3, 40, 16, torch.device("cpu")), []
    assert (seqs.room, seqs.pages) == (48, 9)
    pos, slots, starts = seqs.grow([33, 0, 7])
    assert starts.tolist() == [0, 33, 33, 40] and pos.tolist() == [*range(33), *range(7)]
    used += slots.tolist()
    pos, slots, starts = seqs.grow([2, 5, 1])
    assert pos.tolist() == [33, 34, 0, 1, 2, 3, 4, 7]
    used += slots.tolist()
    pos, slots, starts = seqs.step()
    assert pos.tolist() == [35, 5, 8] and starts.tolist() == [0, 1, 2, 3] and seqs.kv_len.tolist() == [36, 6, 9]
    used += slots.tolist()
    assert len(set(used)) == len(used)
    assert slots.tolist() == [int(seqs.table[i, p // 16]) * 16 + p % 16 for i, p in enumerate(pos.tolist())]
    with pytest.raises(ValueError):
        seqs.grow([14, 0, 0])
    assert seqs.kv_len.tolist() == [36, 6, 9]
