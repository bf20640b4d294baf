"""A batch of requests behind one system prompt, through a layer with a window and first tokens, one that sees everything and
shares the prompt's pages, and one that keeps a state: the prompt, the questions, then tokens from a replayed graph.  What
each layer was given is kept, and its outputs are held to 64 bits over the whole history."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_more_reference as more  # noqa: E402
import linear_reference  # noqa: E402

pytestmark = pytest.mark.gpu

HQ, HK, D, PAGE, WINDOW, SINKS = 8, 2, 64, 16, 24, 4
PROMPT, ASKED, STEPS = 70, [5, 40, 1], 6


class History:
    """What tests/attention_more_reference.py looks at, gathered from the cache at the end."""

    def __init__(self, cache, table, kv, new, q):
        self.k, self.v, self.ks, self.vs = cache.k_pages.cpu(), cache.v_pages.cpu(), None, None
        self.table, self.kv, self.new, self.cache, self.q_type = table.cpu(), kv, new, "f16", torch.float16
        self.kv_len = torch.tensor(kv, dtype=torch.int32)
        self.starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
        self.q, self.scale = q.cpu(), D ** -0.5


class Batch:
    def __init__(self, pkg, dev):
        self.pkg, self.dev, self.n = pkg, dev, len(ASKED)
        self.gen = torch.Generator(device=dev).manual_seed(8)
        width = -(-(PROMPT + max(ASKED) + STEPS) // PAGE)
        common, left = PROMPT // PAGE, width - PROMPT // PAGE
        pages = common + self.n * left
        order = torch.randperm(pages, device=dev, generator=self.gen).to(torch.int32)
        self.table = torch.empty(self.n, width, dtype=torch.int32, device=dev)
        self.table[:, :common] = order[:common]
        self.table[:, common:] = order[common:].view(self.n, left)
        new = lambda: torch.empty(pages, HK, PAGE, D, dtype=torch.float16, device=dev)  # noqa: E731
        self.windowed, self.full = pkg.KVCache(new(), new()), pkg.KVCache(new(), new())
        self.states = torch.zeros(self.n + 1, HQ, D, D, device=dev)
        self.freqs = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        self.decay = -torch.exp(torch.linspace(-1, -6, HQ, device=dev))
        self.shared = torch.tensor([PROMPT], dtype=torch.int32, device=dev)
        self.kv_len = torch.zeros(self.n, dtype=torch.int32, device=dev)
        self.each = torch.arange(self.n + 1, dtype=torch.int32, device=dev)
        self.own = torch.arange(1, self.n + 1, device=dev)
        self.seen = []

    def random(self, tokens):
        """q, k and v of each layer, as projections leave them."""
        rnd = lambda h: torch.randn(tokens, h, D, device=self.dev, generator=self.gen)  # noqa: E731
        return [(rnd(HQ), rnd(HK), rnd(HK)) for _ in range(2)] + [(rnd(HK) / 8, rnd(HK) / 8, rnd(HQ))]

    def slots(self, seq, pos):
        return self.table[seq, (pos // PAGE).long()].long() * PAGE + pos % PAGE

    def layers(self, x, pos, slots, starts, most_q, most_own, src, dst, prompt=False):
        pkg, t = self.pkg, self.table[:1] if prompt else self.table
        turn = dict(freqs=self.freqs, out_type=torch.float16)
        kv_len = self.kv_len[:1] if prompt else self.kv_len
        q0 = pkg.qk_norm_rope_append(*x[0], pos, slots, self.windowed, **turn)
        a = pkg.paged_attention(q0, self.windowed, t, starts, kv_len, most_q, PROMPT + most_own, window=WINDOW, sinks=SINKS,
                                lse=True)
        q1 = pkg.qk_norm_rope_append(*x[1], pos, slots, self.full, **turn)
        if prompt:
            b = pkg.paged_attention(q1, self.full, t, starts, kv_len, most_q, PROMPT, lse=True)
        else:
            b = pkg.shared_attention(q1, self.full, t, starts, kv_len, self.shared, most_q, most_own, PROMPT, lse=True,
                                     path=pkg.SHARED_ONCE)
        c = pkg.linear_attention(*x[2], self.decay, starts, most_q, self.states, src, dst)
        return [q0, *a, q1, *b, c]


def test_prompt_questions_and_steps_of_a_graph(pkg):
    dev = torch.device("cuda:0")
    torch.cuda.set_device(0)
    batch, i64 = Batch(pkg, dev), lambda *v: torch.tensor(v, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    # the prompt once, its state to slot 0; its last page's tokens to every sequence's own page
    x = batch.random(PROMPT)
    pos = torch.arange(PROMPT, dtype=torch.int32, device=dev)
    batch.kv_len.fill_(PROMPT)
    got = [batch.layers(x, pos, batch.slots(0, pos), i32(0, PROMPT), PROMPT, 0, i64(-1), i64(0), prompt=True)]
    inputs = [[[t] for t in x[2]]]
    for cache in (batch.windowed, batch.full):
        for pages in (cache.k_pages, cache.v_pages):
            last = PROMPT // PAGE
            pages[batch.table[1:, last].long(), :, :PROMPT % PAGE] = \
                pages[batch.table[0, last].long(), :, :PROMPT % PAGE].clone()
    # the questions, each from the prompt's state
    total, starts = sum(ASKED), i32(*[sum(ASKED[:i]) for i in range(len(ASKED) + 1)])
    seq = torch.repeat_interleave(torch.arange(len(ASKED), device=dev), i64(*ASKED))
    pos = torch.cat([PROMPT + torch.arange(n, dtype=torch.int32, device=dev) for n in ASKED])
    batch.kv_len.copy_(i32(*[PROMPT + n for n in ASKED]))
    y = batch.random(total)
    got.append(batch.layers(y, pos, batch.slots(seq, pos), starts, max(ASKED), max(ASKED), i64(0, 0, 0), batch.own))
    # steps: captured once, then replayed with the tokens in place
    z = batch.random(batch.n)
    most_own = max(ASKED) + STEPS

    def step():
        batch.kv_len += 1
        at = batch.kv_len - 1
        return batch.layers(z, at, batch.slots(torch.arange(batch.n, device=dev), at), batch.each, 1, most_own, batch.own,
                            batch.own)

    lens, states = batch.kv_len.clone(), batch.states.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
        batch.kv_len.copy_(lens)
        batch.states.copy_(states)
        steps = []
        for _ in range(STEPS):
            for kept, fresh in zip(z, batch.random(batch.n)):
                for a, b in zip(kept, fresh):
                    a.copy_(b)
            before = batch.states.clone()
            graph.replay()
            side.synchronize()
            steps.append(([t.clone() for t in z[2]], [t.clone() for t in outs]))
            after = batch.states.clone()
            batch.kv_len -= 1
            batch.states.copy_(before)
            for a, b in zip(steps[-1][1], step()):
                assert torch.equal(a, b)
            assert torch.equal(batch.states, after)
    torch.cuda.current_stream().wait_stream(side)
    # attention over each sequence's whole history: queries of the prompt (sequence 0), the questions and the steps
    asked = [sum(ASKED[:i]) for i in range(len(ASKED) + 1)]
    for first, cache, sees in ((0, batch.windowed, more.window_and_sinks(True, WINDOW, SINKS)),
                               (3, batch.full, more.window_and_sinks(True, 0, 0))):
        for s in range(batch.n):
            part = [torch.cat([*([got[0][first + j]] if s == 0 else []), got[1][first + j][asked[s]:asked[s + 1]],
                               *[o[first + j][s:s + 1] for _, o in steps]]) for j in range(3)]
            n = PROMPT + ASKED[s] + STEPS
            h = History(cache, batch.table[s:s + 1], [n], [part[0].shape[0]], part[0])
            more.compare(h, part[1].cpu(), part[2].cpu(), sees)
    # the state of each sequence over the prompt, its question and its steps
    for s in range(batch.n):
        q, k, v = (torch.cat([inputs[0][j][0], y[2][j][asked[s]:asked[s + 1]], *[t[j][s:s + 1] for t, _ in steps]])
                   for j in range(3))
        n = PROMPT + ASKED[s] + STEPS
        want = linear_reference.linear(q, k, v, batch.decay, i32(0, n), None, torch.zeros_like(batch.states[:1]), i64(-1),
                                       i64(0))
        out = torch.cat([got[0][6], got[1][6][asked[s]:asked[s + 1]], *[o[6][s:s + 1] for _, o in steps]])
        linear_reference.compare(out, batch.states[s + 1:s + 2], (*want, D))
    assert math.isfinite(float(batch.states.abs().sum()))
