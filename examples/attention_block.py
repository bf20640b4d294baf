"""The attention half of a layer on IQ4_XS weights, from the hidden state to o: prompts of different lengths in one pass,
then tokens one by one for all sequences together, as a captured graph.

    python examples/attention_block.py [--prompts 700,33,2049] [--steps 32] [--cache q8|f16|bf16] [--page 64]

Weights, prompts and gains are synthetic; the layer is the one that bench.py runs, with heads of 128.

    h -> RMS norm -> Q8_1            rms_norm_q8_1
      -> q, k, v                     mul_mat_q8_1_group (one token: rms_norm_mul_mat_group)
      -> head norm, turn, store      qk_norm_rope_append: q in 16 bits, k and v into pages
      -> attention over the pages    paged_attention: fp32 rows
      -> o                           mul_mat
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

pkg = load_package()
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}


def new_cache(pages, heads, page, head, kind, device):
    """Empty pages.  What lies past a sequence's tokens is never looked at, so nothing is cleared."""
    k, v = (torch.empty((pages, heads, page, head), dtype=TYPES[kind], device=device) for _ in range(2))
    if kind != "q8":
        return pkg.KVCache(k, v)
    ks, vs = (torch.empty((pages, heads, page, head // 32), dtype=torch.float16, device=device) for _ in range(2))
    return pkg.KVCache(k, v, ks, vs)


class Sequences:
    """Pages and lengths of a batch.  Each sequence owns pages for `room` tokens from the start; a server would hand them
    out as sequences grow and rewrite the table's rows."""

    def __init__(self, count, room, page, device):
        self.count, self.page, self.device = count, page, device
        self.room = -(-room // page) * page
        width = self.room // page
        self.pages = count * width
        self.table = torch.randperm(self.pages, device=device).to(torch.int32).view(count, width)
        self.kv_len = torch.zeros(count, dtype=torch.int32, device=device)
        self.each = torch.arange(count + 1, dtype=torch.int32, device=device)  # starts of one new token each
        self.rows = torch.arange(count, device=device)
        self.lengths = [0] * count  # on the host, as of the last grow()

    def slots(self, seq, pos):
        """Where tokens go; past the room nowhere, -1, and they are not stored."""
        inside = pos < self.room
        page = self.table[seq, (pos // self.page).clamp(max=self.room // self.page - 1)]
        return torch.where(inside, page.long() * self.page + pos % self.page, -1)

    def grow(self, new):
        """The new tokens of each sequence: (pos, slots, starts), one sequence after another; lengths move on."""
        lengths = [n + m for n, m in zip(self.lengths, new)]
        if len(new) != self.count or max(lengths) > self.room:
            raise ValueError("one count of new tokens for each sequence, within its room")
        new_d = torch.tensor(new, device=self.device)
        starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=self.device)
        seq = self.rows.repeat_interleave(new_d)
        pos = torch.arange(sum(new), device=self.device) - starts[seq] + self.kv_len[seq]
        self.kv_len.add_(new_d.int()).clamp_(max=self.room)
        self.lengths = lengths
        return pos.int(), self.slots(seq, pos), starts

    def step(self):
        """One new token for each sequence, without the host: may be captured.  The caller counts the steps; a sequence
        whose room is full stays as it is, and its new token sees what it holds."""
        pos = self.kv_len.clone()
        self.kv_len.add_(1).clamp_(max=self.room)
        return pos, self.slots(self.rows, pos.long()), self.each


class AttentionBlock:
    """Weights of one layer's attention half: IQ4_XS bytes of q, k, v and o, fp32 gains of the layer and of the heads."""

    def __init__(self, weights, hidden, q_heads, k_heads, head, gain, q_gain, k_gain, freqs, kind, eps=1e-6):
        self.wq, self.wk, self.wv, self.wo = weights
        self.hidden, self.q_heads, self.k_heads, self.head = hidden, q_heads, k_heads, head
        self.gain, self.q_gain, self.k_gain, self.freqs, self.eps = gain, q_gain, k_gain, freqs, eps
        self.q_type = torch.bfloat16 if kind == "bf16" else torch.float16

    def project(self, h):
        """q [tokens, q_heads, head], k and v [tokens, k_heads, head], fp32."""
        m, rows = h.shape[0], [n * self.head for n in (self.q_heads, self.k_heads, self.k_heads)]
        Ws = [self.wq, self.wk, self.wv]
        if m == 1:
            outs = pkg.rms_norm_mul_mat_group(Ws, h, self.hidden, rows, gamma=self.gain, eps=self.eps)
        else:
            ws = pkg.rms_norm_q8_1(h, self.hidden, m, gamma=self.gain, eps=self.eps)
            outs = pkg.mul_mat_q8_1_group(Ws, ws, self.hidden, rows, m)
        return [x.view(m, -1, self.head) for x in outs]

    def attend(self, q, k, v, cache, seqs, where, most_q, most_kv):
        """fp32 rows [tokens, q_heads, head]: the o projection quantises them itself."""
        pos, slots, starts = where
        q = pkg.qk_norm_rope_append(q, k, v, pos, slots, cache, self.freqs, self.q_gain, self.k_gain, self.eps,
                                    out_type=self.q_type)
        return pkg.paged_attention(q, cache, seqs.table, starts, seqs.kv_len, most_q, most_kv, out_type=torch.float32)

    def __call__(self, h, cache, seqs, where, most_q, most_kv):
        out = self.attend(*self.project(h), cache, seqs, where, most_q, most_kv)
        return pkg.mul_mat(self.wo, out, self.q_heads * self.head, self.hidden, h.shape[0])


def synthetic_block(hidden, q_heads, k_heads, head, kind, device, seed=1):
    rows = [q_heads * head, k_heads * head, k_heads * head]
    weights = [pkg.synthetic_weights(hidden, n, seed + i, device=device) for i, n in enumerate(rows)]
    weights.append(pkg.synthetic_weights(rows[0], hidden, seed + 3, device=device))
    g = torch.Generator().manual_seed(seed)
    # the synthetic weights are about 16 each: the gain brings the projections back to about 1
    gain = ((1 + 0.1 * torch.randn(hidden, generator=g)) / (16 * hidden ** 0.5)).to(device)
    q_gain, k_gain = ((1 + 0.1 * torch.randn(head, generator=g)).to(device) for _ in range(2))
    freqs = (1e6 ** (-torch.arange(0, head, 2, dtype=torch.float64) / head)).to(device)
    return AttentionBlock(weights, hidden, q_heads, k_heads, head, gain, q_gain, k_gain, freqs, kind)


def decode_graph(block, cache, seqs, h, most_kv):
    """A step for every sequence as a graph: reads h [sequences, hidden], gives the output that each replay rewrites.
    most_kv is the longest that a sequence may get while the graph is in use."""
    kept = seqs.kv_len.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once outside the graph; its tokens are written again by the first replay
        block(h, cache, seqs, seqs.step(), 1, most_kv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(h, cache, seqs, seqs.step(), 1, most_kv)
    seqs.kv_len.copy_(kept)
    return graph, out


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", default="700,33,2049")
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--cache", choices=list(TYPES), default="q8")
    ap.add_argument("--page", type=int, default=64)
    a = ap.parse_args()
    prompts = [int(n) for n in a.prompts.split(",")]
    device = torch.device("cuda", torch.cuda.current_device())
    hidden, q_heads, k_heads, head = 5120, 64, 8, 128
    block = synthetic_block(hidden, q_heads, k_heads, head, a.cache, device)
    seqs = Sequences(len(prompts), max(prompts) + a.steps, a.page, device)
    cache = new_cache(seqs.pages, k_heads, a.page, head, a.cache, device)

    def clock(fn):
        torch.cuda.synchronize()
        t = time.perf_counter()
        x = fn()
        torch.cuda.synchronize()
        return x, time.perf_counter() - t

    h = pkg.synthetic_activations(sum(prompts) * hidden, 5, device=device).view(-1, hidden)
    out, t = clock(lambda: block(h, cache, seqs, seqs.grow(prompts), max(prompts), max(prompts)))
    print(f"prompts {prompts}: {t * 1e3:.2f} ms with the first call's set-up, |out| {out.abs().mean().item():.4f}")
    h = pkg.synthetic_activations(len(prompts) * hidden, 6, device=device).view(-1, hidden)
    graph, out = decode_graph(block, cache, seqs, h, seqs.room)
    _, t = clock(lambda: [graph.replay() for _ in range(a.steps)])
    print(f"{a.steps} steps of {len(prompts)} sequences: {t / a.steps * 1e6:.1f} us each, lengths "
          f"{seqs.kv_len.tolist()}, |out| {out.abs().mean().item():.4f}")


if __name__ == "__main__":
    main()
