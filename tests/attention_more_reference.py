"""Attention over a paged cache in 64 bits for any choice of seen keys, and what fp32 statistics and 16-bit weights may
be off by.  Works on the CPU."""
import math

import torch

import attention_reference as ref


def attention(p, sees):
    """p: test_gpu_attention.Problem; sees(sequence, places [rows, 1], keys [1, n]) -> bool.  out, lse, the same mean of the
    values' magnitudes, and the largest sum of a score's terms' magnitudes.  Keys that are not seen are not read."""
    heads, d = p.k.shape[1], p.q.shape[2]
    group = p.q.shape[1] // heads
    out = torch.zeros(p.q.shape, dtype=torch.float64)
    lse = torch.full(p.q.shape[:2], -math.inf, dtype=torch.float64)
    size, terms = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(len(p.kv)):
        n, first, end = int(p.kv_len[s]), int(p.starts[s]), int(p.starts[s + 1])
        if end <= first or n <= 0:
            continue
        k, ok = ref.sequence_rows(p.k, p.ks, p.table[s], n)
        v, _ = ref.sequence_rows(p.v, p.vs, p.table[s], n)
        place = n - (end - first) + torch.arange(end - first)[:, None]
        mask = sees(s, place, torch.arange(n)[None]) & ok  # [rows, n]
        used = mask.any(0)
        k, v, mask = k[used], v[used], mask[:, used]
        row = p.q[first:end].double().view(end - first, heads, group, d)
        for h in range(heads):
            r = row[:, h].reshape(-1, d)
            m = mask.repeat_interleave(group, 0)
            z = (r @ k[:, h].t() * p.scale).masked_fill(~m, -math.inf)
            some = m.any(1)
            top = z.amax(1, keepdim=True) if z.shape[1] else torch.full((r.shape[0], 1), -math.inf, dtype=z.dtype)
            w = torch.exp(z - torch.where(top == -math.inf, 0.0, top)).masked_fill(~m, 0)
            total = w.sum(1, keepdim=True)
            scale = torch.where(some[:, None], total, 1.0)
            at = (slice(first, end), slice(h * group, (h + 1) * group))
            out[at] = (w @ v[:, h] / scale).view(-1, group, d)
            size[at] = (w @ v[:, h].abs() / scale).view(-1, group, d)
            lse[at] = torch.where(some, (top + total.log()).squeeze(1), -math.inf).view(-1, group)
            t = (r.abs() @ k[:, h].abs().t()).masked_fill(~m, 0)
            terms[at] = (t.amax(1) if t.shape[1] else torch.zeros(r.shape[0])).view(-1, group) * abs(p.scale)
    return out, lse, size, terms


def compare(p, got, lse, sees):
    """As tests/test_gpu_attention.py derives it: weights are rounded to 16 bits (half a step u), values of an 8-bit cache
    and, of many rows, its keys to fp16, scores are sums of head terms in fp32, exp2 and log2 add 2^-20, and the output is
    rounded once; fp16 weights below its normal range are off by 2^-25 of the largest each.

    With weights w (1 + e), |e| <= u, in the sum of products and in the sum that divides it, o = sum w v / sum w moves by
    sum w e (v - o) / sum w (1 + e), to first order at most u (sum w |v - o| / sum w) <= u (size + |o|): where one of two
    keys has nearly all of the weight and a small value, |v - o| is as large as 2 |v| of the other.  The rounding of the
    output is of the moved value."""
    want, want_lse, size, terms = attention(p, sees)
    d = p.q.shape[-1]
    u = 2.0 ** -8 if p.q_type == torch.bfloat16 and p.cache != "q8" else 2.0 ** -11
    score = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -20
    values = u + (2.0 ** -11 + 127 * 2.0 ** -25 if p.cache == "q8" else 0)
    if p.cache == "q8":
        score = score + 2.0 ** -11 * terms
    tail = max(p.kv + [1]) * 2.0 ** -25 * ref.stored(p.v, p.vs).abs().nan_to_num(posinf=0).max()
    tol = size * (values + 2 * score[..., None]) + u * want.abs() + tail
    tol = tol * (1 + 2 * u) + torch.finfo(got.dtype).eps / 2 * (want.abs() + tol)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol).all()), ((err - tol).max().item(), (err / tol).max().item())
    none = want_lse == -math.inf
    assert bool((lse[none] == -math.inf).all()) and bool((got[none] == 0).all())
    e = (lse.double() - want_lse)[~none].abs()
    assert bool((e <= score[~none] + 2.0 ** -22 * want_lse[~none].abs()).all()), e.max().item()


def window_and_sinks(causal, window, sinks):
    def sees(_, place, key):
        seen = (key <= place) if causal else torch.ones(place.shape[0], key.shape[1], dtype=torch.bool)
        return seen & ((key > place - window) | (key < sinks)) if window else seen

    return sees


def share(p, firsts, lens):
    """Makes the sequences of each group begin with the same tokens: whole pages the same, what is left of a page copied."""
    page = p.k.shape[2]
    for g, n in enumerate(lens):
        a = firsts[g]
        for i in range(firsts[g] + 1, firsts[g + 1]):
            whole = n // page
            p.table[i, :whole] = p.table[a, :whole]
            if n % page:
                x, y = int(p.table[a, whole]), int(p.table[i, whole])
                for t in (p.k, p.v, p.ks, p.vs):
                    if t is not None:
                        t[y, :, :n % page] = t[x, :, :n % page]
    return p
