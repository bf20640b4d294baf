"""The attention half of a layer in 64 bits, from the formulas, for the tests.  Works on the CPU."""
import math

import torch


def frequencies(rot, base=1e6):
    return base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))


def norm_rope(x, pos, freqs, gamma, eps, half):
    """[tokens][heads][d] in 64 bits."""
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if gamma is not None:
        x = x * gamma.double()
    if freqs is None or not freqs.numel():
        return x
    n = freqs.numel()
    t = (pos.double()[:, None] * freqs.double())[:, None]
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    u, w = a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()
    y = torch.cat([u, w], -1) if half else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * n:]], -1)


def codes(x):
    """8-bit codes and fp16 scales of groups of 32 channels, as the cache's format defines them, in fp32."""
    v = x.float().unflatten(-1, (-1, 32))
    d = (v.abs().amax(-1) / 127).clamp(max=65504 / 127).half()
    q = torch.where(d[..., None] > 0, v / d[..., None].float(), torch.zeros_like(v)).round().clamp(-127, 127)
    return q.flatten(-2).to(torch.int8), d


def stored(pages, scales):
    """What a cache's pages stand for, in 64 bits."""
    if scales is None:
        return pages.double()
    return pages.double() * scales.double().repeat_interleave(32, -1)


def sequence_rows(pages, scales, table_row, n):
    """Tokens [n][heads][d] of a sequence; NaN where the page is not in the cache."""
    count, heads, page, d = pages.shape
    out = torch.full((n, heads, d), math.nan, dtype=torch.float64)
    ok = torch.zeros(n, dtype=torch.bool)
    for j in range(0, n, page):
        i = int(table_row[j // page]) if j // page < table_row.numel() else -1
        if 0 <= i < count:
            m = min(page, n - j)
            out[j:j + m] = stored(pages[i], None if scales is None else scales[i])[:, :m].transpose(0, 1)
            ok[j:j + m] = True
    return out, ok


def attention(q, k_pages, v_pages, k_scales, v_scales, table, starts, kv_len, causal, window, scale):
    """Row by row over the keys that the row sees, in 64 bits: out, lse, the same mean of the values' magnitudes, and the
    largest sum of a score's terms' magnitudes (what roundings are relative to).  A key that is not seen is not read."""
    heads, group, d = k_pages.shape[1], q.shape[1] // k_pages.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    size, terms = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(kv_len.numel()):
        n, first, end = int(kv_len[s]), int(starts[s]), int(starts[s + 1])
        k, ok = sequence_rows(k_pages, k_scales, table[s], n)
        v, _ = sequence_rows(v_pages, v_scales, table[s], n)
        for i in range(end - first):
            p = n - (end - first) + i
            hi = min(n, p + 1) if causal else n
            lo = max(0, p + 1 - window) if window else 0
            at = [j for j in range(lo, max(lo, hi)) if ok[j]]
            if not at:
                continue
            row = q[first + i].double().view(heads, group, d)
            z = torch.einsum("hgd,nhd->hgn", row, k[at]) * scale
            most = torch.einsum("hgd,nhd->hgn", row.abs(), k[at].abs()).amax(-1) * abs(scale)
            top = z.amax(-1, keepdim=True)
            w = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = w.sum(-1, keepdim=True)
            o = torch.einsum("hgn,nhd->hgd", w, v[at])
            out[first + i] = torch.where(total == 0, torch.zeros_like(o), o / total).reshape(-1, d)
            lse[first + i] = (top + total.log()).reshape(-1)
            size[first + i] = (torch.einsum("hgn,nhd->hgd", w, v[at].abs()) / total.clamp(min=1e-300)).reshape(-1, d)
            terms[first + i] = most.reshape(-1)
    return out, lse, size, terms
