"""Linear attention with a decay for each head in 64 bits, token by token from its definition, and what fp32 sums may be
off by.  Works on the CPU."""
import torch

U = 2.0 ** -24


def linear(q, k, v, decay, starts, most_q=None, states=None, from_slots=None, to_slots=None, scale=1.0):
    """out, its bound, states, their bound.

    With sums of magnitudes M_t = a M + |k| |v|^T in the state's place: a token's step rounds the decay (exp's two halves of
    a step), its product and the sum, 4 U M_t at most, and what earlier steps were off by decays with the state: E_t = a E +
    4 U M_t.  A chunk of up to 64 tokens instead rounds once for each of them (sums of 64 and of the parts of a product),
    and its weights' exponents (below 2^7, half a step each): 224 U M_t for the states at most.  An output adds a sum of dk
    terms: scale |q| (E + (dk + 224) U M)."""
    total, heads, dv = v.shape
    group, dk = heads // q.shape[1], q.shape[2]
    q, k = (x.double().repeat_interleave(group, 1) for x in (q, k))
    v = v.double()
    a = decay.double().exp().expand(total, heads)
    out = torch.zeros(total, heads, dv, dtype=torch.float64, device=v.device)
    tol = torch.zeros_like(out)
    new = None if states is None else states.double()
    err = None if states is None else torch.zeros_like(new)
    for s in range(starts.numel() - 1):
        first, n = int(starts[s]), int(starts[s + 1]) - int(starts[s])
        n = n if most_q is None else min(n, most_q)
        if n <= 0:
            continue
        S = torch.zeros(heads, dk, dv, dtype=torch.float64, device=v.device)
        if from_slots is not None and 0 <= int(from_slots[s]) < states.shape[0]:
            S = states[int(from_slots[s])].double()
        M, E = S.abs(), torch.zeros_like(S)
        for t in range(first, first + n):
            S = S * a[t, :, None, None] + k[t, :, :, None] * v[t, :, None, :]
            M = M * a[t, :, None, None] + k[t, :, :, None].abs() * v[t, :, None, :].abs()
            E = E * a[t, :, None, None] + 4 * U * M
            out[t] = scale * torch.einsum("hd,hdc->hc", q[t], S)
            tol[t] = abs(scale) * torch.einsum("hd,hdc->hc", q[t].abs(), E + (dk + 224) * U * M)
        if to_slots is not None and 0 <= int(to_slots[s]) < states.shape[0]:
            new[int(to_slots[s])] = S
            err[int(to_slots[s])] = E + 224 * U * M
    return out, tol, new, err


def sizes(tol, dk):
    """Magnitudes of an output's terms, from the smallest that its bound can come from."""
    return tol / ((dk + 224) * U)


def compare(got, states, want):
    """16-bit outputs: what makes them keeps 16 bits of both factors of a product (2^-15 of its terms' magnitudes in all),
    and they are rounded once."""
    out, tol, new, err = want[:4]
    dk = want[4]
    half = torch.finfo(got.dtype).eps / 2
    if got.dtype != torch.float32:
        tol = tol + 2.0 ** -15 * sizes(tol, dk)
    tol = tol + half * (out.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
    e = (got.double() - out).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((e <= tol).all()), ((e - tol).max().item(), (e / tol).max().item())
    if new is not None:
        e = (states.double() - new).abs()
        assert bool((e <= err + 2.0 ** -126).all()), ((e - err).max().item(), (e / err.clamp(min=1e-300)).max().item())
