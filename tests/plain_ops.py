"""Plain 64-bit implementations of the windowed, cached and positional operators, with elementwise error bounds.

A bound counts the roundings that the kernels make: u = half a step of the 16-bit type for each value that is rounded to
it, and for the 32-bit parts ``gamma`` = D * 2^-23 times the sum of the absolute products of a dot product (an
accumulator may truncate) plus 2^-18 for the approximate exp2 / log2 and the sums.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(Sq, Sk, window, sinks, length):
    """[Sq, Sk] bool."""
    p = torch.arange(Sq)[:, None] + Sk - Sq
    j = torch.arange(Sk)[None]
    return (p >= 0) & (p < length) & (j <= p) & ((j > p - window) | (j < sinks))


def attend(q, k, v, mask, scale, dtype):
    """q [B,Hq,S,D], k/v [B,Hkv,n,D] (64 bits), mask [B,S,n] -> out, lse and their bounds for a kernel of type dtype."""
    G = q.shape[1] // k.shape[1]
    if mask.shape[-1] == 0:  # no key at all: one that nobody sees
        k = v = q.new_zeros(q.shape[0], k.shape[1], 1, q.shape[-1])
        mask = mask.new_zeros(*mask.shape[:2], 1)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    m = mask[:, None]
    # what is not visible takes no part, whatever it holds
    unseen = ~mask.any(1)[:, None, :, None]
    k, v = k.masked_fill(unseen, 0.0), v.masked_fill(unseen, 0.0)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).masked_fill(~m, 0.0)
    out = p @ v
    u, D = half_step(dtype), q.shape[-1]
    dot = ((q.abs() @ k.abs().transpose(-1, -2)) * scale).masked_fill(~m, 0.0).amax(-1)
    d = D * 2.0 ** -23 * dot + 2.0 ** -18  # relative error of a probability, absolute one of a score
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # step of the smallest halves, next to the row's largest P of 1
    spread = p @ v.abs()
    tol = (u + 2 * d[..., None]) * spread + u * out.abs() + tiny * (m.double() @ v.abs()) + 1e-30
    lse_tol = 2 * d + 2.0 ** -21 * lse.abs().masked_fill(lse == -math.inf, 0.0)
    return out, lse, tol, lse_tol, p, d


def gradients(q, k, v, dout, mask, scale, dtype, out_tol=None):
    """64-bit dq, dk, dv and their bounds (for kernels that take the 16-bit `out` of a forward kernel)."""
    B, Hq, S, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    out, lse, tol, _, p, d = attend(q, k, v, mask, scale, dtype)
    ke, ve = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    dead = (lse == -math.inf)[..., None]
    unseen = ~mask.any(1)[:, None, :, None]
    ke, ve = ke.masked_fill(unseen, 0.0), ve.masked_fill(unseen, 0.0)
    q, dout = q.masked_fill(dead, 0.0), dout.masked_fill(dead, 0.0)
    dp = dout @ ve.transpose(-1, -2)
    delta = (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    u = half_step(dtype)
    rel = 2 * d[..., None]
    # dS: its rounding and P's error, the dot product dO V, and delta from the rounded out
    d_delta = (tol * dout.abs()).sum(-1, keepdim=True) + 2.0 ** -18 * (out * dout).abs().sum(-1, keepdim=True)
    ds_tol = p * ((u + rel) * (dp - delta).abs() + D * 2.0 ** -23 * (dout.abs() @ ve.abs().transpose(-1, -2)) + d_delta)
    p_tol = p * (u + rel)
    if dtype == torch.float16:
        ds_tol, p_tol = ds_tol + 2.0 ** -25 * mask[:, None], p_tol + 2.0 ** -25 * mask[:, None]

    def shared(x):
        return x.view(B, Hkv, G, *x.shape[2:]).sum(2)

    dq = scale * ds @ ke
    dk, dv = scale * shared(ds.transpose(-1, -2) @ q), shared(p.transpose(-1, -2) @ dout)
    n = mask.shape[1] * 2.0 ** -24 * G  # fp32 sums
    dq_tol = scale * (ds_tol + 2.0 ** -14 * ds.abs()) @ ke.abs() + u * dq.abs() + 1e-30
    dk_tol = scale * shared((ds_tol + n * ds.abs()).transpose(-1, -2) @ q.abs()) + u * dk.abs() + 1e-30
    dv_tol = shared((p_tol + n * p).transpose(-1, -2) @ dout.abs()) + u * dv.abs() + 1e-30
    if dtype == torch.float16:  # results among the smallest halves
        dq_tol, dk_tol, dv_tol = dq_tol + 2.0 ** -25, dk_tol + 2.0 ** -25, dv_tol + 2.0 ** -25
    return (dq, dk, dv), (dq_tol, dk_tol, dv_tol)


def assert_within(got, ref, tol, what):
    got = got.double().cpu()
    assert got.shape == ref.shape, what
    both_inf = torch.isinf(ref) & (got == ref)
    bad = ~(((got - ref).abs() <= tol) | both_inf)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, first at "
                           f"{tuple(bad.nonzero()[0].tolist())}: {got[bad][0].item()} against {ref[bad][0].item()} "
                           f"+- {tol.expand_as(ref)[bad][0].item()}")


def assert_close_norm(got, ref, bound, what):
    """Rounding errors of independent values: the 2-norm of the difference, relative to the result's."""
    got = got.double().cpu()
    off = (got - ref).norm().item() / max(ref.norm().item(), 1e-300)
    assert off <= bound, f"{what}: relative 2-norm {off:.3g} > {bound:.3g}"


def ancestors(parents):
    """Lists of the drafts each draft sees (itself last), None for unused slots."""
    chains = []
    for t, up in enumerate(parents):
        if up == -1:
            chains.append([t])
        elif 0 <= up < t and chains[up] is not None:
            chains.append(chains[up] + [t])
        else:
            chains.append(None)
    return chains


def cached_visible(T, length, window, sinks, parents=None):
    """[T, length] bool for one sequence of `length` tokens whose last T are the new ones."""
    base = length - T
    rank = list(range(length))  # position of each key's text
    at = [base + t for t in range(T)]
    if parents is None:
        chains = [list(range(t + 1)) for t in range(T)]
    else:
        chains = [None if c is None else [u for u in c if base + u >= 0] or None for c in ancestors(parents)]
        for t, c in enumerate(chains):
            if c is not None:
                at[t] = base + len(c) - 1
                if base + t >= 0:
                    rank[base + t] = at[t]
    seen = torch.zeros(T, max(length, 0), dtype=torch.bool)
    for t, c in enumerate(chains):
        if c is None or (parents is None and at[t] < 0):
            continue
        keys = list(range(max(base, 0))) + [base + u for u in c if base + u >= 0]
        for j in keys:
            seen[t, j] = rank[j] > at[t] - window or rank[j] < sinks
    return seen


def rotate(x, positions, inv_freq, axis_pairs, interleaved, inverse=False):
    """x [B,H,S,D] 64 bits, positions [B,S,A]."""
    P = sum(axis_pairs)
    axis = torch.repeat_interleave(torch.arange(len(axis_pairs)), torch.tensor(axis_pairs))
    angle = positions[..., axis].double() * inv_freq.double()
    if inverse:
        angle = -angle
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    out = x.clone()
    a, b = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    # one rounding, and the 32-bit sines (2^-22 of a turn's amplitude) and products
    size = torch.zeros_like(x)
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, size
