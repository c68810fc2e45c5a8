"""Plain forms of the operators for steps of several tokens a row, in Python
integers and float64 on the CPU, written from their definitions
(include/q3s_decode.h)."""
import math

import numpy as np
import torch


def ceil_div(a, b):
    return -(-a // b)


def rotary_axes(pairs, sections, interleaved):
    """The axis of every pair."""
    if not sections:
        return [0] * pairs
    if interleaved:
        n = len(sections)
        return [i % n if i < n * sections[i % n] else 0 for i in range(pairs)]
    return [a for a, m in enumerate(sections) for _ in range(m)]


def rotary(x, positions, inv_freq, sections=(), interleaved=False, adjacent=False, scale=1.0):
    """(y, size, angle) in float64: y, and per element |x1| + |x2| of its pair and the angle it turned by (0 where copied)."""
    x = x.double().cpu()
    T, _, D = x.shape
    P = inv_freq.numel()
    positions = positions.cpu().reshape(-1, T)
    axis = rotary_axes(P, sections, interleaved)
    y, size, angle = x.clone(), torch.zeros_like(x), torch.zeros_like(x)
    for i in range(P):
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + P)
        # the angle as an exact product of integers and dyadic fractions, then reduced with Python's own floats
        turn = torch.tensor([int(p) * float(inv_freq[i]) for p in positions[axis[i] % len(positions)]], dtype=torch.float64)
        c, s = scale * turn.cos()[:, None], scale * turn.sin()[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        for e in (a, b):
            size[..., e] = (x[..., a].abs() + x[..., b].abs()) * abs(scale)
            angle[..., e] = turn.abs()[:, None]
    return y, size, angle


def cache_trim(lengths, removed, table, ring, state, *, block_size):
    table, ring = [list(r) for r in table], list(ring)
    room, (head, count), error, out = len(table[0]) * block_size if table else 0, state, 0, []
    for b, (n, gone) in enumerate(zip(lengths, removed)):
        had = min(max(n, 0), room)
        cut = min(max(gone, 0), had)
        error |= had != n or cut != gone
        for j in range(ceil_div(had - cut, block_size), ceil_div(had, block_size)):
            if count < len(ring):
                ring[(head + count) % len(ring)] = table[b][j]
            count += 1
        out.append(had - cut)
    if count > len(ring):
        error |= 4
    return dict(lengths=out, ring=ring, free_state=[head, min(count, len(ring))], error_word=[int(error)])


def verify_drafts(logits, ids, offsets, uniforms, probs=None, temperature=None, slot_map=None):
    """Lists; logits fp32 and probs fp32 numpy [T, V], temperature one number a row."""
    T, V = logits.shape
    B = len(offsets) - 1
    tokens, accepted, rejected, fresh, error = [-1] * T, [0] * B, [0] * B, [-1] * B, 0

    def target(t, heat):
        """(p, argmax); p None: no distribution"""
        x = logits[t].astype(np.float64)
        kept = np.where(np.isnan(x), -np.inf, x)
        best = int(np.argmax(kept))
        if np.isnan(x).any() or not np.isfinite(kept[best]):
            return None, best
        if not heat >= 2.0 ** -100:
            p = np.zeros(V)
            p[best] = 1
            return p, best
        p = np.exp((x - x[best]) / float(heat))
        return p / math.fsum(p), best

    for b in range(B):
        t, end = offsets[b], offsets[b + 1]
        if t == end or (slot_map is not None and min(slot_map[t:end]) < 0):
            continue
        start, outside = t, False
        while True:
            p, best = target(t, temperature[b])
            if t + 1 == end:
                rest = p
                break
            d = ids[t + 1]
            outside = not 0 <= d < V
            q = None
            if not outside:
                q = probs[t + 1].astype(np.float64) if probs is not None else np.eye(1, V, d)[0]
                if p is not None and float(uniforms[t + 1]) * q[d] < p[d]:
                    tokens[t] = d
                    t += 1
                    continue
            rest = p
            if p is not None:
                if probs is not None:
                    q = probs[t + 1].astype(np.float64)
                if q is not None:
                    with np.errstate(invalid="ignore"):
                        rest = np.fmax(p - q, 0)
                    if not rest.any():
                        rest = p
            break
        if p is None:
            tokens[t] = best
        elif not temperature[b] >= 2.0 ** -100:
            tokens[t] = best
        else:
            edges = np.cumsum(rest)
            over = np.flatnonzero(edges > float(uniforms[start]) * edges[-1])
            tokens[t] = int(over[0]) if over.size else int(np.flatnonzero(rest)[-1])
        if p is None or outside:
            error |= 64
        accepted[b], rejected[b], fresh[b] = t - start, end - 1 - t, tokens[t]
    return dict(tokens=tokens, accepted=accepted, rejected=rejected, next_ids=fresh, error=error)


def chunk_attention(q, k_cache, v_cache, offsets, table, lengths, prefix_blocks, prefix_length, scale, window=0, slot_map=None):
    """(out, lse, spread, mass) in float64 on the tensors' device: spread = sum p |v - out|, which bounds what rounding p
    moves where out is divided by the sum of the rounded p, and mass = sum p |v|."""
    T, Hq, D = q.shape
    H, bs = k_cache.shape[1], k_cache.shape[2]
    G = Hq // H
    zero = dict(dtype=torch.float64, device=q.device)
    out, spread, mass = (torch.zeros(T, Hq, D, **zero) for _ in range(3))
    lse = torch.full((T, Hq), -math.inf, **zero)

    def gather(cache, blocks, n):
        nb = ceil_div(n, bs)
        return cache[blocks[:nb].long()].double().transpose(1, 2).reshape(-1, H, D)[:n]

    for b in range(len(lengths)):
        t0, t1, length = int(offsets[b]), int(offsets[b + 1]), int(lengths[b])
        n = t1 - t0
        if n <= 0:
            continue
        k, v = (torch.cat([gather(x, prefix_blocks, prefix_length), gather(x, table[b], length)]) for x in (k_cache, v_cache))
        key = torch.arange(len(k), device=q.device)
        own = length - n + torch.arange(n, device=q.device) + 1  # own tokens that each query sees
        pos = prefix_length + own - 1
        seen = (key < prefix_length) | (key - prefix_length < own[:, None])
        if window:
            seen &= key > pos[:, None] - window
        if slot_map is not None:
            seen &= (slot_map[t0:t1] >= 0)[:, None]
        for h in range(Hq):
            s = torch.where(seen, scale * (q[t0:t1, h].double() @ k[:, h // G].t()), -math.inf)
            any_key = seen.any(1)
            p = torch.where(any_key[:, None], torch.softmax(s, 1), 0.0)
            lse[t0:t1, h] = torch.logsumexp(s, 1)
            vh = torch.where(seen.any(0)[:, None], v[:, h // G], 0.0)  # what nobody sees counts for nothing
            o = p @ vh
            out[t0:t1, h] = o
            mass[t0:t1, h] = p @ vh.abs()
            for c in range(0, n, 16):
                spread[t0 + c:min(t0 + c + 16, t1), h] = torch.einsum("nk,nkd->nd", p[c:c + 16], (vh[None] - o[c:c + 16, None]).abs())
    return out, lse, spread, mass
