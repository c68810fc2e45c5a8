"""Plain forms of the decode step's operators, in Python integers and float64
on the CPU, written from their definitions (include/q3s_decode.h)."""
import numpy as np
import torch


def ceil_div(a, b):
    return -(-a // b)


def cache_tables(context, new, table, ring, state, *, block_size, max_tokens, released=None):
    """Lists in, a dict of numpy arrays out; `table` and `ring` are copied."""
    table, ring = [list(r) for r in table], list(ring)
    old_ring, n = list(ring), len(ring)
    width = len(table[0]) if table else 0
    head, count = state
    gone = list(released) if released is not None else [0] * len(context)
    error, wanted, taken, tail = 0, 0, 0, head + count
    lengths, slots, positions, offsets = [], [], [], [0]
    for b, (c, m) in enumerate(zip(context, new)):  # blocks given back, in row order
        if c < 0 or m < 0 or c > width * block_size:
            error |= 1
        c = min(max(c, 0), width * block_size)
        for j in range(ceil_div(c, block_size) if gone[b] else 0):
            ring[tail % n] = table[b][j]
            tail += 1
    for b, (c, m) in enumerate(zip(context, new)):
        start = 0 if gone[b] else min(max(c, 0), width * block_size)
        m = max(m, 0)
        end = start + m
        need = range(ceil_div(start, block_size), ceil_div(end, block_size))
        ok = end <= width * block_size
        if not ok:
            error |= 2
        else:
            wanted += len(need)
            if len(need) and wanted > count:
                ok, error = False, error | 4
        if ok:
            for k, j in enumerate(need):
                table[b][j] = old_ring[(head + wanted - len(need) + k) % n]
            if len(need):
                taken = wanted
        lengths.append(end if ok else start)
        for p in range(start, end):
            slots.append(table[b][p // block_size] * block_size + p % block_size if ok else -1)
            positions.append(p)
        offsets.append(offsets[-1] + m)
    if len(slots) > max_tokens:
        error |= 8
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    positions = (positions + [0] * max_tokens)[:max_tokens]
    return dict(query_offsets=np.array(offsets, np.int32), slot_map=np.array(slots, np.int64).reshape(-1),
                positions=np.array(positions, np.int32).reshape(-1), lengths=np.array(lengths, np.int32).reshape(-1),
                free_state=np.array([(head + taken) % n, min(count - taken + tail - head - count, n)], np.int32),
                error_word=np.array([error], np.int32), table=np.array(table, np.int32).reshape(len(context), width),
                ring=np.array(ring, np.int32))


def prefix_attention(q, k_cache, v_cache, offsets, table, lengths, prefix_blocks, prefix_length, scale):
    """(out, lse, mass) in float64; mass = sum p |v|, which bounds what
    rounding p to 16 bits can move.  All arguments on the CPU."""
    q = q.double()
    T, Hq, D = q.shape
    H, bs = k_cache.shape[1], k_cache.shape[2]
    out, mass = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -float("inf"), dtype=torch.float64)

    def gather(cache, blocks, n):
        nb = ceil_div(n, bs)
        if nb == 0:
            return torch.zeros(0, H, D, dtype=torch.float64)
        return cache[blocks[:nb].long()].double().transpose(1, 2).reshape(-1, H, D)[:n]

    k0, v0 = gather(k_cache, prefix_blocks, prefix_length), gather(v_cache, prefix_blocks, prefix_length)
    for b in range(len(lengths)):
        n = int(offsets[b + 1] - offsets[b])
        if n <= 0:
            continue
        k1, v1 = (gather(x, table[b], int(lengths[b])) for x in (k_cache, v_cache))
        for i in range(n):
            t = int(offsets[b]) + i
            seen = max(int(lengths[b]) - n + i + 1, 0)
            k, v = torch.cat([k0, k1[:seen]]), torch.cat([v0, v1[:seen]])
            if not len(k):
                continue
            k, v = k.repeat_interleave(Hq // H, 1), v.repeat_interleave(Hq // H, 1)
            s = scale * torch.einsum("hd,lhd->hl", q[t], k)
            lse[t] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            out[t] = torch.einsum("hl,lhd->hd", p, v)
            mass[t] = torch.einsum("hl,lhd->hd", p, v.abs())
    return out, lse, mass


def quantize_rows(x):
    """numpy fp32 [M, K] -> (int8 values, fp32 scales), IEEE 32-bit arithmetic."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.max(np.abs(x), axis=1)
        bad = ~np.isfinite(top)
        tiny = top < np.float32(2.0 ** -100)
        unit = np.where(tiny | bad, np.float32(0), np.float32(127) / np.where(tiny | bad, np.float32(1), top)).astype(np.float32)
        scale = np.where(bad, np.float32(np.nan), np.where(tiny, np.float32(0), top / np.float32(127))).astype(np.float32)
        values = np.where(bad[:, None], 0, np.rint(np.where(np.isfinite(x), x, 0) * unit[:, None]))
    return values.astype(np.int8), scale
