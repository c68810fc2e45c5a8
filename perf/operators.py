"""Measured passes through the decode step's operators beside the sampler.

Four operators, each as a decode engine calls it once per step (or per layer of a step):

* ``tables``     block tables, slot map and positions of a paged key/value cache, built on the GPU from the requests'
                 lengths (``q3s.cache_tables``);
* ``append``     the step's new keys and values written through the slot map (``q3s.cache_append``);
* ``attention``  attention of the batch over one shared prefix and each row's own cached tokens
                 (``q3s.prefix_attention``);
* ``linear``     activations quantised to 8 bits per token and multiplied with an 8-bit weight that has a scale per
                 output channel (``q3s.int8_linear``).

``own`` chooses between the plain form below (elementary torch operations, 32-bit arithmetic) and the package's kernels.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_package = None


def _q3s():
    global _package
    if _package is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3tts-streaming_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import q3s

        _package = q3s
    return _package


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a handful of live streams, one new token each: the latency of the step's first launch
        dict(name="tables 8 rows", op="tables", rows=8, context=700, chunk=1, prefill=0.0, released=0.0, block=16, idle=0.0),
        # a full serving batch where some rows decode, some prefill a chunk, some have just ended
        dict(name="tables 1500 rows mixed", op="tables", rows=1500, context=2000, chunk=512, prefill=0.25, released=0.05, block=32, idle=0.1),
        # one layer's append for a small decode batch
        dict(name="append 8 tokens", op="append", tokens=8, kv_heads=8, dim=128, block=16, skipped=0.0, dtype="bf16"),
        # one layer's append for prefill chunks, sliced out of a fused projection, some tokens without a slot
        dict(name="append 12289 tokens f16", op="append", tokens=12289, kv_heads=8, dim=128, block=32, skipped=0.02, dtype="f16"),
        # a single voice stream behind its speaker prompt
        dict(name="attend 1 row", op="attention", rows=1, q_heads=16, kv_heads=8, dim=128, prefix=600, own=150, queries=1, block=16, dtype="bf16"),
        # an ordinary serving batch on one voice
        dict(name="attend 96 rows", op="attention", rows=96, q_heads=16, kv_heads=8, dim=128, prefix=1500, own=500, queries=1, block=16, dtype="bf16"),
        # long streams: the rows' own caches dominate
        dict(name="attend 61 long rows f16", op="attention", rows=61, q_heads=16, kv_heads=2, dim=64, prefix=333, own=6000, queries=1, block=64, dtype="f16"),
        # several queries a row (draft tokens, short text chunks), ragged, with idle rows
        dict(name="attend 40 ragged rows", op="attention", rows=40, q_heads=32, kv_heads=8, dim=128, prefix=2049, own=900, queries=9, block=32, dtype="bf16"),
        # a large batch behind a long instruction: the shared prefix dominates
        dict(name="attend 256 rows long prefix", op="attention", rows=256, q_heads=32, kv_heads=8, dim=128, prefix=16000, own=200, queries=1, block=16, dtype="bf16"),
        # one token through a square projection
        dict(name="linear 1 x 2048 x 2048", op="linear", tokens=1, inputs=2048, outputs=2048, dtype="bf16"),
        # a decode batch through an up projection of odd width
        dict(name="linear 130 x 2048 x 5000", op="linear", tokens=130, inputs=2048, outputs=5000, dtype="f16"),
        # prefill through an up projection
        dict(name="linear 8192 x 2048 x 8192", op="linear", tokens=8192, inputs=2048, outputs=8192, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "linear"])
    if op == "tables":
        return dict(op=op, rows=_log(rng, 1, 4000), context=_log(rng, 1, 4000), chunk=_log(rng, 1, 512),
                    prefill=rng.choice([0.0, 0.1, 0.25]), released=rng.choice([0.0, 0.03, 0.1]),
                    block=rng.choice([16, 32, 64]), idle=rng.choice([0.0, 0.2]))
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 12000), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                    block=rng.choice([16, 32, 64]), skipped=rng.choice([0.0, 0.02, 0.2]), dtype=rng.choice(["bf16", "f16"]))
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        rows = _log(rng, 1, 256)
        queries = rng.choice([1, 1, 1, 2, 5, 12])
        prefix = rng.choice([0, 1]) * _log(rng, 1, 250) if rng.random() < 0.2 else _log(rng, 16, 16000)
        limit = 256 * 32 * 16000 // (rows * queries * kv * group)  # scores of the largest listed case
        return dict(op=op, rows=rows, q_heads=kv * group, kv_heads=kv, dim=rng.choice([64, 128]),
                    prefix=min(prefix, limit), own=min(_log(rng, 1, 6000), 366000 // rows, limit), queries=queries,
                    block=rng.choice([16, 32, 64]), dtype=rng.choice(["bf16", "f16"]))
    return dict(op=op, tokens=_log(rng, 1, 8000), inputs=16 * _log(rng, 4, 128), outputs=_log(rng, 32, 8000),
                dtype=rng.choice(["bf16", "f16", "f32"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"tables": _prepare_tables, "append": _prepare_append, "attention": _prepare_attention,
            "linear": _prepare_linear}[case["op"]](case, rng, gen)


def _ints(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _ceil(a, b):
    return -(-a // b)


def _table_rows(c):
    """The rows of a tables case before they are put in order: context lengths, new tokens and which have ended."""
    B = c["rows"]
    ended, idle, chunks = int(B * c["released"]), int(B * c["idle"]), int(B * c["prefill"])
    new = np.ones(B, np.int64)
    new[:ended + idle] = 0
    new[B - chunks:] = np.linspace(1, c["chunk"], chunks).astype(np.int64)
    return np.linspace(0, 2 * c["context"], B).astype(np.int64), new, np.arange(B) < ended


def _prepare_tables(c, rng, gen):
    B, bs = c["rows"], c["block"]
    context, new, released = _table_rows(c)
    pool = int(_ceil(context, bs).sum() + _ceil(new, bs).sum()) + B  # a pool with room to spare
    context = context[rng.permutation(B)]
    order = rng.permutation(B)
    new, released = new[order], released[order]
    held = _ceil(context, bs)
    width = int(_ceil(2 * c["context"] + c["chunk"], bs)) + 1
    order = rng.permutation(pool)
    table = np.full((B, width), -1, np.int64)
    used = np.arange(width)[None, :] < held[:, None]
    table[used] = order[: int(held.sum())]
    free = order[int(held.sum()):]
    head = int(rng.randint(0, pool))
    ring = np.full(pool, -1, np.int64)
    ring[(head + np.arange(free.size)) % pool] = free
    return dict(op="tables", block=bs, max_tokens=int(new.sum()) + 3, context=_ints(context), new=_ints(new),
                released=torch.from_numpy(released).cuda(), table=_ints(table), ring=_ints(ring),
                state=_ints(np.array([head, free.size])))


def _prepare_append(c, rng, gen):
    T, H, D, bs = c["tokens"], c["kv_heads"], c["dim"], c["block"]
    blocks = _ceil(T, bs) + 3
    slots = rng.permutation(blocks * bs)[:T] if T < 64 else (rng.permutation(blocks)[:, None] * bs + np.arange(bs)).reshape(-1)[:T]
    slots = np.where(rng.rand(T) < c["skipped"], -1, slots)
    dt = DTYPES[c["dtype"]]
    qkv = torch.randn(T, 4 * H, D, device="cuda", generator=gen).to(dt)  # a fused projection: two parts queries, one keys, one values
    cache = torch.randn(2, blocks, H, bs, D, device="cuda", generator=gen).to(dt)
    return dict(op="append", k=qkv[:, 2 * H:3 * H], v=qkv[:, 3 * H:], k_cache=cache[0], v_cache=cache[1], slots=_ints(slots, torch.int64))


def _attention_rows(c):
    """The rows of an attention case before they are put in order: new queries, and own tokens with them."""
    n = np.linspace(c["queries"], 0 if c["queries"] > 1 else 1, c["rows"]).round().astype(np.int64)
    return n, np.linspace(c["own"], _ceil(c["own"], 4), c["rows"]).astype(np.int64)


def _prepare_attention(c, rng, gen):
    B, Hq, H, D, L, bs = c["rows"], c["q_heads"], c["kv_heads"], c["dim"], c["prefix"], c["block"]
    n, lengths = _attention_rows(c)
    n = n[rng.permutation(B)]
    lengths = np.maximum(lengths[rng.permutation(B)], n)
    held = _ceil(lengths, bs)
    width = int(held.max()) + 1
    shared = _ceil(L, bs)
    blocks = int(held.sum()) + shared + 2
    order = rng.permutation(blocks)
    table = np.full((B, width), -1, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = order[shared: shared + int(held.sum())]
    offsets = np.concatenate([[0], np.cumsum(n)])
    dt = DTYPES[c["dtype"]]
    cache = torch.empty(2, blocks, H, bs, D, device="cuda", dtype=dt).normal_(generator=gen)
    q = torch.empty(int(offsets[-1]), Hq, D, device="cuda", dtype=dt).normal_(generator=gen)
    return dict(op="attention", q=q, k_cache=cache[0], v_cache=cache[1], offsets=_ints(offsets), table=_ints(table),
                lengths=_ints(lengths), shared=_ints(order[:shared]), prefix=L, queries=int(n.max()), scale=D ** -0.5)


def _prepare_linear(c, rng, gen):
    M, K, N = c["tokens"], c["inputs"], c["outputs"]
    dt = DTYPES[c["dtype"]]
    x = torch.randn(M, K, device="cuda", generator=gen)
    x *= torch.exp(0.5 * torch.randn(K, device="cuda", generator=gen))  # channels of uneven size, as activations have
    w = torch.randint(-127, 128, (N, K), device="cuda", generator=gen, dtype=torch.int8)
    w_scale = (0.5 + torch.rand(N, device="cuda", generator=gen)) * (0.02 / K ** 0.5)
    return dict(op="linear", x=x.to(dt), w=w, w_scale=w_scale)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _own_tables(s):
    t = _q3s().cache_tables(s["context"], s["new"], s["table"], s["ring"], s["state"], block_size=s["block"],
                            max_tokens=s["max_tokens"], released=s["released"])
    return (s["table"], s["ring"], t.free_state, t.lengths, t.query_offsets, t.slot_map, t.positions)


def _own_append(s):
    _q3s().cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    return s["k_cache"], s["v_cache"]


def _own_attention(s):
    return _q3s().prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["offsets"], s["table"], s["lengths"],
                                   prefix_blocks=s["shared"], prefix_length=s["prefix"], scale=s["scale"], return_lse=True)


def _own_linear(s):
    y, values, scales = _q3s().int8_linear(s["x"], s["w"], s["w_scale"], return_quantized=True)
    return y, values, scales


_OWN = {"tables": _own_tables, "append": _own_append, "attention": _own_attention, "linear": _own_linear}


def _plain_tables(s):
    bs, table, ring = s["block"], s["table"], s["ring"]
    width, pool = table.shape[1], ring.numel()
    head, count = s["state"][0], s["state"][1]
    before, new = s["context"], s["new"]
    context = torch.where(s["released"], 0, before)
    held = (context + bs - 1) // bs
    end = context + new
    fits = end <= width * bs
    need = torch.where(fits, (end + bs - 1) // bs - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= count))
    take = torch.where(granted, need, 0)
    column = torch.arange(width, device=table.device)
    # blocks of released rows go to the ring's end, in row order
    back = torch.where(s["released"], (before + bs - 1) // bs, 0)
    place = (head + count + (back.cumsum(0) - back)[:, None] + column) % pool
    place = torch.where(column < back[:, None], place, pool)
    longer = torch.cat([ring, ring.new_zeros(1)]).scatter(0, place.reshape(-1), table.reshape(-1))
    # new blocks come from the ring's start, in row order
    rank = column - held[:, None]
    fresh = ring[(head + (upto - need)[:, None] + rank) % pool]
    table = torch.where((rank >= 0) & (rank < take[:, None]), fresh, table)
    offsets = torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)
    token = torch.arange(s["max_tokens"], device=table.device)
    row = torch.searchsorted(offsets[1:], token, right=True)
    live = row < new.numel()
    row = row.clamp(max=new.numel() - 1)
    position = context[row] + token - offsets[row]
    inside = (position // bs).clamp(max=width - 1)
    slot = table[row, inside].to(torch.int64) * bs + position % bs
    slot = torch.where(live & granted[row], slot, -1)
    state = torch.stack([(head + take.sum()) % pool, count - take.sum() + back.sum()]).to(torch.int32)
    lengths = torch.where(granted, end, context)
    return table, longer[:pool], state, lengths, offsets, slot, torch.where(live, position, 0).to(torch.int32)


def _plain_append(s):
    kept = s["slots"] >= 0
    slot = s["slots"][kept]
    block, place = slot // s["k_cache"].shape[2], slot % s["k_cache"].shape[2]
    s["k_cache"][block, :, place] = s["k"][kept]
    s["v_cache"][block, :, place] = s["v"][kept]
    return s["k_cache"], s["v_cache"]


def _plain_attention(s):
    q, table, lengths, offsets = s["q"], s["table"], s["lengths"], s["offsets"]
    T, Hq, D = q.shape
    _, H, bs, _ = s["k_cache"].shape
    B, L, n = table.shape[0], s["prefix"], s["queries"]
    counts = offsets[1:] - offsets[:-1]
    i = torch.arange(n, device=q.device)
    token = (offsets[:-1, None] + i).clamp(max=max(T - 1, 0))
    padded = q[token].float().reshape(B, n, H, Hq // H, D) * s["scale"]

    def gathered(cache):
        own_part = cache[table.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
        shared = cache[s["shared"]].float().permute(1, 0, 2, 3).reshape(H, -1, D)[:, :L]
        return shared, own_part

    k_shared, k_own = gathered(s["k_cache"])
    v_shared, v_own = gathered(s["v_cache"])
    shared = torch.einsum("bnhgd,hld->bhngl", padded, k_shared)
    local = torch.einsum("bnhgd,bhld->bhngl", padded, k_own)
    j = torch.arange(local.shape[-1], device=q.device)
    last = (lengths - counts)[:, None] + i  # the newest own token that query i sees
    local.masked_fill_((j > last[:, :, None])[:, None, :, None], -math.inf)
    top = torch.maximum(shared.amax(-1) if L else local.amax(-1), local.amax(-1))
    top = torch.where(top == -math.inf, 0.0, top)
    shared, local = (shared - top[..., None]).exp(), (local - top[..., None]).exp()
    total = shared.sum(-1) + local.sum(-1)
    out = torch.einsum("bhngl,hld->bnhgd", shared, v_shared) + torch.einsum("bhngl,bhld->bnhgd", local, v_own)
    out = out / total.permute(0, 2, 1, 3)[..., None].clamp(min=1e-30)
    lse = (total.log() + top).permute(0, 2, 1, 3)
    packed = torch.arange(T, device=q.device)
    row = torch.searchsorted(offsets[1:], packed.to(offsets.dtype), right=True)
    at = packed - offsets[row]
    return out[row, at].reshape(T, Hq, D).to(q.dtype), lse[row, at].reshape(T, Hq)


def _plain_linear(s):
    x = s["x"].float()
    top = x.abs().amax(1)
    full = torch.full_like(top, 127.0)
    scales = top / full
    values = torch.round(x * torch.where(top > 0, full / top, 0.0)[:, None]).clamp(-127, 127)
    y = (values @ s["w"].float().t()) * scales[:, None] * s["w_scale"]
    return y.to(s["x"].dtype), values.to(torch.int8), scales


_PLAIN = {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention, "linear": _plain_linear}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op == "tables":
        context, new, ended = _table_rows(c)
        tokens = int(new.sum())
        blocks = tokens / c["block"] + float(_ceil(context, c["block"]).mean()) * int(ended.sum())
        # lengths and flags in, lengths and offsets out; slots and positions out; block ids read and written
        return {"bytes": c["rows"] * (4 + 4 + 1 + 4 + 4) + tokens * 12 + 8 * blocks, "flops": 0}
    if op == "append":
        part = c["tokens"] * (1 - c["skipped"]) * c["kv_heads"] * c["dim"] * 2
        return {"bytes": 4 * part + 8 * c["tokens"], "flops": 0}
    if op == "attention":
        n, lengths = _attention_rows(c)
        tokens, size = int(n.sum()), 2 * c["dim"]
        keys = c["prefix"] + int(lengths.sum())
        pairs = tokens * (c["prefix"] + float(lengths.mean()))
        return {"bytes": 2 * keys * c["kv_heads"] * size + 2 * tokens * c["q_heads"] * size + 4 * tokens * c["q_heads"],
                "flops": 4 * pairs * c["q_heads"] * c["dim"]}
    M, K, N = c["tokens"], c["inputs"], c["outputs"]
    size = 4 if c["dtype"] == "f32" else 2
    return {"bytes": M * K * (size + 1) + 4 * M + N * K + 4 * N + size * M * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits (whole numbers with Python's own integers)
# ---------------------------------------------------------------------------

def exact(case, seed):
    return {"tables": _exact_tables, "append": _exact_append, "attention": _exact_attention,
            "linear": _exact_linear}[case["op"]](prepare(case, seed))


def _exact_tables(s):
    bs, pool = s["block"], s["ring"].numel()
    table, ring = s["table"].tolist(), s["ring"].tolist()
    head, count = s["state"].tolist()
    new, gone = s["new"].tolist(), s["released"].tolist()
    start = [0 if g else c for c, g in zip(s["context"].tolist(), gone)]
    tail = head + count
    for r, c in enumerate(s["context"].tolist()):
        for k in range(_ceil(c, bs) if gone[r] else 0):
            ring[tail % pool] = table[r][k]
            tail += 1
    wanted, taken, lengths, slots, positions, offsets = 0, 0, [], [], [], [0]
    old = s["ring"].tolist()
    for r in range(len(new)):
        offsets.append(offsets[-1] + new[r])
        end = start[r] + new[r]
        blocks = range(_ceil(start[r], bs), _ceil(end, bs))
        allowed = end <= bs * len(table[r])
        if allowed:
            wanted += len(blocks)
            allowed = not len(blocks) or wanted <= count
        for k in blocks if allowed else ():
            table[r][k] = old[(head + taken) % pool]
            taken += 1
        lengths.append(end if allowed else start[r])
        slots += [table[r][p // bs] * bs + p % bs if allowed else -1 for p in range(start[r], end)]
        positions += list(range(start[r], end))
    rest = s["max_tokens"] - len(slots)
    whole = lambda x, t=torch.int32: torch.tensor(x, dtype=t)  # noqa: E731
    return (whole(table), whole(ring), whole([(head + taken) % pool, tail - head - taken]), whole(lengths), whole(offsets),
            whole(slots + [-1] * rest, torch.int64), whole(positions + [0] * rest))


def _exact_append(s):
    out = []
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        blocks, heads, bs, dim = cache.shape
        flat = cache.double().transpose(1, 2).reshape(blocks * bs, heads, dim)
        rows = s["slots"].cpu().numpy()
        where = torch.from_numpy(np.flatnonzero(rows >= 0)).cuda()
        flat.index_copy_(0, s["slots"][where], new[where].double())
        out.append(flat.reshape(blocks, bs, heads, dim).transpose(1, 2))
    return out


def _exact_attention(s):
    q = s["q"].double()
    T, Hq, D = q.shape
    _, H, bs, _ = s["k_cache"].shape
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()

    def keys(blocks, length, cache):
        return torch.cat([cache[blocks[: _ceil(length, bs)].long()].transpose(1, 2).reshape(-1, H, D)[:length]]).double()

    out, lse = torch.zeros_like(q), torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    k0, v0 = (keys(s["shared"], s["prefix"], x) for x in (s["k_cache"], s["v_cache"]))
    for b in range(len(lengths)):
        k1, v1 = (keys(s["table"][b], lengths[b], x) for x in (s["k_cache"], s["v_cache"]))
        for t in range(offsets[b], offsets[b + 1]):
            seen = lengths[b] - (offsets[b + 1] - 1 - t)
            if s["prefix"] + max(seen, 0) == 0:
                continue
            k = torch.cat([k0, k1[: max(seen, 0)]]).repeat_interleave(Hq // H, 1)
            v = torch.cat([v0, v1[: max(seen, 0)]]).repeat_interleave(Hq // H, 1)
            score = s["scale"] * (k * q[t]).sum(-1)
            lse[t] = torch.logsumexp(score, 0)
            out[t] = (torch.softmax(score, 0)[..., None] * v).sum(0)
    return out, lse


def _exact_linear(s):
    # the 8-bit values and their scales are defined in 32-bit arithmetic; everything after them in 64
    x = s["x"].float()
    top = torch.linalg.vector_norm(x, ord=math.inf, dim=1)
    unit = torch.div(torch.full_like(top, 127.0), top).masked_fill(top == 0, 0.0)
    values = (x * unit.unsqueeze(1)).round()
    y = torch.matmul(values.double(), s["w"].double().t()) * s["w_scale"].double() * (top.double() / 127).unsqueeze(1)
    return y, values.to(torch.int8), top.double() / 127
