"""Measured passes through the operators of a decode step that takes several tokens of a row: drafted tokens that are
verified, and prompts that arrive in chunks.

* ``rotary``   rotary positions with several axes, alone (``q3s.rotary``) or with the append of the rotated keys and
               the values to the paged cache (``q3s.rotary_append``);
* ``chunk``    attention of every row's chunk of new tokens over its pages, behind a shared prefix, optionally within a
               sliding window (``q3s.chunk_attention``);
* ``verify``   drafted tokens verified against the target's probabilities from given random numbers
               (``q3s.verify_drafts``);
* ``trim``     rows cut back to what was accepted, their pages returned to the free ring (``q3s.cache_trim``).

``own`` chooses between the plain form below (elementary torch operations) and the package's kernels.
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
        # one stream's last token and five drafts: the latency of the step's first launch of a layer
        dict(name="rotate 6 tokens", op="rotary", tokens=6, q_heads=16, kv_heads=8, dim=128, pairs=64, sections="24,20,20",
             interleaved=True, adjacent=False, append=True, skipped=0.0, block=16, far=700, dtype="bf16"),
        # prefill chunks of a serving batch out of a fused projection, some tokens without a slot
        dict(name="rotate 8191 tokens f16", op="rotary", tokens=8191, q_heads=16, kv_heads=8, dim=128, pairs=64,
             sections="64", interleaved=False, adjacent=False, append=True, skipped=0.02, block=32, far=30000, dtype="f16"),
        # part of each head turned, far positions, neighbouring pairs, 32 bits
        dict(name="rotate 5000 tokens partly f32", op="rotary", tokens=5000, q_heads=12, kv_heads=2, dim=80, pairs=18,
             sections="8,5,5", interleaved=False, adjacent=True, append=False, skipped=0.0, block=16, far=1000000, dtype="f32"),
        # one stream's last token and four drafts behind its voice prompt
        dict(name="chunk 1 row of 5", op="chunk", rows=1, q_heads=16, kv_heads=8, dim=128, prefix=200, own=700, queries=5,
             window=0, block=16, dtype="bf16"),
        # a serving batch's drafts, ragged, some rows idle
        dict(name="chunk 48 rows up to 9", op="chunk", rows=48, q_heads=32, kv_heads=8, dim=128, prefix=333, own=1200,
             queries=9, window=0, block=32, dtype="bf16"),
        # text chunks of a batch through a layer with a sliding window
        dict(name="chunk 13 rows window f16", op="chunk", rows=13, q_heads=16, kv_heads=4, dim=64, prefix=0, own=3000,
             queries=700, window=512, block=64, dtype="f16"),
        # two long prompts behind what is cached already
        dict(name="chunk 2 rows of 4096", op="chunk", rows=2, q_heads=16, kv_heads=8, dim=128, prefix=150, own=3500,
             queries=4096, window=0, block=16, dtype="bf16"),
        # one stream's drafts over the codec vocabulary
        dict(name="verify 1 row of 5", op="verify", rows=1, queries=5, vocab=2048, drafts=True, keep=50, greedy=0.0, dtype="bf16"),
        # a serving batch's drafts without probabilities (a lookup), over what top-k left, some rows greedy
        dict(name="verify 200 rows up to 6", op="verify", rows=200, queries=6, vocab=2051, drafts=False, keep=50, greedy=0.2,
             dtype="f32"),
        # a serving batch over a text vocabulary
        dict(name="verify 64 rows of 65000", op="verify", rows=64, queries=8, vocab=65000, drafts=True, keep=0, greedy=0.1,
             dtype="bf16"),
        # a serving batch's refused drafts
        dict(name="trim 48 rows", op="trim", rows=48, context=900, removed=8, ended=0.0, block=16),
        # a full batch, some rows ended
        dict(name="trim 1500 rows", op="trim", rows=1500, context=3000, removed=40, ended=0.1, block=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "chunk", "chunk", "chunk", "verify", "verify", "trim"])
    if op == "rotary":
        dim, dtype = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice(["bf16", "f16", "f32"])
        pairs = dim // 2 if rng.random() < 0.6 else rng.randint(1, dim // 2)
        axes = rng.choice([1, 1, 2, 3, 3])
        parts = [pairs // axes] * axes
        parts[0] += pairs - sum(parts)
        q_heads, kv_heads = rng.choice([1, 3, 8, 16]), rng.choice([1, 2, 8])
        most = 8000 * 32 * 128 // ((q_heads + 2 * kv_heads) * dim * (2 if dtype == "f32" else 1))  # the listed case's bytes
        return dict(op=op, tokens=min(_log(rng, 1, 8000), most), q_heads=q_heads, kv_heads=kv_heads, dim=dim, pairs=pairs,
                    sections=",".join(map(str, parts)), interleaved=rng.random() < 0.5, adjacent=rng.random() < 0.3,
                    append=rng.random() < 0.7, skipped=rng.choice([0.0, 0.02, 0.2]), block=rng.choice([16, 32, 64]),
                    far=_log(rng, 100, 1000000), dtype=dtype)
    if op == "chunk":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        rows = _log(rng, 1, 64)
        queries = _log(rng, 1, 2500)
        pairs = 2 * 4096 * 16 * 7700 // (rows * queries * kv * group)  # keys, by the scores of the largest listed case
        queries = min(queries, max(pairs // 2, 1))
        rest = max(pairs - queries, 1)
        own_tokens = min(_log(rng, 1, 6000), max(rest // 2, 1), 200000 // rows)
        return dict(op=op, rows=rows, q_heads=kv * group, kv_heads=kv, dim=rng.choice([64, 128]),
                    prefix=min(rng.choice([0, 1]) * _log(rng, 1, 2000), rest // 2), own=own_tokens, queries=queries,
                    window=rng.choice([0, 0, 1]) * _log(rng, 16, 2000), block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]))
    if op == "verify":
        vocab = rng.choice([1024, 2048, 2051]) if rng.random() < 0.5 else _log(rng, 100, 65000)
        queries = rng.randint(1, 9)
        return dict(op=op, rows=min(_log(rng, 1, 256), 64 * 8 * 65000 // (queries * vocab)), queries=queries, vocab=vocab,
                    drafts=rng.random() < 0.6, keep=rng.choice([0, 0, 50]), greedy=rng.choice([0.0, 0.2]),
                    dtype=rng.choice(["bf16", "f32", "f16"]))
    return dict(op=op, rows=_log(rng, 1, 4000), context=_log(rng, 1, 4000), removed=_log(rng, 1, 100),
                ended=rng.choice([0.0, 0.05, 0.2]), block=rng.choice([16, 32, 64]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"rotary": _prepare_rotary, "chunk": _prepare_chunk, "verify": _prepare_verify,
            "trim": _prepare_trim}[case["op"]](case, rng, gen)


def _ints(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _ceil(a, b):
    return -(-a // b)


def _sections(c):
    return [int(x) for x in c["sections"].split(",")]


def _prepare_rotary(c, rng, gen):
    T, Hq, H, D, bs = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["block"]
    dt = DTYPES[c["dtype"]]
    sections = _sections(c)
    inv_freq = torch.from_numpy((1.0e6 ** (-np.arange(c["pairs"]) / c["pairs"])).astype(np.float32)).cuda()
    # time runs on from somewhere in the stream; the other axes follow it or stay within a picture
    start = int(rng.randint(0, c["far"]))
    places = [start + np.arange(T) // 3] + [start + rng.randint(0, 60, T) for _ in sections[1:]]
    qkv = torch.empty(T, Hq + 2 * H, D, device="cuda").normal_(generator=gen).to(dt)  # a fused projection
    s = dict(op="rotary", append=c["append"], q=qkv[:, :Hq], inv_freq=inv_freq, sections=sections,
             interleaved=c["interleaved"], adjacent=c["adjacent"],
             positions=_ints(np.stack(places)) if len(sections) > 1 else _ints(places[0]))
    if c["append"]:
        blocks = _ceil(T, bs) + 2
        slots = (rng.permutation(blocks)[:, None] * bs + np.arange(bs)).reshape(-1)[:T]
        slots = np.where(rng.rand(T) < c["skipped"], -1, slots)
        cache = torch.empty(2, blocks, H, bs, D, device="cuda", dtype=dt).normal_(generator=gen)
        s.update(k=qkv[:, Hq:Hq + H], v=qkv[:, Hq + H:], k_cache=cache[0], v_cache=cache[1], slots=_ints(slots, torch.int64))
    return s


def _chunk_rows(c):
    """The rows of a chunk case before they are put in order: new queries, and own tokens with them."""
    n = np.linspace(c["queries"], c["queries"] // 2 if c["rows"] < 4 else 0, c["rows"]).round().astype(np.int64)
    return n, np.linspace(c["own"], _ceil(c["own"], 4), c["rows"]).astype(np.int64) + n


def _prepare_chunk(c, rng, gen):
    B, Hq, H, D, L, bs = c["rows"], c["q_heads"], c["kv_heads"], c["dim"], c["prefix"], c["block"]
    n, lengths = _chunk_rows(c)
    order = rng.permutation(B)
    n, lengths = n[order], lengths[order]
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
    return dict(op="chunk", q=q, k_cache=cache[0], v_cache=cache[1], offsets=_ints(offsets), table=_ints(table),
                lengths=_ints(lengths), shared=_ints(order[:shared]), prefix=L, queries=int(n.max()), window=c["window"],
                scale=D ** -0.5)


def _verify_rows(c):
    """Tokens of the rows of a verify case (the last accepted token and its drafts) before they are put in order."""
    return np.linspace(c["queries"], min(c["queries"], 1), c["rows"]).round().astype(np.int64)


def _prepare_verify(c, rng, gen):
    B, V = c["rows"], c["vocab"]
    n = _verify_rows(c)
    n = n[rng.permutation(B)]
    offsets = np.concatenate([[0], np.cumsum(n)])
    T = int(offsets[-1])
    dt = DTYPES[c["dtype"]]
    logits = torch.empty(T, V, device="cuda").normal_(generator=gen) * 3.0
    drafter = logits + torch.empty(T, V, device="cuda").normal_(generator=gen)  # a smaller model: near the target, not equal
    if 0 < c["keep"] < V:  # what top-k left
        least = logits.topk(c["keep"], dim=1).values[:, -1:]
        logits = torch.where(logits < least, -math.inf, logits)
    proposals = torch.softmax(drafter, -1)
    ids = torch.randint(0, V, (T,), device="cuda", generator=gen)
    probabilities = None
    if T > 1:
        first = torch.zeros(T, dtype=torch.bool, device="cuda")
        first[_ints(offsets[:-1], torch.int64)] = True
        # entry t holds what token t was drawn from: the drafter's distribution one place earlier
        before = torch.cat([proposals[:1], proposals[:-1]])
        if c["drafts"]:
            probabilities = before
            drawn = torch.multinomial(before, 1, generator=gen)[:, 0]
        else:  # a lookup proposes the likeliest token
            drawn = before.argmax(1)
        ids = torch.where(first, ids, drawn)
    elif c["drafts"]:
        probabilities = proposals
    temperature = np.where(rng.permutation(B) < int(B * c["greedy"]), 0.0, 0.8)
    return dict(op="verify", logits=logits.to(dt), ids=ids, offsets=_ints(offsets), probabilities=probabilities,
                uniforms=torch.rand(T, device="cuda", generator=gen),
                temperature=torch.from_numpy(temperature).float().cuda(), queries=int(n.max()))


def _trim_rows(c):
    """The rows of a trim case before they are put in order: lengths, and tokens that go."""
    B = c["rows"]
    lengths = np.linspace(0, 2 * c["context"], B).astype(np.int64)
    gone = np.minimum((np.arange(B) * 7919) % (c["removed"] + 1), lengths)
    ended = (np.arange(B) * 104729) % max(B, 1) < int(B * c["ended"])
    return lengths, np.where(ended, lengths, gone)


def _prepare_trim(c, rng, gen):
    B, bs = c["rows"], c["block"]
    lengths, gone = _trim_rows(c)
    order = rng.permutation(B)
    lengths, gone = lengths[order], gone[order]
    held = _ceil(lengths, bs)
    pool = int(held.sum()) + B
    width = _ceil(2 * c["context"], bs) + 1
    order = rng.permutation(pool)
    table = np.full((B, width), -1, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = order[: int(held.sum())]
    free = order[int(held.sum()):]
    head = int(rng.randint(0, pool))
    ring = np.full(pool, -1, np.int64)
    ring[(head + np.arange(free.size)) % pool] = free
    return dict(op="trim", block=bs, lengths=_ints(lengths), removed=_ints(gone), table=_ints(table), ring=_ints(ring),
                state=_ints(np.array([head, free.size])))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _own_rotary(s):
    how = dict(sections=s["sections"], interleaved=s["interleaved"], adjacent=s["adjacent"])
    if not s["append"]:
        return _q3s().rotary(s["q"], s["positions"], s["inv_freq"], **how)
    q = _q3s().rotary_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"], **how)
    return q, s["k_cache"], s["v_cache"]


def _own_chunk(s):
    return _q3s().chunk_attention(s["q"], s["k_cache"], s["v_cache"], s["offsets"], s["table"], s["lengths"],
                                  prefix_blocks=s["shared"], prefix_length=s["prefix"], window=s["window"],
                                  scale=s["scale"], return_lse=True)


def _own_verify(s):
    r = _q3s().verify_drafts(s["logits"], s["ids"], s["offsets"], s["uniforms"], draft_probs=s["probabilities"],
                             temperature=s["temperature"])
    return r.tokens, r.accepted, r.rejected, r.next_ids


def _own_trim(s):
    t = _q3s().cache_trim(s["lengths"], s["removed"], s["table"], s["ring"], s["state"], block_size=s["block"])
    return s["ring"], t.free_state, t.lengths


_OWN = {"rotary": _own_rotary, "chunk": _own_chunk, "verify": _own_verify, "trim": _own_trim}


def _plain_rotary(s):
    positions = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    P, sections = s["inv_freq"].numel(), s["sections"]
    i = torch.arange(P, device=positions.device)
    if s["interleaved"]:
        bound = torch.tensor(sections, device=positions.device) * len(sections)
        axis = torch.where(i < bound[i % len(sections)], i % len(sections), 0)
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=positions.device),
                                       torch.tensor(sections, device=positions.device), output_size=P)
    # far positions: the angle in 64 bits
    angle = positions[axis].t().double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        y = x.float().clone()
        a = slice(0, 2 * P, 2) if s["adjacent"] else slice(0, P)
        b = slice(1, 2 * P, 2) if s["adjacent"] else slice(P, 2 * P)
        x1, x2 = x[..., a].float(), x[..., b].float()
        y[..., a] = x1 * cos - x2 * sin
        y[..., b] = x1 * sin + x2 * cos
        return y.to(x.dtype)

    q = turned(s["q"])
    if not s["append"]:
        return q
    kept = s["slots"] >= 0
    slot = s["slots"][kept]
    block, place = slot // s["k_cache"].shape[2], slot % s["k_cache"].shape[2]
    s["k_cache"][block, :, place] = turned(s["k"])[kept]
    s["v_cache"][block, :, place] = s["v"][kept]
    return q, s["k_cache"], s["v_cache"]


def _plain_chunk(s):
    q, table, lengths, offsets = s["q"], s["table"], s["lengths"], s["offsets"]
    T, Hq, D = q.shape
    _, H, bs, _ = s["k_cache"].shape
    B, L, n = table.shape[0], s["prefix"], s["queries"]
    counts = offsets[1:] - offsets[:-1]
    i = torch.arange(n, device=q.device)
    token = (offsets[:-1, None] + i).clamp(max=max(T - 1, 0))
    padded = (q[token].float() * s["scale"]).reshape(B, n, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)

    def gathered(cache):
        own_part = cache[table.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
        shared = cache[s["shared"]].float().permute(1, 0, 2, 3).reshape(1, H, -1, D)[:, :, :L]
        return torch.cat([shared.expand(B, -1, -1, -1), own_part], 2)

    k, v = gathered(s["k_cache"]), gathered(s["v_cache"])
    score = (padded @ k.transpose(2, 3)).reshape(B, H, Hq // H, n, -1)
    j = torch.arange(score.shape[-1], device=q.device)
    last = L + (lengths - counts)[:, None] + i  # the newest key that query i sees
    unseen = j > last[:, :, None]
    if s["window"]:
        unseen |= j <= last[:, :, None] - s["window"]
    score.masked_fill_(unseen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    score = (score - top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.reshape(B, H, -1, score.shape[-1]) @ v).reshape(B, H, Hq // H, n, D) / total.clamp(min=1e-30)
    lse = (total.log() + top)[..., 0]
    packed = torch.arange(T, device=q.device)
    row = torch.searchsorted(offsets[1:], packed.to(offsets.dtype), right=True)
    at = packed - offsets[row]
    out, lse = out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D), lse.permute(0, 3, 1, 2).reshape(B, n, Hq)
    return out[row, at].to(q.dtype), lse[row, at]


def _plain_verify(s):
    # 64 bits: a draw may fall next to a border
    logits, ids, offsets = s["logits"], s["ids"], s["offsets"]
    T, V = logits.shape
    B = offsets.numel() - 1
    token = torch.arange(T, device=ids.device)
    row = torch.searchsorted(offsets[1:], token.to(offsets.dtype), right=True)
    heat = s["temperature"][row].double()[:, None]
    x = logits.double()
    top = x.amax(1, keepdim=True)
    p = ((x - top) / torch.where(heat > 0, heat, 1.0)).exp()
    p = p / p.sum(1, keepdim=True)
    place = torch.arange(V, device=ids.device)
    best = torch.where(x == top, place, V).amin(1)
    p = torch.where(heat > 0, p, (place == best[:, None]).double())
    # token t + 1 was proposed after token t
    after = (token + 1).clamp(max=T - 1)
    has_draft = (token + 1 < offsets[row + 1])
    proposed = ids[after]
    if s["probabilities"] is None:
        q = (place == proposed[:, None]).double()
    else:
        q = s["probabilities"][after].double()
    chance = q.gather(1, proposed[:, None])[:, 0]
    passed = has_draft & (s["uniforms"][after].double() * chance < p.gather(1, proposed[:, None])[:, 0])
    # drafts accepted: those before the first that was not
    failed = (~passed).long().cumsum(0)
    start = offsets[:-1].long()
    n = (offsets[1:] - offsets[:-1]).long()
    base = torch.where(start > 0, failed[(start - 1).clamp(min=0)], 0)
    accepted = torch.zeros(B, dtype=torch.long, device=ids.device).index_add_(0, row, (passed & (failed == base[row])).long())
    at = (start + accepted).clamp(max=T - 1)
    rest = torch.where(has_draft[at][:, None], (p[at] - q[at]).clamp(min=0), p[at])
    total = rest.sum(1, keepdim=True)
    rest = torch.where(total > 0, rest, p[at])
    edge = rest.cumsum(1)
    aim = s["uniforms"][start.clamp(max=T - 1)].double()[:, None] * torch.where(total > 0, total, 1.0)
    last = torch.where(rest > 0, place, -1).amax(1)
    fresh = torch.where(edge > aim, place, V).amin(1)
    fresh = torch.where(fresh < V, fresh, last)
    fresh = torch.where(n > 0, fresh, -1)
    inside = token - start[row]
    tokens = torch.where(inside < accepted[row], proposed, torch.where(inside == accepted[row], fresh[row], -1))
    accepted = accepted.to(torch.int32)
    rejected = torch.where(n > 0, n - 1 - accepted, 0).to(torch.int32)
    return tokens, accepted, rejected, fresh


def _plain_trim(s):
    bs, table, ring = s["block"], s["table"], s["ring"]
    pool, width = ring.numel(), table.shape[1]
    head, count = s["state"][0], s["state"][1]
    kept = s["lengths"] - s["removed"]
    first, held = (kept + bs - 1) // bs, (s["lengths"] + bs - 1) // bs
    back = held - first
    column = torch.arange(width, device=table.device)
    rank = column - first[:, None]
    place = (head + count + (back.cumsum(0) - back)[:, None] + rank) % pool
    place = torch.where((rank >= 0) & (column < held[:, None]), place, pool)
    longer = torch.cat([ring, ring.new_zeros(1)]).scatter(0, place.reshape(-1), table.reshape(-1))
    return longer[:pool], torch.stack([head, count + back.sum()]).to(torch.int32), kept.to(torch.int32)


_PLAIN = {"rotary": _plain_rotary, "chunk": _plain_chunk, "verify": _plain_verify, "trim": _plain_trim}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op == "rotary":
        size = 4 if c["dtype"] == "f32" else 2
        heads = c["q_heads"] + (2 * c["kv_heads"] * (1 - c["skipped"]) if c["append"] else 0)
        places = 4 * c["tokens"] * len(_sections(c)) + (8 * c["tokens"] if c["append"] else 0)
        turned = c["q_heads"] + (c["kv_heads"] if c["append"] else 0)
        return {"bytes": 2 * c["tokens"] * heads * c["dim"] * size + places, "flops": 6 * c["tokens"] * turned * c["pairs"]}
    if op == "chunk":
        n, lengths = _chunk_rows(c)
        size, W = 2 * c["dim"], c["window"]
        keys, pairs = c["prefix"], 0
        for m, length in zip(n.tolist(), lengths.tolist()):
            seen = c["prefix"] + length - m + np.arange(1, m + 1)  # keys up to and including each query's own
            pairs += int((np.minimum(seen, W) if W else seen).sum())
            reach = c["prefix"] + length
            keys += (min(reach, W + m - 1) if W else length) if m else 0
        tokens = int(n.sum())
        return {"bytes": 2 * keys * c["kv_heads"] * size + 2 * tokens * c["q_heads"] * size + 4 * tokens * c["q_heads"],
                "flops": 4 * pairs * c["q_heads"] * c["dim"]}
    if op == "verify":
        tokens = int(_verify_rows(c).sum())
        size = 4 if c["dtype"] == "f32" else 2
        drafts = max(tokens - c["rows"], 0) if c["drafts"] else 0
        return {"bytes": tokens * c["vocab"] * size + drafts * c["vocab"] * 4 + tokens * 20 + c["rows"] * 24,
                "flops": 4 * tokens * c["vocab"] + 3 * c["rows"] * c["vocab"]}
    lengths, gone = _trim_rows(c)
    blocks = int((_ceil(lengths, c["block"]) - _ceil(lengths - gone, c["block"])).sum())
    return {"bytes": 12 * c["rows"] + 8 * blocks + 16, "flops": 0}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits (whole numbers with Python's own integers)
# ---------------------------------------------------------------------------

def exact(case, seed):
    return {"rotary": _exact_rotary, "chunk": _exact_chunk, "verify": _exact_verify,
            "trim": _exact_trim}[case["op"]](prepare(case, seed))


def _exact_rotary(s):
    sections, P = s["sections"], s["inv_freq"].numel()
    axes = len(sections)
    if s["interleaved"]:
        axis = [i % axes if i < axes * sections[i % axes] else 0 for i in range(P)]
    else:
        axis = [a for a, m in enumerate(sections) for _ in range(m)]
    where = s["positions"].reshape(axes, -1)
    turn = torch.stack([where[a].double() * s["inv_freq"][i].double() for i, a in enumerate(axis)], 1)
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]  # each pair as a complex number

    def apply(x):
        y = x.double().clone()
        first = [2 * i if s["adjacent"] else i for i in range(P)]
        second = [2 * i + 1 if s["adjacent"] else i + P for i in range(P)]
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q = apply(s["q"])
    if not s["append"]:
        return q
    out = [q]
    for new, cache in ((apply(s["k"]), s["k_cache"]), (s["v"].double(), s["v_cache"])):
        blocks, heads, bs, dim = cache.shape
        flat = cache.double().transpose(1, 2).reshape(blocks * bs, heads, dim)
        where = torch.from_numpy(np.flatnonzero(s["slots"].cpu().numpy() >= 0)).cuda()
        flat.index_copy_(0, s["slots"][where], new[where])
        out.append(flat.reshape(blocks, bs, heads, dim).transpose(1, 2))
    return tuple(out)


def _exact_chunk(s):
    q = s["q"].double()
    T, Hq, D = q.shape
    _, H, bs, _ = s["k_cache"].shape
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()

    def keys(blocks, length, cache):
        return cache[blocks[: _ceil(length, bs)].long()].transpose(1, 2).reshape(-1, H, D)[:length].double()

    out, lse = torch.zeros_like(q), torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    k0, v0 = (keys(s["shared"], s["prefix"], x) for x in (s["k_cache"], s["v_cache"]))
    for b in range(len(lengths)):
        k = torch.cat([k0, keys(s["table"][b], lengths[b], s["k_cache"])])
        v = torch.cat([v0, keys(s["table"][b], lengths[b], s["v_cache"])])
        end = k.shape[0]
        for t0 in range(offsets[b], offsets[b + 1], 512):
            t1 = min(t0 + 512, offsets[b + 1])
            at = torch.arange(t0, t1, device=q.device)[:, None] + (end - offsets[b + 1])  # place of each query's own key
            j = torch.arange(end, device=q.device)[None]
            seen = (j <= at) & ((j > at - s["window"]) if s["window"] else True)
            for h in range(Hq):
                score = torch.where(seen, s["scale"] * (q[t0:t1, h] @ k[:, h // (Hq // H)].t()), -math.inf)
                lse[t0:t1, h] = torch.logsumexp(score, 1)
                out[t0:t1, h] = torch.nan_to_num(torch.softmax(score, 1)) @ v[:, h // (Hq // H)]
    return out, lse


def _exact_verify(s):
    logits, ids, offsets = s["logits"].float().cpu().numpy(), s["ids"].tolist(), s["offsets"].tolist()
    proposals = None if s["probabilities"] is None else s["probabilities"].cpu().numpy()
    uniforms = s["uniforms"].double().tolist()
    heat = s["temperature"].double().tolist()
    T, V = logits.shape
    tokens, accepted, rejected, fresh = [-1] * T, [], [], []

    def target(t, b):
        x = logits[t].astype(np.float64)
        if heat[b] == 0:
            p = np.zeros(V)
            p[int(np.argmax(x))] = 1
            return p
        p = np.exp((x - x.max()) / heat[b])
        return p / math.fsum(p)

    for b in range(len(offsets) - 1):
        t, end, got = offsets[b], offsets[b + 1], 0
        if t == end:
            accepted.append(0)
            rejected.append(0)
            fresh.append(-1)
            continue
        u = uniforms[t]
        while True:
            p = target(t, b)
            if t + 1 == end:
                break
            d = ids[t + 1]
            q = np.eye(1, V, d)[0] if proposals is None else proposals[t + 1].astype(np.float64)
            if not uniforms[t + 1] * q[d] < p[d]:
                rest = np.maximum(p - q, 0)
                p = rest if rest.any() else p
                break
            tokens[t] = d
            got += 1
            t += 1
        over = np.flatnonzero(np.cumsum(p) > u * p.sum())
        tokens[t] = int(over[0]) if over.size else int(np.flatnonzero(p)[-1])
        accepted.append(got)
        rejected.append(end - 1 - t)
        fresh.append(tokens[t])
    return (torch.tensor(tokens), torch.tensor(accepted, dtype=torch.int32), torch.tensor(rejected, dtype=torch.int32),
            torch.tensor(fresh))


def _exact_trim(s):
    bs, table, ring = s["block"], s["table"].tolist(), s["ring"].tolist()
    head, count = s["state"].tolist()
    lengths = []
    for row, (length, gone) in zip(table, zip(s["lengths"].tolist(), s["removed"].tolist())):
        lengths.append(length - gone)
        for j in range(_ceil(length - gone, bs), _ceil(length, bs)):
            ring[(head + count) % len(ring)] = row[j]
            count += 1
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (ring, [head, count], lengths))
