"""The operators for steps of several tokens a row, on the GPU, against their
definitions in Python integers and float64 (tests/several_reference.py).

Tolerances, from the arithmetic:

* rotary: an angle is off by 3 * 2^-53 of itself (a 64-bit product of three
  factors) and by 2^-24 of what is left of it (at most pi / 4); sin and cos by
  two units of the last place, 2^-22 (CUDA's bound is below that), times scale
  2^-24; the two products 2^-24 each.  So |err| <= (|x1| + |x2|) scale (2^-21 +
  2^-51 |angle|) before the rounding to the type, half a step: r |y| with r =
  2^-8 bf16, 2^-11 f16, 2^-24 fp32 (and half the type's smallest number).
* trimming and verification: equal.
"""
import numpy as np
import pytest
import torch

import several_reference as R
import q3s

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


@pytest.fixture(scope="module")
def dev(cuda_device):
    q3s.load_torch_ops()
    return cuda_device


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


# ---- rotary -------------------------------------------------------------------

def check_turned(got, x, positions, inv_freq, **how):
    want, size, angle = R.rotary(x, positions, inv_freq.cpu(), **how)
    tol = size * (2.0 ** -21 + 2.0 ** -51 * angle)
    tol = torch.where(size > 0, tol * (1 + ROUNDOFF[got.dtype]) + ROUNDOFF[got.dtype] * want.abs() + SMALLEST[got.dtype], 0.0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def frequencies(pairs, dev, base=1e4):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,heads,dim,pairs,sections,interleaved,adjacent", [
    (1, 1, 2, 1, (), False, False),
    (1, 16, 128, 64, (24, 20, 20), True, False),
    (5, 3, 128, 64, (24, 20, 20), False, False),
    (700, 4, 64, 32, (), False, False),
    (33, 2, 80, 20, (8, 6, 6), False, True),
    (17, 5, 96, 48, (16, 16, 16), True, True),
    (9, 2, 256, 128, (50, 78), False, False),
    (7, 2, 130, 61, (20, 20, 21), False, False),
    (7, 2, 67, 13, (13, 0), False, True),
    (3, 1, 1024, 512, (128, 128, 128, 128), True, False),
    (2500, 1, 128, 8, (), False, False)])
def test_rotary(dev, T, heads, dim, pairs, sections, interleaved, adjacent, dtype):
    g = torch.Generator(device=dev).manual_seed(T + dim)
    x = torch.randn(T, heads, dim, device=dev, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (max(len(sections), 1), T), device=dev, generator=g, dtype=torch.int32)
    how = dict(sections=sections, interleaved=interleaved, adjacent=adjacent)
    f = frequencies(pairs, dev)
    y = q3s.rotary(x, pos if sections else pos[0], f, **how)
    assert y.is_contiguous() and y.dtype == dtype
    check_turned(y, x, pos, f, **how)


def test_rotary_far_and_negative_positions_and_scale(dev):
    pos = i32([0, 1, -1, -1000003, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 123456789], dev)
    x = torch.randn(8, 2, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(0))
    f = frequencies(32, dev)
    check_turned(q3s.rotary(x, pos, f, scale=1.25), x, pos, f, scale=1.25)
    check_turned(q3s.rotary(x, pos, f * 1e-3), x, pos, f * 1e-3)


def test_rotary_one_list_of_positions_serves_all_axes(dev):
    x = torch.randn(9, 2, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).bfloat16()
    f, pos = frequencies(64, dev), i32(np.arange(9) * 7, dev)
    y = q3s.rotary(x, pos, f, sections=(24, 20, 20), interleaved=True)
    assert torch.equal(y, q3s.rotary(x, pos, f)) and torch.equal(y, q3s.rotary(x, pos.repeat(3, 1), f, sections=(24, 20, 20)))


def test_rotary_of_views(dev):
    """Strides, a head whose vectors are not aligned, and no tokens or heads."""
    g = torch.Generator(device=dev).manual_seed(2)
    base = torch.randn(40, 6, 300, device=dev, generator=g).bfloat16()
    f, pos = frequencies(32, dev), i32(np.arange(40) * 3, dev)
    for x in (base[:, 1:4, 8:136], base[:, :, 1:65], base[::2, ::3, 5:69], base[:, 1:2, :64]):
        p = pos[:x.shape[0]]
        check_turned(q3s.rotary(x, p, f), x, p, f)
        check_turned(q3s.rotary(x, p, f, adjacent=True), x, p, f, adjacent=True)
    assert q3s.rotary(base[:0, :, :64], pos[:0], f).shape == (0, 6, 64)
    assert q3s.rotary(base[:, :0, :64], pos, f).shape == (40, 0, 64)


def make_caches(dev, dtype, blocks, heads, bs, dim, order, g):
    if order == "heads":
        c = torch.randn(2, blocks, heads, bs, dim, device=dev, generator=g).to(dtype)
        return c[0], c[1]
    c = torch.randn(2, blocks, bs, heads, dim, device=dev, generator=g).to(dtype)
    return c[0].transpose(1, 2), c[1].transpose(1, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,dim,pairs,bs,order", [
    (1, 16, 8, 128, 64, 16, "heads"), (6, 16, 8, 128, 64, 16, "tokens"), (333, 3, 2, 80, 18, 48, "heads"),
    (3000, 4, 1, 64, 32, 32, "tokens"), (50, 0, 2, 128, 64, 16, "heads"), (21, 2, 3, 66, 33, 5, "heads")])
def test_rotary_append(dev, T, hq, hk, dim, pairs, bs, order, dtype):
    rng = np.random.RandomState(T)
    g = torch.Generator(device=dev).manual_seed(T)
    blocks = R.ceil_div(T, bs) + 3
    kc, vc = make_caches(dev, dtype, blocks, hk, bs, dim, order, g)
    before = kc.clone(), vc.clone()
    qkv = torch.randn(T, hq + 2 * hk, dim, device=dev, generator=g).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    slots = rng.permutation(blocks * bs)[:T]
    slots[rng.rand(T) < 0.2] = -1
    slot_map = torch.as_tensor(slots, device=dev)
    pos = torch.randint(0, 100000, (3, T), device=dev, generator=g, dtype=torch.int32)
    sections = (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)
    f = frequencies(pairs, dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    out = q3s.rotary_append(q, k, v, pos, f, kc, vc, slot_map, sections=sections, interleaved=True, error_word=err)
    how = dict(sections=sections, interleaved=True)
    check_turned(out, q, pos, f, **how)
    kept = slots >= 0
    at = torch.as_tensor(slots[kept], device=dev)
    rows = torch.as_tensor(np.flatnonzero(kept), device=dev)
    got_k, got_v = kc[at // bs, :, at % bs], vc[at // bs, :, at % bs]
    check_turned(got_k, k[rows], pos[:, rows], f, **how)
    assert torch.equal(got_v, v[rows]) and int(err) == 0
    if hq:  # a stored key is the same as one that only turns
        assert torch.equal(got_k, q3s.rotary(k, pos, f, **how)[rows])
    untouched = torch.ones(blocks, bs, dtype=torch.bool, device=dev)
    untouched[at // bs, at % bs] = False
    for now, was in ((kc, before[0]), (vc, before[1])):
        assert torch.equal(now.transpose(1, 2)[untouched], was.transpose(1, 2)[untouched])


def test_rotary_append_reports_slots_outside_the_cache(dev):
    kc, vc = (torch.zeros(4, 2, 16, 64, device=dev) for _ in range(2))
    x = torch.ones(3, 2, 64, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    slots = torch.tensor([64, 5, 2 ** 40], device=dev)
    q3s.rotary_append(x, x, x, i32([0, 0, 0], dev), frequencies(32, dev), kc, vc, slots, error_word=err)
    assert int(err) == q3s.decode.DECERR_BLOCK_ID
    assert torch.equal(kc[0, :, 5], x[1]) and float(kc.sum()) == float(vc.sum()) == 128.0


def test_rotary_not_finite_values_stay_in_their_pair(dev):
    x = torch.ones(2, 2, 64, device=dev)
    x[0, 1, 3], x[1, 0, 40] = float("nan"), float("inf")
    y = q3s.rotary(x, i32([3, 4], dev), frequencies(16, dev))
    bad = ~torch.isfinite(y)
    assert bad.nonzero().tolist() == [[0, 1, 3], [0, 1, 19], [1, 0, 40]]


def test_rotary_in_place_through_the_c_abi(dev):
    import ctypes as C

    lib = q3s._lib.load()
    x = torch.randn(50, 4, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).bfloat16()
    f, pos = frequencies(64, dev), i32(np.arange(50), dev)
    want = q3s.rotary(x, pos, f)
    d = q3s._lib.RotaryDesc(struct_size=C.sizeof(q3s._lib.RotaryDesc), tokens=50, q_heads=4, dim=128, pairs=64, axes=1, scale=1.0,
                            elem=q3s._lib.ELEM_BF16, positions=pos.data_ptr(), inv_freq=f.data_ptr(), q=x.data_ptr(),
                            q_token_stride=512, q_head_stride=128, out=x.data_ptr(), out_token_stride=512, out_head_stride=128)
    d.sections[0] = 64
    q3s._lib.check(lib.q3s_rotary(C.byref(d), torch.cuda.current_stream().cuda_stream), "q3s_rotary")
    assert torch.equal(x, want)


def test_rotary_object(dev):
    r = q3s.Rotary(128, base=1e6, sections=(24, 20, 20), interleaved=True, device=dev)
    x = torch.randn(5, 2, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    pos = i32(np.arange(15).reshape(3, 5) * 11, dev)
    check_turned(r(x, pos), x, pos, r.inv_freq, sections=(24, 20, 20), interleaved=True)
    with pytest.raises(ValueError):
        q3s.Rotary(128, sections=(1, 2), device=dev)
    with pytest.raises(ValueError):
        q3s.Rotary(128, pairs=65, device=dev)


# ---- rows cut back ----------------------------------------------------------------

def make_trim(rng, rows, block, context, removed, ended=0.0, spare=20, count=None):
    lengths = rng.randint(0, context + 1, rows)
    gone = np.minimum(rng.randint(0, removed + 1, rows), lengths)
    gone = np.where(rng.rand(rows) < ended, lengths, gone)
    held = R.ceil_div(lengths, block)
    pool, width = int(held.sum()) + spare, R.ceil_div(context, block) + 1
    ids = rng.permutation(pool)
    table = np.full((rows, width), -7, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = ids[:int(held.sum())]
    head = int(rng.randint(0, pool))
    ring = np.full(pool, -9, np.int64)
    ring[(head + np.arange(spare)) % pool] = ids[int(held.sum()):]
    return dict(lengths=lengths, removed=gone, table=table, ring=ring, state=[head, spare if count is None else count])


def check_trim(c, dev, block):
    want = R.cache_trim(c["lengths"].tolist(), c["removed"].tolist(), c["table"].tolist(), c["ring"].tolist(), c["state"], block_size=block)
    table, ring, lengths = i32(c["table"], dev), i32(c["ring"], dev), i32(c["lengths"], dev)
    t = q3s.cache_trim(lengths, i32(c["removed"], dev), table, ring, i32(c["state"], dev), block_size=block)
    for name in ("lengths", "free_state", "error_word"):
        assert getattr(t, name).tolist() == want[name], name
    assert ring.tolist() == want["ring"]
    assert torch.equal(table, i32(c["table"], dev)) and torch.equal(lengths, i32(c["lengths"], dev))
    return want


@pytest.mark.parametrize("rows,block,context,removed,ended", [
    (1, 16, 5, 1, 0.0), (1, 1, 9, 9, 1.0), (31, 16, 100, 5, 0.1), (128, 16, 300, 40, 0.1), (129, 48, 300, 9, 0.3),
    (1024, 32, 600, 33, 0.2), (1025, 16, 100, 5, 0.2), (2049, 64, 900, 70, 0.1), (5000, 16, 50, 9, 0.5), (40, 16, 3000, 2900, 0.2)])
def test_trim_matches_definition(dev, rows, block, context, removed, ended):
    assert check_trim(make_trim(np.random.RandomState(rows), rows, block, context, removed, ended), dev, block)["error_word"] == [0]


def test_trim_no_rows_and_odd_values(dev):
    t = q3s.cache_trim(i32([], dev), i32([], dev), torch.zeros(0, 4, dtype=torch.int32, device=dev), i32([1, 2], dev), i32([1, 1], dev),
                       block_size=16)
    assert t.lengths.tolist() == [] and t.free_state.tolist() == [1, 1] and t.error_word.tolist() == [0]
    rng = np.random.RandomState(3)
    c = make_trim(rng, 60, 16, 100, 30)
    c["removed"][7], c["removed"][9], c["lengths"][11] = -4, 1000, 5000
    assert check_trim(c, dev, 16)["error_word"] == [1]
    c = make_trim(rng, 60, 16, 100, 30, ended=0.5)
    c["state"][1] = len(c["ring"]) - 3  # a ring that is nearly full
    assert check_trim(c, dev, 16)["error_word"] == [4]


def test_trim_and_tables_take_turns(dev):
    """What is cut back is drawn again, row for row as the definitions have it."""
    import decode_reference as D

    rng = np.random.RandomState(5)
    B, bs, width = 50, 16, 12
    table, ring, state = np.full((B, width), -1), np.arange(400), [0, 400]
    lengths = np.zeros(B, np.int64)
    t_table, t_ring, t_state, t_len = i32(table, dev), i32(ring, dev), i32(state, dev), i32(lengths, dev)
    for step in range(8):
        new = np.minimum(rng.randint(0, 40, B), width * bs - lengths)
        a = D.cache_tables(lengths.tolist(), new.tolist(), table.tolist(), ring.tolist(), state, block_size=bs, max_tokens=int(new.sum()))
        x = q3s.cache_tables(t_len, i32(new, dev), t_table, t_ring, t_state, block_size=bs, max_tokens=int(new.sum()))
        assert x.slot_map.tolist() == a["slot_map"].tolist() and x.error_word.item() == a["error_word"][0] == 0
        gone = np.minimum(rng.randint(0, 60, B), a["lengths"])
        b = R.cache_trim(a["lengths"].tolist(), gone.tolist(), a["table"].tolist(), a["ring"].tolist(), a["free_state"].tolist(), block_size=bs)
        y = q3s.cache_trim(x.lengths, i32(gone, dev), t_table, t_ring, x.free_state, block_size=bs)
        t_len, t_state = y.lengths, y.free_state
        lengths, table, ring, state = np.array(b["lengths"]), a["table"], np.array(b["ring"]), b["free_state"]
        assert t_ring.tolist() == ring.tolist() and t_state.tolist() == state and t_len.tolist() == lengths.tolist()
        held = [table[r, j] for r in range(B) for j in range(R.ceil_div(int(lengths[r]), bs))]
        free = [ring[(state[0] + j) % 400] for j in range(state[1])]
        assert sorted(held + free) == list(range(400))  # every block is in one place


# ---- verification -------------------------------------------------------------------

def make_verify(seed, rows, queries, vocab, *, dtype=torch.float32, probs=True, keep=0, greedy=0.0, idle=0.0, pad=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.RandomState(seed)
    n = rng.randint(1, queries + 1, rows)
    n[0] = queries
    n[1:][rng.rand(rows - 1) < idle] = 0
    offsets = np.concatenate([[0], np.cumsum(n)]).astype(np.int64)
    T = int(offsets[-1])
    logits = torch.randn(T + pad, vocab, generator=g) * spread
    drafter = logits + torch.randn(T + pad, vocab, generator=g)
    if 0 < keep < vocab:
        logits = torch.where(logits < logits.topk(keep, 1).values[:, -1:], -torch.inf, logits)
    q = torch.softmax(drafter, 1).roll(1, 0)
    ids = torch.multinomial(q, 1, generator=g)[:, 0] if probs else q.argmax(1)
    heat = np.where(rng.rand(rows) < greedy, 0.0, 0.8).astype(np.float32)
    return dict(logits=logits.to(dtype), ids=ids, offsets=offsets, uniforms=torch.rand(T + pad, generator=g), probs=q if probs else None,
                heat=heat, slot_map=None)


def check_verify(c, dev, logits=None, probs=None):
    """`logits` / `probs`: the same values on the GPU in another layout."""
    want = R.verify_drafts(c["logits"].float().numpy(), c["ids"].tolist(), c["offsets"].tolist(), c["uniforms"].tolist(),
                           None if c["probs"] is None else c["probs"].numpy(), c["heat"].tolist(),
                           None if c["slot_map"] is None else c["slot_map"].tolist())
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    r = q3s.verify_drafts(c["logits"].to(dev) if logits is None else logits, c["ids"].to(dev), i32(c["offsets"], dev),
                          c["uniforms"].to(dev), draft_probs=(None if c["probs"] is None else c["probs"].to(dev)) if probs is None else probs,
                          temperature=torch.as_tensor(c["heat"], device=dev), error_word=err,
                          slot_map=None if c["slot_map"] is None else c["slot_map"].to(dev))
    for name in ("accepted", "rejected", "next_ids", "tokens"):
        assert getattr(r, name).tolist() == want[name], name
    assert int(err) == want["error"]
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,queries,vocab,probs,keep,greedy", [
    (1, 1, 1, True, 0, 0.0), (3, 2, 2, True, 0, 0.0), (20, 3, 7, False, 0, 0.3), (40, 5, 100, True, 0, 0.2), (1, 5, 2048, True, 50, 0.0),
    (200, 6, 2051, False, 50, 0.2), (64, 4, 8192, True, 0, 0.1), (30, 4, 8193, True, 0, 0.1), (9, 20, 1000, True, 0, 0.0),
    (3, 40, 300, False, 0, 0.0), (12, 4, 40001, True, 0, 0.2), (5, 3, 70001, False, 0, 0.0), (2, 2, 1 << 18, True, 0, 0.0)])
def test_verify_matches_definition(dev, rows, queries, vocab, probs, keep, greedy, dtype):
    want = check_verify(make_verify(rows + vocab, rows, queries, vocab, dtype=dtype, probs=probs, keep=keep, greedy=greedy), dev)
    assert want["error"] == 0


def test_verify_idle_and_refused_rows_and_padding(dev):
    c = make_verify(1, 60, 5, 500, idle=0.3, pad=17)
    check_verify(c, dev)
    slots = torch.arange(c["logits"].shape[0])
    for b in (3, 10, 59):
        if c["offsets"][b] < c["offsets"][b + 1]:
            slots[c["offsets"][b + 1] - 1] = -1
    slots[int(c["offsets"][-1]):] = -1
    c["slot_map"] = slots
    want = check_verify(c, dev)
    assert 0 in want["accepted"] and want["tokens"][-17:] == [-1] * 17


def test_verify_places_before_the_first_row(dev):
    g = torch.Generator().manual_seed(44)
    logits, ids, u = torch.randn(600, 50, generator=g) * 2, torch.randint(0, 50, (600,), generator=g), torch.rand(600, generator=g)
    for offsets in ([530, 540, 540, 541], [600, 600]):
        rows = len(offsets) - 1
        want = R.verify_drafts(logits.numpy(), ids.tolist(), offsets, u.tolist(), None, [1.0] * rows)
        on_gpu = logits.to(dev), ids.to(dev), i32(offsets, dev), u.to(dev)
        torch.full((600,), 7, dtype=torch.int64, device=dev)  # freed: what the next allocation of that size finds
        r = q3s.verify_drafts(*on_gpu)
        for name in ("accepted", "rejected", "next_ids", "tokens"):
            assert getattr(r, name).tolist() == want[name], name


def test_verify_no_rows(dev):
    z = torch.zeros(3, 10, device=dev)
    r = q3s.verify_drafts(z, torch.zeros(3, dtype=torch.int64, device=dev), i32([0], dev), z[:, 0].contiguous())
    assert r.tokens.tolist() == [-1] * 3 and r.accepted.numel() == r.next_ids.numel() == 0
    r = q3s.verify_drafts(z[:0], torch.zeros(0, dtype=torch.int64, device=dev), i32([0, 0, 0], dev), z[:0, 0].contiguous())
    assert r.next_ids.tolist() == [-1, -1] and r.rejected.tolist() == [0, 0]


@pytest.mark.parametrize("dtype,shift", [(torch.bfloat16, 1), (torch.bfloat16, 8), (torch.float16, 3), (torch.float32, 1), (torch.float32, 4)])
def test_verify_logits_of_any_alignment(dev, dtype, shift):
    c = make_verify(2, 30, 4, 700, dtype=dtype)
    T = c["logits"].shape[0]
    wide = torch.full((T, 711), float("nan"), dtype=dtype, device=dev)
    wide[:, shift:shift + 700] = c["logits"].to(dev)
    q = torch.full((T, 720), float("nan"), device=dev)
    q[:, 1:701] = c["probs"].to(dev)
    check_verify(c, dev, wide[:, shift:shift + 700], q[:, 1:701])


@pytest.mark.parametrize("vocab", [50, 3000, 20000])
def test_verify_decisions_next_to_the_border(dev, vocab):
    """Uniforms that are the 32-bit numbers next to p(draft): 32-bit sums cannot tell; the 64-bit ones decide."""
    c = make_verify(3, 80, 6, vocab, probs=False)
    logits, ids, off = c["logits"].double().numpy(), c["ids"].numpy(), c["offsets"]
    u = c["uniforms"].numpy()
    held = 0
    for b in range(80):
        for t in range(off[b], off[b + 1] - 1):
            x = logits[t] / float(c["heat"][b])
            p = np.exp(x - x.max())
            near = np.float32(p[ids[t + 1]] / p.sum())
            u[t + 1] = near if (b + t) % 3 else np.nextafter(near, np.float32(0), dtype=np.float32)
    want = check_verify(c, dev)
    held = sum(want["accepted"])
    assert held > 20 and sum(want["rejected"]) > 20


def test_verify_draws_at_both_ends(dev):
    for u in (0.0, 1.0 - 2.0 ** -24):
        c = make_verify(4, 50, 3, 900)
        c["uniforms"][torch.as_tensor(c["offsets"][:-1])] = u
        check_verify(c, dev)
    c = make_verify(5, 50, 3, 900)
    c["logits"][:, 0] = -torch.inf
    c["logits"][:, 890:] = -torch.inf
    c["uniforms"][:] = 0.0
    check_verify(c, dev)


def test_verify_nothing_left_of_p(dev):
    """Draft probabilities that are too large everywhere: the draw is from p."""
    c = make_verify(6, 40, 3, 600)
    p = torch.softmax(c["logits"].double() / 0.8, 1)
    c["probs"] = (4 * p).roll(1, 0).float()
    c["uniforms"][:] = 0.6
    want = check_verify(c, dev)
    assert sum(want["accepted"]) == 0


def test_verify_odd_temperatures(dev):
    c = make_verify(7, 12, 4, 300)
    c["heat"] = np.array([0.0, -1.0, np.nan, 1e-31, 1e-3, 1e-20, 50.0, 1e30, 0.5, 1.0, 2.0, 1e-10], np.float32)
    check_verify(c, dev)
    r = q3s.verify_drafts(c["logits"].to(dev), c["ids"].to(dev), i32(c["offsets"], dev), c["uniforms"].to(dev), temperature=0.0)
    s = q3s.verify_drafts(c["logits"].to(dev), c["ids"].to(dev), i32(c["offsets"], dev), c["uniforms"].to(dev),
                          temperature=torch.zeros(12, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(r, s))


def test_verify_greedy_ties_go_to_the_lowest_index(dev):
    c = make_verify(8, 30, 4, 5000, probs=False)
    c["logits"] = torch.round(c["logits"].clamp(max=4))
    c["heat"][:] = 0
    check_verify(c, dev)


def test_verify_logits_without_a_distribution(dev):
    c = make_verify(9, 8, 3, 200)
    first = c["offsets"][:-1]
    c["logits"][first[0], 70] = float("nan")
    c["logits"][first[1]] = -torch.inf
    c["logits"][first[2], 50], c["logits"][first[2], 60] = torch.inf, torch.inf
    c["logits"][first[3]] = float("nan")
    c["heat"][:2] = [0.8, 0.0]
    assert check_verify(c, dev)["error"] == 64
    c = make_verify(10, 8, 3, 200)  # a place that the row does not reach
    c["uniforms"][1] = 1.0 - 2.0 ** -24
    c["logits"][0, c["ids"][1]] = -20.0
    c["logits"][1, 5] = float("nan")
    assert check_verify(c, dev)["error"] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab,places", [
    (2051, (0, 1, 2, 3, 2047, 2050)),  # places that do not begin on 16 bytes: the first entries, taken alone, and the last
    (2048, (0, 5, 1023, 2047)),
    (40001, (0, 1, 39999, 40000))])
@pytest.mark.parametrize("around", ["finite", "left out", "nothing else"])
def test_verify_a_nan_wherever_it_stands(dev, dtype, vocab, places, around):
    """A place that holds a NaN has no distribution: also where the NaN is the first entry that a thread sees, alone or among
    what top-k left out (-inf)."""
    c = make_verify(45, 2 * len(places), 3, vocab, dtype=dtype, probs=False)
    logits, first = c["logits"], c["offsets"][:-1]
    for i, at in enumerate(places):
        for t in (int(first[2 * i]), int(first[2 * i + 1])):  # two rows, whose places begin at other addresses
            if around == "left out":
                logits[t, max(at - 300, 0):at + 300] = -torch.inf
            elif around == "nothing else":
                keep = (at + vocab // 2) % vocab
                x = float(logits[t, keep])
                logits[t] = -torch.inf
                logits[t, keep] = x
            logits[t, at] = float("nan")
    c["heat"][1::4] = 0.0  # some greedy
    want = check_verify(c, dev)
    assert want["error"] == 64 and want["accepted"] == [0] * (2 * len(places))


@pytest.mark.parametrize("probs", [True, False])
def test_verify_drafts_outside_the_vocabulary(dev, probs):
    c = make_verify(11, 20, 4, 200, probs=probs)
    ids = c["ids"]
    for b, d in ((0, -1), (4, 200), (7, 2 ** 40)):
        if c["offsets"][b] + 1 < c["offsets"][b + 1]:
            ids[c["offsets"][b] + 1] = d
    assert check_verify(c, dev)["error"] == 64


def test_verify_large_logits_and_wide_spread(dev):
    check_verify(make_verify(12, 40, 4, 3000, spread=300.0), dev)
    c = make_verify(13, 40, 4, 3000)
    c["logits"] += 30000.0
    check_verify(c, dev)
    c["logits"][:, 1000:] = -1e9
    check_verify(c, dev)


def test_verify_captured_step_follows_its_inputs(dev):
    """A captured graph of verification and cut, replayed on other inputs of the same sizes."""
    cases = [make_verify(s, 6, 4, 400) for s in (20, 21)]
    T = max(c["logits"].shape[0] for c in cases)
    logits, probs = torch.zeros(T, 400, device=dev), torch.zeros(T, 400, device=dev)
    ids, u, off = torch.zeros(T, dtype=torch.int64, device=dev), torch.zeros(T, device=dev), i32(np.zeros(7), dev)
    lengths, ring, state = i32([64] * 6, dev), i32(np.arange(40), dev), i32([0, 4], dev)
    table = i32(np.arange(24).reshape(6, 4) + 10, dev)
    q3s.cache_trim(lengths, i32([0] * 6, dev), table, ring.clone(), state, block_size=16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        r = q3s.verify_drafts(logits, ids, off, u, draft_probs=probs, temperature=0.8)
        t = q3s.cache_trim(lengths, r.rejected, table, ring, state, block_size=16)
    for c in cases:
        n = c["logits"].shape[0]
        for to, x in ((logits, c["logits"]), (probs, c["probs"]), (ids, c["ids"]), (u, c["uniforms"])):
            to[:n] = x.to(dev)
        off.copy_(i32(c["offsets"], dev))
        graph.replay()
        heat = float(np.float32(0.8))
        want = R.verify_drafts(logits.cpu().numpy(), ids.tolist(), c["offsets"].tolist(), u.tolist(), probs.cpu().numpy(), [heat] * 6)
        assert r.next_ids.tolist() == want["next_ids"] and r.rejected.tolist() == want["rejected"] and r.tokens.tolist() == want["tokens"]
        assert t.lengths.tolist() == [64 - x for x in want["rejected"]]


# ---- a step of several tokens, as it is used ----------------------------------------

def test_steps_with_drafts_on_a_paged_cache(dev):
    """Prompt, then steps of drafts: tables, turn and append, attention, verification and cut, each against its definition
    on the state that the step has."""
    B, hq, hk, dim, bs, V, prefix = 5, 4, 2, 64, 16, 300, 20
    rng = np.random.RandomState(0)
    g = torch.Generator(device=dev).manual_seed(0)
    cache = q3s.PagedCache(B, 60, layers=1, kv_heads=hk, dim=dim, block_size=bs, max_blocks=9, prefix_blocks=2, device=dev)
    rotary = q3s.Rotary(dim, device=dev)
    kv = torch.randn(2, prefix, hk, dim, device=dev, generator=g).bfloat16()
    cache.write_prefix(0, kv[0], kv[1])
    rows = [torch.zeros(0, hk, dim, dtype=torch.bfloat16, device=dev) for _ in range(B)]  # turned keys, as they should be stored
    for step in range(6):
        new = rng.randint(20, 60, B) if step == 0 else rng.randint(0, 5, B)
        new[0] = max(new[0], 1)
        T = int(new.sum())
        t = cache.step(i32(new, dev), max_tokens=T + 3)
        qkv = torch.randn(T + 3, hq + 2 * hk, dim, device=dev, generator=g).bfloat16()
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        turned = cache.append_rotary(0, q, k, v, rotary, cache.positions)
        before = [len(r) for r in rows]
        pos = np.concatenate([prefix + before[b] + np.arange(new[b]) for b in range(B)] + [np.full(3, prefix)])
        check_turned(turned, q, i32(pos, dev), rotary.inv_freq)
        off = np.concatenate([[0], np.cumsum(new)])
        stored = q3s.rotary(k, i32(pos, dev), rotary.inv_freq)
        for b in range(B):
            rows[b] = torch.cat([rows[b], stored[off[b]:off[b + 1]]])
        window = 0 if step % 2 else 50
        out = cache.attend_chunk(0, turned, window=window)
        want, _, spread, mass = R.chunk_attention(turned, cache.k[0], cache.v[0], off.tolist(), cache.table, cache.lengths.tolist(),
                                                  cache.prefix, prefix, dim ** -0.5, window)
        tol = 2.0 ** -8 * want.abs() + 1.02 * 2.0 ** -8 * spread + 2.0 ** -16 * mass
        assert bool(((out.double() - want).abs() <= tol).all()) and not out[T:].any()
        for b in range(B):  # the row's keys are where its table says
            j = torch.arange(len(rows[b]), device=dev)
            assert torch.equal(cache.k[0][cache.table[b, j // bs].long(), :, j % bs], rows[b])
        c = dict(logits=torch.randn(T + 3, V, generator=torch.Generator().manual_seed(step)) * 2, offsets=off, slot_map=t.slot_map.cpu(),
                 uniforms=torch.rand(T + 3, generator=torch.Generator().manual_seed(step)), probs=None, heat=np.full(B, 0.5, np.float32))
        c["ids"] = c["logits"].argmax(1).roll(1, 0)
        verdict = check_verify(c, dev)
        r = q3s.verify_drafts(c["logits"].to(dev), c["ids"].to(dev), t.query_offsets, c["uniforms"].to(dev), temperature=0.5,
                              slot_map=t.slot_map)
        assert r.rejected.tolist() == verdict["rejected"]
        cache.trim(r.rejected)
        for b in range(B):
            rows[b] = rows[b][:len(rows[b]) - verdict["rejected"][b]]
        assert cache.lengths.tolist() == [len(r) for r in rows]
        held = [int(cache.table[b, j]) for b in range(B) for j in range(R.ceil_div(len(rows[b]), bs))]
        head, count = cache.ring_state.tolist()
        free = [int(cache.ring[(head + j) % 58]) for j in range(count)]
        assert sorted(held + free) == list(range(2, 60)) and int(cache.error_word) == 0 == int(t.error_word)


def test_example_of_draft_steps_runs(dev):
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "draft_step.py"
    spec = importlib.util.spec_from_file_location("draft_step", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    tokens, held, cache = module.main(rows=6, steps=4, drafts=3, prompt=21)
    assert tokens.shape == (6, 1 + 4 * 4) and held.shape == (4, 6) and int(held.min()) >= 0 and int(held.max()) <= 3
    # the prompt, and of each step the token that was settled and the drafts that held
    assert cache.lengths.tolist() == (21 + 4 + held.sum(0)).tolist()
    assert (tokens >= 0).sum(1).tolist() == (1 + 4 + held.sum(0)).tolist() and int(tokens.max()) < 1024
