"""The decode step's operators beside the sampler, on the GPU, against their
definitions in Python integers and float64 (tests/decode_reference.py).

Tolerances, from the arithmetic:

* tables, append, quantisation: equal.
* 8-bit product: the sum is exact; its conversion to fp32, the two scale
  products and the bias addition round by 2^-24 each, the output by the unit
  roundoff r of its type (2^-8 bf16, 2^-11 f16, 2^-24 fp32):
  |err| <= (r + 2^-22) (|product| + |bias|).
* attention: with u = half the unit roundoff, |err| <= u |out| + (u + 2^-16)
  sum p |v|.  Rounding the output takes 2 u |out|, which is covered since sum
  p |v| >= |out|; ex2 and the fp32 sums take less than 2^-16 of sum p |v| at
  these score sizes; rounding the probabilities has to fit in what is left, u
  (sum p |v| - |out|).  A probability below 2^-14 of the largest is subnormal
  in f16 and off by up to 2^-25, at most N of them.  lse: |err| <= 2^-16 (1 +
  |lse|)."""
import numpy as np
import pytest
import torch

import decode_reference as R
import q3s

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def dev(cuda_device):
    q3s.load_torch_ops()
    return cuda_device


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


# ---- tables -----------------------------------------------------------------

def make_tables(rng, rows, block, *, context=100, new=3, width=None, spare=50, released=0.0, count=None):
    ctx = rng.randint(0, context + 1, rows)
    fresh = rng.randint(0, new + 1, rows)
    gone = (rng.rand(rows) < released).astype(np.uint8)
    width = width or R.ceil_div(context + new, block) + 1
    held = R.ceil_div(ctx, block)
    pool = int(held.sum()) + R.ceil_div(fresh, block).sum() + rows + spare
    ids = rng.permutation(pool)
    table = np.full((rows, width), -7, np.int64)
    used = np.arange(width)[None, :] < held[:, None]
    table[used] = ids[: int(used.sum())]
    free = ids[int(used.sum()):]
    head = int(rng.randint(0, pool))
    ring = np.full(pool, -9, np.int64)
    ring[(head + np.arange(len(free))) % pool] = free
    return dict(context=ctx, new=fresh, table=table, ring=ring, state=[head, len(free) if count is None else count], gone=gone)


def check_tables(c, dev, block, max_tokens=None, released=True):
    total = int(np.maximum(c["new"], 0).sum())
    max_tokens = total + 5 if max_tokens is None else max_tokens
    want = R.cache_tables(c["context"].tolist(), c["new"].tolist(), c["table"].tolist(), c["ring"].tolist(), c["state"],
                          block_size=block, max_tokens=max_tokens, released=c["gone"].tolist() if released else None)
    table, ring = i32(c["table"], dev), i32(c["ring"], dev)
    gone = torch.as_tensor(c["gone"], device=dev).bool() if released else None
    t = q3s.cache_tables(i32(c["context"], dev), i32(c["new"], dev), table, ring, i32(c["state"], dev), block_size=block,
                         max_tokens=max_tokens, released=gone)
    for name in ("query_offsets", "lengths", "free_state", "error_word", "slot_map", "positions"):
        np.testing.assert_array_equal(getattr(t, name).cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(table.cpu().numpy(), want["table"])
    np.testing.assert_array_equal(ring.cpu().numpy(), want["ring"])
    return want


@pytest.mark.parametrize("rows,block,context,new,released", [
    (1, 16, 5, 1, 0.0), (1, 1, 3, 2, 1.0), (31, 16, 100, 1, 0.1), (128, 16, 300, 2, 0.1), (129, 48, 300, 40, 0.3),
    (700, 16, 200, 90, 0.05), (1024, 32, 600, 3, 0.2), (1025, 16, 100, 5, 0.2), (2049, 64, 900, 70, 0.1),
    (5000, 16, 50, 9, 0.5), (40, 16, 3000, 2000, 0.2)])
def test_tables_match_definition(dev, rows, block, context, new, released):
    rng = np.random.RandomState(rows + block + new)
    want = check_tables(make_tables(rng, rows, block, context=context, new=new, released=released), dev, block)
    assert want["error_word"][0] == 0


def test_tables_no_rows_no_tokens(dev):
    c = make_tables(np.random.RandomState(0), 3, 16, new=0)
    check_tables(c, dev, 16, max_tokens=0)
    e = dict(dev=dev, dtype=torch.int32)
    t = q3s.cache_tables(i32([], dev), i32([], dev), torch.zeros(0, 4, dtype=torch.int32, device=dev), i32([1, 2], dev),
                         i32([1, 1], dev), block_size=16, max_tokens=3)
    assert t.query_offsets.tolist() == [0] and t.slot_map.tolist() == [-1] * 3 and t.free_state.tolist() == [1, 1]


@pytest.mark.parametrize("rows", [5, 300, 3000])
def test_tables_pool_runs_out(dev, rows):
    """Rows are served in order until the ring cannot; later rows that need no block still get their slots."""
    rng = np.random.RandomState(rows)
    c = make_tables(rng, rows, 16, context=100, new=20, released=0.1)
    c["state"][1] = rows // 3
    want = check_tables(c, dev, 16)
    assert want["error_word"][0] == R_POOL
    assert (want["slot_map"] >= 0).any()
    c["state"][1] = 0
    check_tables(c, dev, 16)


R_POOL, R_TABLE, R_LENGTHS, R_TOKENS = 4, 2, 1, 8


def test_tables_row_outgrows_its_table_and_bad_lengths(dev):
    rng = np.random.RandomState(1)
    c = make_tables(rng, 60, 16, context=100, new=30, width=7)
    assert check_tables(c, dev, 16)["error_word"][0] == R_TABLE
    c = make_tables(rng, 60, 16, context=60, new=30)
    c["context"][7] = -4
    c["new"][11] = -3
    assert check_tables(c, dev, 16)["error_word"][0] & R_LENGTHS
    c = make_tables(rng, 60, 16, context=60, new=30)
    c["context"][3] = 10 ** 9
    assert check_tables(c, dev, 16)["error_word"][0] & R_LENGTHS


def test_tables_fewer_slots_than_tokens(dev):
    c = make_tables(np.random.RandomState(2), 200, 16, new=30)
    assert check_tables(c, dev, 16, max_tokens=1000)["error_word"][0] == R_TOKENS


def test_tables_sums_past_31_bits_saturate(dev):
    c = make_tables(np.random.RandomState(3), 4, 16, new=1)
    new = i32([2 ** 31 - 1, 2 ** 31 - 1, 5, 1], dev)
    t = q3s.cache_tables(i32(c["context"], dev), new, i32(c["table"], dev), i32(c["ring"], dev), i32(c["state"], dev),
                         block_size=16, max_tokens=64)
    assert t.query_offsets.tolist() == [0] + [2 ** 31 - 1] * 4
    assert int(t.error_word) & R_TOKENS and int(t.error_word) & R_TABLE
    assert t.slot_map.tolist() == [-1] * 64


@pytest.mark.parametrize("rows", [40, 1500])
def test_tables_released_row_is_readmitted_in_the_same_step(dev, rows):
    rng = np.random.RandomState(4)
    c = make_tables(rng, rows, 16, context=900, new=700, released=0.5, spare=5)
    c["new"][:] = rng.randint(1, 700, rows)
    c["state"][1] = len(c["ring"]) - int(R.ceil_div(c["context"], 16).sum())
    check_tables(c, dev, 16)


def test_tables_strided_table_and_many_steps(dev):
    """A run of steps on the same device state equals the definition, step by step."""
    rng = np.random.RandomState(5)
    B, block, width, pool = 70, 16, 40, 800
    wide = torch.full((B, width + 9), -1, dtype=torch.int32, device=dev)
    table = wide[:, :width]
    ring, state = i32(rng.permutation(pool), dev), i32([700, pool], dev)
    lengths = i32(np.zeros(B), dev)
    for step in range(40):
        new = np.where(rng.rand(B) < 0.1, rng.randint(0, 200, B), rng.randint(0, 2, B))
        gone = rng.rand(B) < 0.15
        want = R.cache_tables(lengths.tolist(), new.tolist(), table.tolist(), ring.tolist(), state.tolist(),
                              block_size=block, max_tokens=int(new.sum()), released=gone.tolist())
        t = q3s.cache_tables(lengths, i32(new, dev), table, ring, state, block_size=block, max_tokens=int(new.sum()),
                             released=torch.as_tensor(gone, device=dev))
        lengths, state = t.lengths, t.free_state
        for name in ("query_offsets", "lengths", "free_state", "error_word", "slot_map", "positions"):
            np.testing.assert_array_equal(getattr(t, name).cpu().numpy(), want[name], err_msg=f"{step} {name}")
        np.testing.assert_array_equal(table.cpu().numpy(), want["table"])
        np.testing.assert_array_equal(ring.cpu().numpy(), want["ring"])
    assert bool((wide[:, width:] == -1).all())


# ---- append -------------------------------------------------------------------

@pytest.mark.parametrize("tokens,heads,dim,block,dtype,skip", [
    (1, 8, 128, 16, torch.bfloat16, 0), (7, 2, 64, 32, torch.float16, 0.3), (300, 8, 128, 16, torch.float16, 0.1),
    (3000, 4, 128, 64, torch.bfloat16, 0.0), (50, 3, 20, 5, torch.float32, 0.1), (50, 1, 7, 3, torch.bfloat16, 0.1)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_append(dev, tokens, heads, dim, block, dtype, skip, layout):
    rng = np.random.RandomState(tokens)
    blocks = R.ceil_div(tokens, block) + 2
    g = torch.Generator(device=dev).manual_seed(tokens)
    qkv = torch.randn(tokens, 4 * heads, dim, device=dev, generator=g).to(dtype)
    k, v = qkv[:, heads:2 * heads], qkv[:, 3 * heads:]
    shape = (blocks, heads, block, dim) if layout == "heads" else (blocks, block, heads, dim)
    caches = [torch.randn(shape, device=dev, generator=g).to(dtype) for _ in range(2)]
    if layout == "tokens":
        caches = [c.transpose(1, 2) for c in caches]
    slots = rng.permutation(blocks * block)[:tokens]
    slots = np.where(rng.rand(tokens) < skip, -1, slots)
    want = [c.clone() for c in caches]
    for x, c in zip((k, v), want):
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                c[s // block, :, s % block] = x[t]
    q3s.cache_append(k, v, *caches, torch.as_tensor(slots, device=dev))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_append_slot_outside_the_cache_is_skipped_and_reported(dev):
    k = torch.ones(3, 1, 8, device=dev)
    cache = torch.zeros(2, 1, 4, 8, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    q3s.cache_append(k, k, cache, cache.clone(), torch.tensor([0, 8, 2 ** 40], device=dev), error_word=err)
    assert int(err) == 16 and float(cache.sum()) == 8
    q3s.cache_append(k[:0], k[:0], cache, cache, torch.zeros(0, dtype=torch.int64, device=dev))


def test_append_more_tokens_than_one_grid_takes(dev):
    """Rows of 257 elements, one token a group: 262140 tokens fill a grid."""
    T = 262140 + 77
    k = torch.randint(-1000, 1000, (T, 1, 257), dtype=torch.int16, device=dev).view(torch.bfloat16)
    v = torch.randint(-1000, 1000, (T, 1, 257), dtype=torch.int16, device=dev).view(torch.bfloat16)
    kc = torch.zeros(T // 7 + 1, 1, 7, 257, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    slots = torch.arange(T, device=dev).flip(0)
    q3s.cache_append(k, v, kc, vc, slots)
    for x, c in ((k, kc), (v, vc)):
        assert torch.equal(c.view(torch.int16).reshape(-1, 257)[:T].flip(0), x.view(torch.int16).reshape(T, 257))


# ---- attention ------------------------------------------------------------------

def make_attention(dev, *, n, lengths, prefix, q_heads, kv_heads, dim, block, dtype, seed=0, layout="heads", spread=1.0,
                   poison=True):
    """Rows with n[b] queries and lengths[b] own tokens.  With `poison` every
    cache element that no query may see is NaN or infinite."""
    rng = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    n, lengths = np.asarray(n), np.asarray(lengths)
    B, T = len(n), int(n.sum())
    held, shared = R.ceil_div(lengths, block), R.ceil_div(prefix, block)
    width = int(held.max()) + 1 if B else 1
    blocks = int(held.sum()) + shared + 3
    ids = rng.permutation(blocks)
    table = np.full((B, width), -1, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = ids[shared:shared + int(held.sum())]
    k = spread * torch.randn(blocks, kv_heads, block, dim, generator=g)
    v = torch.randn(blocks, kv_heads, block, dim, generator=g)
    if poison:
        live = torch.zeros(blocks, block, dtype=torch.bool)
        for b in range(B):
            for j in range(int(lengths[b])):
                live[table[b, j // block], j % block] = True
        for j in range(prefix):
            live[ids[j // block], j % block] = True
        dead = ~live[:, None, :, None]
        k = torch.where(dead, torch.tensor(float("nan")), k)
        v = torch.where(dead, torch.tensor(float("inf")), v)
    k, v = k.to(dtype).to(dev), v.to(dtype).to(dev)
    if layout == "tokens":
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    qkv = torch.randn(T, q_heads + 2, dim, generator=g).to(dtype).to(dev)
    return dict(q=qkv[:, :q_heads], k=k, v=v, offsets=i32(np.concatenate([[0], np.cumsum(n)]), dev), table=i32(table, dev),
                lengths=i32(lengths, dev), prefix_blocks=i32(ids[:shared], dev), prefix=prefix, scale=dim ** -0.5)


def run_attention(c, **kw):
    return q3s.prefix_attention(c["q"], c["k"], c["v"], c["offsets"], c["table"], c["lengths"],
                                prefix_blocks=c["prefix_blocks"], prefix_length=c["prefix"], scale=c["scale"],
                                return_lse=True, **kw)


def check_attention(c, out, lse):
    want, want_lse, mass = R.prefix_attention(c["q"].cpu(), c["k"].cpu(), c["v"].cpu(), c["offsets"].cpu(), c["table"].cpu(),
                                              c["lengths"].cpu(), c["prefix_blocks"].cpu(), c["prefix"], c["scale"])
    u = HALF_UNIT[c["q"].dtype]
    keys = c["prefix"] + int(c["lengths"].max()) if len(c["lengths"]) else c["prefix"]
    tol = u * want.abs() + (u + 2.0 ** -16) * mass + 1e-7
    if c["q"].dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * 5
    d = (out.cpu().double() - want).abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max())} of the tolerance, max |d| {float(d.max())}"
    got = lse.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want_lse))
    fin = ~torch.isinf(want_lse)
    assert bool(((got - want_lse)[fin].abs() <= 2.0 ** -16 * (1 + want_lse[fin].abs())).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,n,length", [(64, 2, 3, 19), (128, 4, 9, 40), (64, 1, 20, 20), (128, 1, 33, 33)])
def test_attention_odd_values_reach_only_who_sees_them(dev, dtype, dim, group, n, length):
    """NaN and infinities in V of the step's own tokens: a query before them is
    as if they were finite; one that sees them has them, in their dims."""
    c = make_attention(dev, n=[n, 2], lengths=[length, 5], prefix=7, q_heads=2 * group, kv_heads=2, dim=dim,
                       block=16, dtype=dtype, poison=False)
    clean = dict(c, v=c["v"].clone())
    table = c["table"].cpu()
    for back, x in ((1, float("nan")), (2, float("inf"))):  # the row's last token and the one before it
        j = length - back
        c["v"][int(table[0, j // 16]), :, j % 16, 3::5] = x
    out, lse = run_attention(c)
    hit = torch.zeros(dim, dtype=torch.bool)
    hit[3::5] = True
    assert bool(torch.isposinf(out[n - 2][..., hit]).all()) and bool(torch.isnan(out[n - 1][..., hit]).all())
    out[n - 2:n, :, 3::5] = run_attention(clean)[0][n - 2:n, :, 3::5]  # checked above
    check_attention(clean, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_heads,kv_heads,dim,block", [(16, 8, 128, 16), (8, 1, 64, 32), (3, 3, 128, 64), (32, 2, 64, 128),
                                                        (10, 2, 128, 16)])
@pytest.mark.parametrize("prefix,lengths", [
    (0, [1]), (1, [1]), (33, [1, 2, 17, 31, 32, 33, 64, 100]), (300, [5]), (0, [700, 3, 90]), (1000, [40, 1, 129])])
def test_attention_one_query_a_row(dev, dtype, q_heads, kv_heads, dim, block, prefix, lengths):
    c = make_attention(dev, n=[1] * len(lengths), lengths=lengths, prefix=prefix, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                       block=block, dtype=dtype, seed=prefix + len(lengths))
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("n,lengths", [([3, 0, 1, 8], [3, 50, 77, 64]), ([40], [40]), ([17, 1, 0], [200, 1, 0]),
                                       ([0, 0, 5], [10, 0, 5]), ([100, 30], [300, 31])])
@pytest.mark.parametrize("prefix", [0, 65, 513])
@pytest.mark.parametrize("dim,dtype,layout", [(128, torch.bfloat16, "heads"), (64, torch.float16, "tokens")])
def test_attention_many_queries_a_row(dev, n, lengths, prefix, dim, dtype, layout):
    c = make_attention(dev, n=n, lengths=lengths, prefix=prefix, q_heads=12, kv_heads=4, dim=dim, block=16, dtype=dtype,
                       layout=layout, seed=sum(n))
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("rows,prefix,group", [(64, 500, 2), (150, 1030, 4), (300, 257, 1), (33, 2000, 16), (257, 64, 3)])
@pytest.mark.parametrize("dim,dtype,block", [(128, torch.bfloat16, 16), (64, torch.float16, 64), (128, torch.float16, 128)])
def test_attention_large_batch_on_a_prefix(dev, rows, prefix, group, dim, dtype, block):
    rng = np.random.RandomState(rows)
    lengths = rng.randint(1, 30, rows)
    c = make_attention(dev, n=[1] * rows, lengths=lengths, prefix=prefix, q_heads=group * 2, kv_heads=2, dim=dim, block=block,
                       dtype=dtype, seed=rows)
    check_attention(c, *run_attention(c))


def test_attention_queries_that_see_nothing(dev):
    """No prefix, no own tokens (or more queries than tokens): 0 and -inf."""
    c = make_attention(dev, n=[2, 1, 4], lengths=[2, 0, 2], prefix=0, q_heads=4, kv_heads=2, dim=64, block=16,
                       dtype=torch.bfloat16)
    out, lse = run_attention(c)
    check_attention(c, out, lse)
    assert float(out[2:5].float().abs().sum()) == 0 and bool((lse[2:5] == -float("inf")).all())


def test_attention_tokens_past_the_last_row(dev):
    """A padded batch: queries beyond the rows' see nothing, whatever they hold."""
    c = make_attention(dev, n=[1, 1], lengths=[20, 5], prefix=40, q_heads=4, kv_heads=2, dim=64, block=16, dtype=torch.bfloat16)
    pad = torch.full((3, 4, 64), float("nan"), dtype=torch.bfloat16, device=dev)
    out, lse = run_attention(c)
    c["q"] = torch.cat([c["q"], pad])
    out2, lse2 = run_attention(c)
    assert torch.equal(out2[:2], out) and torch.equal(lse2[:2], lse)
    assert float(out2[2:].float().abs().sum()) == 0 and bool((lse2[2:] == -float("inf")).all())


@pytest.mark.parametrize("rows", [2, 200])
def test_attention_large_scores(dev, rows):
    """Scores of hundreds: probabilities underflow to a few keys, the running maximum moves."""
    c = make_attention(dev, n=[1] * rows, lengths=[150] * rows, prefix=300, q_heads=4, kv_heads=2, dim=64, block=16,
                       dtype=torch.float16, spread=30.0)
    out, lse = run_attention(c)
    want, want_lse, mass = R.prefix_attention(c["q"].cpu(), c["k"].cpu(), c["v"].cpu(), c["offsets"].cpu(), c["table"].cpu(),
                                              c["lengths"].cpu(), c["prefix_blocks"].cpu(), c["prefix"], c["scale"])
    # a score of size s is off by up to 2^-22 s: the probabilities by that, relatively
    s = 30.0 * 64 ** 0.5
    u = 2.0 ** -12
    tol = u * want.abs() + (u + 2.0 ** -20 * s) * mass + 450 * 2.0 ** -25 * 5
    assert bool(((out.cpu().double() - want).abs() <= tol).all())
    assert bool(((lse.cpu().double() - want_lse).abs() <= 2.0 ** -20 * s + 2.0 ** -20 * want_lse.abs()).all())


def test_attention_bad_block_id_and_lengths_are_reported(dev):
    c = make_attention(dev, n=[1, 1], lengths=[20, 40], prefix=0, q_heads=4, kv_heads=2, dim=64, block=16,
                       dtype=torch.bfloat16, poison=False)
    good, _ = run_attention(c)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    c["table"][1, 1] = 10 ** 6
    out, _ = run_attention(c, error_word=err)
    assert int(err) == 16 and torch.equal(out[0], good[0]) and bool(torch.isfinite(out.float()).all())
    err.zero_()
    c["lengths"][1] = 10 ** 8  # cut to the table
    run_attention(c, error_word=err)
    assert int(err) & 1


def test_attention_prefix_split_joins_by_lse(dev):
    """out over prefix and rows = the two parts joined by their lse."""
    c = make_attention(dev, n=[1] * 40, lengths=[30] * 40, prefix=200, q_heads=8, kv_heads=2, dim=128, block=16,
                       dtype=torch.bfloat16, poison=False)
    out, lse = run_attention(c)
    a, la = run_attention(dict(c, prefix=0))
    nothing = i32(np.zeros(40), dev)
    b, lb = run_attention(dict(c, lengths=nothing))
    wa, wb = (torch.exp(x.double() - lse.double())[..., None] for x in (la, lb))
    joined = wa * a.double() + wb * b.double()
    assert float((joined - out.double()).abs().max()) <= 3 * 2.0 ** -9 * float(out.double().abs().max())


def test_attention_same_result_every_time_and_on_another_stream(dev):
    c = make_attention(dev, n=[1] * 90, lengths=list(range(1, 91)), prefix=777, q_heads=8, kv_heads=2, dim=128, block=16,
                       dtype=torch.bfloat16)
    out, lse = run_attention(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            o2, l2 = run_attention(c)
            assert torch.equal(o2, out) and torch.equal(l2, lse)
    torch.cuda.current_stream().wait_stream(s)


def test_attention_in_a_cuda_graph_follows_device_lengths(dev):
    c = make_attention(dev, n=[1] * 20, lengths=[100] * 20, prefix=90, q_heads=4, kv_heads=2, dim=64, block=16,
                       dtype=torch.bfloat16, poison=False)
    run_attention(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = run_attention(c)
    for ln in (1, 37, 100):
        c["lengths"].fill_(ln)
        g.replay()
        torch.cuda.synchronize()
        check_attention(c, out, lse)


def test_attention_cache_past_32_bit_offsets(dev):
    """Blocks whose element offsets pass 2^31 (a 5 GB cache)."""
    block, H, D = 64, 4, 128
    blocks = (2 ** 31 + 2 ** 28) // (H * block * D)
    k = torch.zeros(blocks, H, block, D, dtype=torch.bfloat16, device=dev)
    ids = [blocks - 1, 0, blocks - 2]
    g = torch.Generator(device=dev).manual_seed(1)
    for i in ids:
        k[i] = torch.randn(H, block, D, device=dev, generator=g).to(torch.bfloat16)
    q = torch.randn(70, 2 * H, D, device=dev, generator=g).to(torch.bfloat16)
    table = i32([[ids[0]]] * 70, dev)
    args = dict(query_offsets=i32(np.arange(71), dev), lengths=i32([50] * 70, dev), prefix_length=100, return_lse=True)
    out, lse = q3s.prefix_attention(q, k, k, block_table=table, prefix_blocks=i32([ids[2], ids[1]], dev), **args)
    small = torch.stack([k[i] for i in ids])
    out2, lse2 = q3s.prefix_attention(q, small, small, block_table=i32([[0]] * 70, dev), prefix_blocks=i32([2, 1], dev), **args)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    slots = torch.tensor([blocks * block - 1], device=dev)
    x = torch.ones(1, H, D, dtype=torch.bfloat16, device=dev)
    q3s.cache_append(x, x, k, k, slots)
    assert float(k[-1, :, -1].float().sum()) == H * D and float(k[5].float().abs().sum()) == 0


# ---- 8-bit projections ------------------------------------------------------------

@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 7), (5, 2048), (130, 1040), (2, 5000), (64, 4096), (1, 20000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_rows(dev, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    for y in (x, torch.cat([x, x], 1)[:, cols // 2:cols // 2 + cols] if cols > 2 else x):  # and unaligned, strided rows
        v, s = q3s.quantize_rows(y.to(dev) if y is x else torch.cat([x, x], 1).to(dev)[:, cols // 2:cols // 2 + cols])
        wv, ws = R.quantize_rows(y.float().numpy())
        np.testing.assert_array_equal(s.cpu().numpy(), ws)
        np.testing.assert_array_equal(v.cpu().numpy(), wv)


def test_quantize_rows_of_odd_values(dev):
    """Zeros, values that overflow 127 / max, ties, infinities and NaN, each in rows of their own."""
    big = 3.3e38
    x = torch.tensor([[0, 0, 0, 0], [1e-38, -1e-39, 0, 0], [big, -big, big / 2, 1], [127, 0.5, 1.5, 2.5],
                      [-127, -0.5, -1.5, -2.5], [float("inf"), 1, 2, 3], [1, float("nan"), 2, 3], [-float("inf"), 0, 0, 0],
                      [2.0 ** -100, -2.0 ** -101, 2.0 ** -102, 0], [2.0 ** -101, 0, 0, 0]]).repeat(1, 5)
    v, s = q3s.quantize_rows(x.to(dev))
    wv, ws = R.quantize_rows(x.numpy())
    np.testing.assert_array_equal(s.cpu().numpy(), ws)
    np.testing.assert_array_equal(v.cpu().numpy(), wv)
    w = torch.ones(32, 20, dtype=torch.int8, device=dev)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        q3s.int8_linear(x.to(dev), w, torch.ones(32, device=dev))
    y = q3s.int8_linear(x.repeat(1, 4).to(dev), w.repeat(1, 4), torch.ones(32, device=dev))
    assert torch.isnan(y[5:8]).all() and torch.isfinite(y[[0, 1, 3, 4, 8, 9]]).all() and not y[0].any()


@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (1, 2048, 2048), (2, 64, 100), (7, 144, 33), (8, 2048, 513), (9, 2048, 513),
                                   (16, 4096, 96), (17, 512, 1000), (64, 1040, 257), (128, 2048, 2048), (129, 2048, 96),
                                   (130, 2064, 5000), (300, 768, 768), (513, 128, 2050), (1000, 16, 130), (2000, 2048, 1024),
                                   (3, 16384, 130), (8, 16000, 40), (300, 16400, 96), (2300, 528, 5001), (4096, 2048, 2304),
                                   (250, 144, 20000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_int8_matmul(dev, M, K, N, dtype):
    g = torch.Generator(device=dev).manual_seed(M + K + N)
    a = torch.randint(-128, 128, (M, K), device=dev, generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), device=dev, generator=g, dtype=torch.int8)
    a_s = (torch.rand(M, device=dev, generator=g) + 0.5) / 127 / K ** 0.5
    w_s = (torch.rand(N, device=dev, generator=g) + 0.5) / 127
    bias = torch.randn(N, device=dev, generator=g)
    prod = (a.double() @ w.double().t()) * a_s.double()[:, None] * w_s.double()
    for b in (None, bias):
        y = q3s.int8_matmul(a, a_s, w, w_s, dtype=dtype, bias=b)
        want = prod + (0 if b is None else b.double())
        tol = (ROUNDOFF[dtype] + 2.0 ** -22) * (prod.abs() + (0 if b is None else b.abs().double()))
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25  # results below 2^-14 are subnormal
        assert y.dtype == dtype and bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("M,K", [(8, 3056), (8, 3088), (8, 6144), (4, 6144), (3, 6160), (2, 12288), (1, 24576), (1, 24592),
                                 (2, 24576), (1, 49152)])
def test_int8_few_rows_of_many_inputs(dev, M, K):
    """On both sides of the size up to which few rows are one launch, and where their bytes are 48 KB."""
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g)
    w = torch.randint(-128, 128, (19, K), generator=g, dtype=torch.int8)
    ws = torch.rand(19, generator=g) + 0.5
    values, scales = (torch.from_numpy(y).double() for y in R.quantize_rows(x.numpy()))
    want = (values @ w.double().t()) * scales[:, None] * ws.double()
    y = q3s.int8_linear(x.to(dev), w.to(dev), ws.to(dev))
    z = q3s.int8_matmul(*q3s.quantize_rows(x.to(dev)), w.to(dev), ws.to(dev), dtype=torch.float32)
    assert bool(((y.cpu().double() - want).abs() <= (ROUNDOFF[torch.float32] + 2.0 ** -22) * want.abs()).all())
    assert torch.equal(y, z)


def test_int8_matmul_largest_sums_and_strides(dev):
    """The longest K at full scale and operands that are slices."""
    K = 131056
    a = torch.full((3, K), 127, dtype=torch.int8, device=dev)
    w = torch.full((40, K), 127, dtype=torch.int8, device=dev)
    w[::2] = -128
    one = torch.ones(40, device=dev)
    y = q3s.int8_matmul(a, one[:3], w, one, dtype=torch.float32)
    want = (a.double() @ w.double().t())
    assert bool(((y.double() - want).abs() <= 2.0 ** -24 * want.abs()).all())
    for M in (3, 200):
        g = torch.Generator(device=dev).manual_seed(M)
        big = torch.randint(-128, 128, (M + 70, 512), device=dev, generator=g, dtype=torch.int8)
        a, w = big[:M, 16:16 + 256], big[M:, 256:]
        s = torch.ones(M + 70, device=dev)
        y = q3s.int8_matmul(a, s[:M], w, s[:70], dtype=torch.float32)
        assert torch.equal(y.double(), a.double() @ w.double().t())


@pytest.mark.parametrize("shape", [(2048,), (1, 2048), (3, 2, 2048), (0, 2048), (200, 2048)])
def test_int8_linear_is_quantise_then_product(dev, shape):
    g = torch.Generator(device=dev).manual_seed(len(shape))
    x = torch.randn(shape, device=dev, generator=g).to(torch.bfloat16)
    lin = q3s.Int8Linear(torch.randn(700, 2048, device=dev, generator=g), torch.randn(700, device=dev, generator=g))
    y = lin(x)
    assert y.shape == shape[:-1] + (700,)
    y2, v, s = q3s.int8_linear(x, lin.weight, lin.scales, bias=lin.bias, return_quantized=True)
    assert v.shape == x.shape and s.shape == shape[:-1] and torch.equal(y, y2)
    v2, s2 = q3s.quantize_rows(x)
    assert torch.equal(v, v2) and torch.equal(s, s2)
    if x.numel():
        y3 = q3s.int8_matmul(v2.reshape(-1, 2048), s2.reshape(-1), lin.weight, lin.scales, bias=lin.bias)
        assert torch.equal(y3.reshape(y.shape), y)
        full = x.double() @ (lin.weight.double() * lin.scales.double()[:, None]).t() + lin.bias.double()
        # the activations' rounding: each off by at most half a step, weights as they are
        step = s.double()[..., None] / 2 * (lin.weight.double() * lin.scales.double()[:, None]).abs().sum(1)
        assert bool(((y.double() - full).abs() <= step * 1.001 + 2.0 ** -8 * (full.abs() + step) + 1e-6).all())


def test_example_decode_step(dev):
    """The example runs, twice the same, and its cache lengths follow what was drawn."""
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("decode_step", Path(__file__).resolve().parents[1] / "examples" / "decode_step.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    drawn, lengths = example.main(rows=20, steps=30, voice_tokens=70)
    again, _ = example.main(rows=20, steps=30, voice_tokens=70)
    assert torch.equal(drawn, again) and drawn.shape == (30, 20)
    for r in range(20):
        ended = (drawn[:-1, r] == 7).nonzero()
        start = int(ended[-1]) + 1 if len(ended) else 0
        assert int(lengths[r]) == 30 - start


def test_products_wait_for_weights_made_just_before(dev):
    """Weights quantised by the kernel right before the product (and rows made right before them)."""
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(300, 4096, device=dev, generator=g).bfloat16()
    for rows in (1, 8, 40, 300):
        for _ in range(5):
            w = torch.randn(3000, 4096, device=dev, generator=g)
            torch.cuda.synchronize()
            v, s = q3s.quantize_rows(w)
            y = q3s.int8_linear(x[:rows], v, s)
            v.fill_(1)
            torch.cuda.synchronize()
            v2, s2 = q3s.quantize_rows(w)
            torch.cuda.synchronize()
            assert torch.equal(y, q3s.int8_linear(x[:rows], v2, s2))
