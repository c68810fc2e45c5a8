"""Attention of chunks over pages, on the GPU, against its definition in
float64 (tests/several_reference.py).

Tolerance, from the arithmetic, with U the type's unit roundoff (2^-8 bf16,
2^-11 f16): p is rounded once (U) and the result divided by the sum of the
rounded p, so it moves by U sum p |v - out| (and terms of U^2: U is taken 1.02
times); the output is rounded once, U |out|; scores (fp32 sums of D products),
ex2 and the fp32 sums take less than 2^-16 of sum p |v| at these score sizes.  A
probability below 2^-14 is subnormal in f16 and off by up to 2^-25; the sum of p
is at least 1: N 2^-25 max |v| for N keys.  lse: |err| <= 2^-16 (1 + |lse|)."""
import ctypes as C

import numpy as np
import pytest
import torch

import several_reference as R
import q3s

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def dev(cuda_device):
    q3s.load_torch_ops()
    return cuda_device


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


def make(dev, seed, news, owns, *, hq=8, hk=4, dim=128, bs=16, prefix=0, dtype=torch.bfloat16, order="heads", spare=3, width=None):
    """`news[b]` query tokens of row b behind `owns[b]` cached ones."""
    rng = np.random.RandomState(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    news, lengths = np.array(news), np.array(news) + np.array(owns)
    held = R.ceil_div(lengths, bs)
    width = width or int(held.max(initial=0)) + 2
    shared = R.ceil_div(prefix, bs)
    blocks = int(held.sum()) + shared + spare
    ids = rng.permutation(blocks)
    table = np.full((len(news), width), -7)
    table[np.arange(width)[None, :] < held[:, None]] = ids[shared:shared + int(held.sum())]
    shape = (2, blocks, hk, bs, dim) if order == "heads" else (2, blocks, bs, hk, dim)
    cache = torch.randn(shape, device=dev, generator=g).to(dtype)
    if order == "tokens":
        cache = cache.transpose(2, 3)
    T = int(news.sum())
    q = torch.randn(T, hq, dim, device=dev, generator=g).to(dtype)
    return dict(q=q, k=cache[0], v=cache[1], off=i32(np.concatenate([[0], np.cumsum(news)]), dev), table=i32(table, dev),
                len=i32(lengths, dev), shared=i32(ids[:shared], dev), prefix=prefix)


def run(c, **kw):
    return q3s.chunk_attention(c["q"], c["k"], c["v"], c["off"], c["table"], c["len"], prefix_blocks=c["shared"],
                               prefix_length=c["prefix"], return_lse=True, **kw)


EVERYTHING = 2 ** 31 - 1  # a window that leaves nothing out: always the kernel with tiles of 128 query rows


def check(c, window=0, scale=None, slot_map=None, k=None, v=None):
    """`k`, `v`: what the definition reads in place of the caches.  Without a window both kernels: few queries go to the
    one of prefix_attention otherwise."""
    if window == 0:
        check(c, EVERYTHING, scale, slot_map, k, v)
    D = c["q"].shape[2]
    err = torch.zeros(1, dtype=torch.int32, device=c["q"].device)
    out, lse = run(c, window=window, scale=scale, error_word=err, slot_map=slot_map)
    assert int(err) == 0
    want, want_lse, spread, mass = R.chunk_attention(c["q"], c["k"] if k is None else k, c["v"] if v is None else v, c["off"].tolist(),
                                                     c["table"], c["len"].tolist(), c["shared"], c["prefix"],
                                                     D ** -0.5 if scale is None else scale, window, slot_map)
    U = ROUNDOFF[out.dtype]
    keys = int(c["len"].max()) + c["prefix"] if c["len"].numel() else 0
    tiny = keys * 2.0 ** -25 * 6.0 if out.dtype == torch.float16 else 0.0  # |v| of a normal distribution: below 6
    tol = U * want.abs() + 1.02 * U * spread + 2.0 ** -16 * mass + torch.where(mass > 0, tiny, 0.0)
    assert bool(((out.double() - want).abs() <= tol).all()), float(((out.double() - want).abs() - tol).max())
    none = want_lse == -float("inf")
    assert bool((lse[none] == -float("inf")).all()) and bool((out[none] == 0).all())
    assert bool(((lse.double() - want_lse).abs()[~none] <= 2.0 ** -16 * (1 + want_lse.abs()[~none])).all())
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news,owns,hq,hk,bs,prefix,window", [
    ([1], [0], 1, 1, 16, 0, 0),                        # one token that sees itself
    ([1], [0], 2, 1, 16, 1, 0),
    ([5], [700], 16, 8, 16, 200, 0),                   # drafts, all keys cut over the GPU
    ([128], [0], 4, 4, 16, 0, 0),                      # one tile, the diagonal only
    ([129], [127], 2, 2, 32, 0, 0),
    ([300], [0], 2, 1, 128, 0, 0),                     # two items, three tiles
    ([3, 0, 9, 1, 7], [40, 300, 129, 0, 1000], 12, 4, 32, 333, 0),
    ([17, 40], [100, 5], 3, 1, 16, 127, 0),            # a group that does not divide 128
    ([17, 40], [100, 5], 5, 1, 64, 129, 30),
    ([70, 3], [100, 500], 16, 1, 16, 0, 0),
    ([200, 64], [600, 0], 4, 2, 64, 0, 100),           # windows that begin inside a step, or leave steps out
    ([200, 64], [600, 0], 4, 2, 16, 150, 1),
    ([33], [500], 4, 2, 16, 500, 400),                 # a window that begins in the prefix
    ([33], [500], 4, 2, 16, 500, 100000),
    ([1] * 50, list(range(0, 500, 10)), 8, 2, 16, 64, 0)])
def test_matches_definition(dev, news, owns, hq, hk, bs, prefix, window, dim, dtype):
    check(make(dev, len(news) + dim, news, owns, hq=hq, hk=hk, dim=dim, bs=bs, prefix=prefix, dtype=dtype), window)


@pytest.mark.parametrize("hq,hk", [(128, 1), (64, 1), (40, 2), (7, 7)])
def test_large_groups_and_many_heads(dev, hq, hk):
    check(make(dev, hq, [5, 3], [200, 10], hq=hq, hk=hk, dim=64))


@pytest.mark.parametrize("rows", [330, 700])
def test_many_rows(dev, rows):
    """More rows than a CTA has threads, more segments than it lists at a time."""
    rng = np.random.RandomState(rows)
    check(make(dev, rows, rng.randint(0, 4, rows), rng.randint(0, 60, rows), hq=32, hk=32, dim=64))


def test_more_segments_than_a_list_holds(dev):
    rng = np.random.RandomState(9)
    check(make(dev, 9, rng.randint(1, 3, 600), rng.randint(0, 20, 600), hq=32, hk=32, dim=128, prefix=5), 0)


def test_long_rows(dev):
    check(make(dev, 5, [1500, 700], [2000, 1], hq=2, hk=1, dim=128))
    check(make(dev, 6, [1500, 700], [2000, 1], hq=2, hk=1, dim=64, prefix=300, dtype=torch.float16), 700)


def test_agrees_with_prefix_attention(dev):
    c = make(dev, 7, [9, 1, 30, 0], [700, 64, 3, 10], hq=8, hk=4, prefix=500)
    out, lse = check(c)
    other, other_lse = q3s.prefix_attention(c["q"], c["k"], c["v"], c["off"], c["table"], c["len"], prefix_blocks=c["shared"],
                                            prefix_length=500, return_lse=True)
    U = ROUNDOFF[torch.bfloat16]
    assert float((out.float() - other.float()).abs().max()) <= 4 * U * float(c["v"].abs().max())
    assert float((lse - other_lse).abs().max()) < 2.0 ** -12


def test_rows_shorter_than_their_queries(dev):
    """Lengths that do not count the step's tokens (a state that cache_tables does not leave): as prefix_attention."""
    for prefix in (0, 40):
        c = make(dev, 8, [20, 300], [30, 50], hq=4, hk=2, prefix=prefix)
        c["len"] = i32([7, 120], dev)
        check(c)
        check(c, window=25)


def test_queries_without_a_slot_and_tokens_of_no_row(dev):
    c = make(dev, 10, [20, 130, 5], [30, 50, 3], hq=4, hk=2, prefix=20)
    slots = torch.arange(155, device=dev)
    slots[20:150] = -1
    slots[153] = -1
    check(c, slot_map=slots)
    c["q"] = torch.cat([c["q"], c["q"][:40]])  # a padded batch
    check(c)
    c["off"] = i32([3, 20, 150, 155], dev)  # tokens before the first row
    c["len"] = i32([47, 180, 8], dev)
    check(c)


def test_no_rows_no_tokens_no_keys(dev):
    c = make(dev, 11, [4], [0])
    z = dict(c, off=i32([0], dev), table=c["table"][:0], len=i32([], dev))
    for window in (0, EVERYTHING):
        out, lse = run(z, window=window)
        assert not out.any() and bool((lse == -float("inf")).all())
        out, lse = run(dict(c, len=i32([0], dev)), window=window)
        assert not out.any() and bool((lse == -float("inf")).all())
    out, lse = run(dict(c, q=c["q"][:0], off=i32([0, 0], dev)))
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)


def test_strides(dev):
    c = make(dev, 12, [40, 7], [100, 30], hq=4, hk=2, dim=64, order="tokens", prefix=50)
    check(c)
    wide = torch.randn(47, 12, 64, device=dev).bfloat16()
    check(dict(c, q=wide[:, 4:8]))
    big = torch.zeros(c["table"].shape[0], 50, dtype=torch.int32, device=dev)
    big[:, 3:3 + c["table"].shape[1]] = c["table"]
    check(dict(c, table=big[:, 3:3 + c["table"].shape[1]]))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("news,owns,prefix,window", [([200], [77], 0, 0), ([40, 5], [300, 20], 70, 0), ([200], [477], 30, 64)])
def test_values_that_a_query_does_not_see_do_not_reach_it(dev, news, owns, prefix, window, value):
    """K and V behind every row's end, and of pages of nobody, hold NaN or infinity; and so do tokens that only some queries see."""
    c = make(dev, 13, news, owns, hq=4, hk=2, dim=64, bs=32, prefix=prefix)
    k, v = c["k"].clone(), c["v"].clone()
    used = torch.zeros(k.shape[0], 32, dtype=torch.bool, device=dev)
    for b, n in enumerate(c["len"].tolist()):
        for j in range(n):
            used[c["table"][b, j // 32], j % 32] = True
    for j in range(prefix):
        used[c["shared"][j // 32], j % 32] = True
    for x in (k, v):
        x.transpose(1, 2)[~used] = value
    check(dict(c, k=k, v=v), window, k=c["k"], v=c["v"])
    # the last token of the first row: only its last query sees it
    last = int(c["len"][0]) - 1
    where = (c["table"][0, last // 32], slice(None), last % 32)
    v[where] = value
    n = news[0]
    out, lse = run(dict(c, k=k, v=v), window=window or EVERYTHING)
    keep = torch.ones(out.shape[0], dtype=torch.bool, device=dev)
    keep[n - 1] = False
    want, want_lse, spread, mass = R.chunk_attention(c["q"], c["k"], c["v"], c["off"].tolist(), c["table"], c["len"].tolist(), c["shared"],
                                                     prefix, 0.125, window)
    U = ROUNDOFF[torch.bfloat16]
    tol = U * want.abs() + 1.02 * U * spread + 2.0 ** -16 * mass
    assert bool(((out.double() - want).abs() <= tol)[keep].all())
    assert torch.isfinite(lse).all()
    assert bool((out[n - 1] == value).all()) if value == float("inf") else bool(out[n - 1].isnan().all())


def test_peaked_scores_and_large_ones(dev):
    for factor in (8.0, 40.0):
        c = make(dev, 14, [150, 20], [300, 100], hq=4, hk=2)
        c["q"] = (c["q"].float() * factor).bfloat16()
        out, _ = run(c, window=EVERYTHING)
        want, _, spread, mass = R.chunk_attention(c["q"], c["k"], c["v"], c["off"].tolist(), c["table"], c["len"].tolist(), c["shared"], 0,
                                                  128 ** -0.5)
        U = ROUNDOFF[torch.bfloat16]
        # scores up to 6 * factor (|q . k| / sqrt(D)) are off by 2^-22 of the sum of their products' magnitudes (at most 20 factor)
        tol = U * want.abs() + (1.02 * U + 2 * 20 * factor * 2.0 ** -22) * spread + 2.0 ** -16 * mass
        assert bool(((out.double() - want).abs() <= tol).all())


def test_bad_block_ids_read_as_zeros(dev):
    c = make(dev, 15, [30], [100], hq=2, hk=1, dim=64)
    bad = c["table"].clone()
    bad[0, 2], bad[0, 4] = 10 ** 6, -1
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = run(dict(c, table=bad), error_word=err, window=EVERYTHING)
    assert int(err) == q3s.decode.DECERR_BLOCK_ID
    k, v = c["k"].clone(), c["v"].clone()
    for j in (2, 4):
        k[c["table"][0, j]] = 0
        v[c["table"][0, j]] = 0
    want, want_lse = run(dict(c, k=k, v=v), window=EVERYTHING)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("window", [0, EVERYTHING])
@pytest.mark.parametrize("news,hq", [([5], 2), ([200, 3], 2)])
@pytest.mark.parametrize("past", [0, 1, 5])
def test_the_first_id_past_the_cache_is_reported(dev, news, hq, window, past):
    """An id equal to the number of blocks is outside too, in a row's table and in the prefix, whichever kernel a call goes to."""
    c = make(dev, 21, news, [90] * len(news), hq=hq, hk=1, dim=64, prefix=40)
    blocks = c["k"].shape[0]
    k, v = c["k"].clone(), c["v"].clone()
    bad, shared = c["table"].clone(), c["shared"].clone()
    where = {"table": (bad, (0, 2)), "prefix": (shared, (1,))}
    for name, (ids, at) in where.items():
        was, block = int(ids[at]), int(ids[at])
        ids[at] = blocks + past
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        out, lse = run(dict(c, table=bad, shared=shared), error_word=err, window=window)
        assert int(err) == q3s.decode.DECERR_BLOCK_ID, name
        kept = k[block].clone(), v[block].clone()
        k[block], v[block] = 0, 0
        want, want_lse = run(dict(c, k=k, v=v), window=window)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        k[block], v[block] = kept
        ids[at] = was


@pytest.mark.parametrize("queries", [5, 90])
def test_prefix_attention_reports_the_first_id_past_the_cache(dev, queries):
    """With few queries the prefix is read by the key-split kernel, with many by the kernel of its own."""
    c = make(dev, 22, [1] * queries, [3] * queries, hq=8, hk=2, dim=64, prefix=2000)
    for past in (0, 1):
        shared = c["shared"].clone()
        shared[7] = c["k"].shape[0] + past
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        q3s.prefix_attention(c["q"], c["k"], c["v"], c["off"], c["table"], c["len"], prefix_blocks=shared, prefix_length=2000, error_word=err)
        assert int(err) == q3s.decode.DECERR_BLOCK_ID


@pytest.mark.parametrize("window", [0, EVERYTHING])
@pytest.mark.parametrize("rows", [3, 500])
@pytest.mark.parametrize("what", ["a negative length", "a length past the table", "offsets past the tokens", "offsets that descend", "a negative offset"])
def test_lengths_that_are_cut_are_reported(dev, rows, what, window):
    """Whichever kernel a call goes to, and in every row (500: more than a CTA has threads)."""
    c = make(dev, 23, [2] * rows, [20] * rows, hq=2, hk=1, dim=64)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    run(c, window=window, error_word=err)
    assert int(err) == 0
    row, T = rows - 1, 2 * rows
    length, off = c["len"].clone(), c["off"].clone()
    if what == "a negative length":
        length[row] = -3
    elif what == "a length past the table":
        length[row] = c["table"].shape[1] * 16 + 1
        c["table"][row] = 0
    elif what == "offsets past the tokens":
        off[-1] = T + 4
    elif what == "offsets that descend":
        off[row], off[row + 1] = T, T - 2
    else:
        off[0] = -1
    run(dict(c, len=length, off=off), window=window, error_word=err)
    assert int(err) == q3s.decode.DECERR_LENGTHS


def test_same_call_same_result_and_side_stream(dev):
    c = make(dev, 16, [300, 20, 7], [900, 100, 2000], hq=8, hk=4, prefix=100)
    first = run(c, window=EVERYTHING)
    for _ in range(5):
        again = run(c, window=EVERYTHING)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run(c, window=EVERYTHING)
    s.synchronize()
    assert torch.equal(first[0], other[0])


def test_two_streams_at_once(dev):
    c, d = make(dev, 17, [600], [900], hq=8, hk=4), make(dev, 18, [64, 64], [700, 700], hq=8, hk=4)
    want = run(c), run(d)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s, x in zip(streams, (c, d)):
            with torch.cuda.stream(s):
                got.append(run(x))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])


def test_captured_call_follows_the_lengths(dev):
    c = make(dev, 19, [40, 30], [10, 900], hq=4, hk=2, prefix=64)
    run(c, window=EVERYTHING)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = run(c, window=EVERYTHING)
    for lengths, off in (([50, 930], [0, 40, 70]), ([45, 100], [0, 5, 70]), ([50, 930], [0, 0, 30])):
        c["len"].copy_(i32(lengths, dev))
        c["off"].copy_(i32(off, dev))
        graph.replay()
        o, l = run(c, window=EVERYTHING)
        assert torch.equal(out, o) and torch.equal(lse, l)
        check(c)


def test_output_strides_through_the_c_abi(dev):
    c = make(dev, 20, [140, 7], [100, 900], hq=4, hk=2)
    want, want_lse = run(c)
    lib, L = q3s._lib.load(), q3s._lib
    out = torch.zeros(147, 9, 136, dtype=torch.bfloat16, device=dev)
    d = L.ChunkAttentionDesc(
        struct_size=C.sizeof(L.ChunkAttentionDesc), batch=2, tokens=147, q_heads=4, kv_heads=2, dim=128, block_size=16,
        blocks=c["k"].shape[0], elem=L.ELEM_BF16, max_blocks=c["table"].shape[1], scale=128 ** -0.5, q=c["q"].data_ptr(),
        q_token_stride=512, q_head_stride=128, k_cache=c["k"].data_ptr(), v_cache=c["v"].data_ptr(), query_offsets=c["off"].data_ptr(),
        block_table=c["table"].data_ptr(), block_table_stride=c["table"].stride(0), lengths=c["len"].data_ptr(), out=out.data_ptr(),
        out_token_stride=9 * 136, out_head_stride=2 * 136)
    for name, x in (("k", c["k"]), ("v", c["v"])):
        for key, axis in (("block", 0), ("head", 1), ("place", 2)):
            setattr(d, f"{name}_{key}_stride", x.stride(axis))
    n = C.c_int64()
    L.check(lib.q3s_chunk_attention_workspace(C.byref(d), C.byref(n)), "workspace")
    ws = torch.full((n.value,), 255, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
    L.check(lib.q3s_chunk_attention(C.byref(d), torch.cuda.current_stream().cuda_stream), "q3s_chunk_attention")
    assert torch.equal(out[:, 0:8:2, :128], want)
    out[:, 0:8:2, :128] = 0
    assert not out.any()
