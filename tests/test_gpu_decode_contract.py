"""What the decode step's operators promise about order, odd values and reports,
on the GPU, against plain forms in Python integers and float64."""
import subprocess
import sys

import numpy as np
import pytest
import torch

import decode_reference as R
import q3s

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda_device):
    q3s.load_torch_ops()
    return cuda_device


# ---- order of calls -----------------------------------------------------------

def exact_product(a, a_s, w, w_s):
    """(values, tolerance) of an fp32 8-bit product: an exact sum, its conversion and two products, each off by 2^-24."""
    want = (a.double() @ w.double().t()) * a_s.double()[:, None] * w_s.double()
    return want, 2.0 ** -22 * want.abs()


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 40])
def test_returned_values_as_the_next_weight(dev, rows):
    """The values that a one-launch Linear writes are the weight of the product right behind it."""
    g = torch.Generator(device=dev).manual_seed(rows)
    w = torch.randint(-127, 128, (2048, 2048), device=dev, generator=g, dtype=torch.int8)
    ws = torch.rand(2048, device=dev, generator=g) + 0.5
    for _ in range(10):
        x = torch.randn(rows, 2048, device=dev, generator=g).bfloat16()
        torch.cuda.synchronize()
        _, v, s = q3s.int8_linear(x, w, ws, return_quantized=True)
        z = q3s.int8_matmul(v, s, v, s, dtype=torch.float32)
        want, tol = exact_product(v, s, v, s)
        assert bool(((z.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("rows", [1, 8, 40, 300])
def test_weight_written_by_another_kernel_right_before(dev, rows):
    g = torch.Generator(device=dev).manual_seed(rows)
    a = torch.randint(-127, 128, (rows, 2048), device=dev, generator=g, dtype=torch.int8)
    s = torch.rand(5000, device=dev, generator=g) + 0.5
    w = torch.empty(5000, 2048, device=dev, dtype=torch.int8)
    for _ in range(5):
        fresh = torch.randint(-127, 128, (5000, 2048), device=dev, generator=g, dtype=torch.int8)
        torch.cuda.synchronize()
        torch.add(fresh, 0, out=w)
        y = q3s.int8_matmul(a, s[:rows], w, s, dtype=torch.float32)
        want, tol = exact_product(a, s[:rows], fresh, s)
        assert bool(((y.double() - want).abs() <= tol).all())


# ---- attention: one key carries a query ------------------------------------------

@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (128, torch.float16), (64, torch.float16)])
def test_attention_one_key_carries_the_prefix(dev, dtype, dim):
    """A key far above all others, met after the running maximum was set 2^7 to 2^8 below it.

    With U the type's unit roundoff, probabilities rounded to that type and divided by their own sum move the result by U
    sum p |v - out| at most (to first order; U^2 mass for the rest), its own rounding by U |out|, ex2 and the 32-bit sums
    by less than 2^-16 of sum p |v|, and in f16 each of the keys' probabilities, subnormal below 2^-14, by 2^-25."""
    rows, heads, kv_heads, keys, block = 64, 8, 2, 4096, 16
    g = torch.Generator().manual_seed(dim)
    scale = dim ** -0.5
    blocks = keys // block + rows
    k = torch.zeros(blocks, kv_heads, block, dim)
    v = torch.randn(blocks, kv_heads, block, dim, generator=g)
    # scores, in units of log 2, along the first dimension: q is 1 to 8/7 there, times what makes 7 of a key's 1
    unit = 7 * 0.6931471805599453 / scale
    k[..., 0] = -4.0  # the others: 2^-28
    first = k[:keys // block].transpose(1, 2).reshape(keys, kv_heads, dim)
    first[::128, :, 0] = 0.0  # one of each 128 keys sets the running maximum to 0
    first[7 * 128 + 77, :, 0] = 1.0  # and this one is above it
    k[:keys // block] = first.reshape(keys // block, block, kv_heads, dim).transpose(1, 2)
    q = torch.zeros(rows, heads, dim)
    q[..., 0] = unit * (1 + torch.rand(rows, heads, generator=g) / 7.2)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    table = torch.arange(keys // block, blocks, dtype=torch.int32)[:, None]
    offsets = torch.arange(rows + 1, dtype=torch.int32)
    shared, lengths = torch.arange(keys // block, dtype=torch.int32), torch.ones(rows, dtype=torch.int32)
    out, lse = q3s.prefix_attention(q.to(dev), k.to(dev), v.to(dev), offsets.to(dev), table.to(dev), lengths.to(dev),
                                    prefix_blocks=shared.to(dev), prefix_length=keys, scale=scale, return_lse=True)
    want, want_lse, mass = R.prefix_attention(q, k, v, offsets, table, lengths, shared, keys, scale)
    # sum p |v - out|: the key that carries the query, and the rest (whose p sum to 1 - p of it)
    top = v.double()[(7 * 128 + 77) // block, :, (7 * 128 + 77) % block].repeat_interleave(heads // kv_heads, 0)
    p = torch.exp(scale * q.double()[..., 0] * 1.0 - want_lse)[..., None]
    away = p * (top - want).abs() + (mass - p * top.abs()).clamp(min=0) + (1 - p) * want.abs()
    U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tol = U * want.abs() + U * away + (U * U + 2.0 ** -16) * mass + (keys * 2.0 ** -25 * 5 if dtype == torch.float16 else 0)
    d = (out.cpu().double() - want).abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max())} of the tolerance"
    assert bool(((lse.cpu().double() - want_lse).abs() <= 2.0 ** -16 * (1 + want_lse.abs())).all())


# ---- attention: infinities in V -----------------------------------------------------

@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("rows,prefix", [(1, 0), (3, 40), (100, 600)])
@pytest.mark.parametrize("n", [1, 2])
def test_attention_infinity_that_a_query_sees(dev, dim, dtype, rows, prefix, n):
    """+inf in one dim of V and -inf in another, of a row's first own key or of a key of the prefix, taken by either kernel:
    the queries that see it have that infinity there, and nothing else changes."""
    heads, kv_heads, own, block = 4, 2, 21, 16
    g = torch.Generator(device=dev).manual_seed(rows + n)
    shared = -(-prefix // block)
    blocks = shared + 2 * rows
    k, v = (torch.randn(blocks, kv_heads, block, dim, device=dev, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(rows * n, heads, dim, device=dev, generator=g).to(dtype)
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.arange(shared, blocks, **i32).view(rows, 2)
    args = dict(prefix_blocks=torch.arange(shared, **i32), prefix_length=prefix, return_lse=True)
    rest = (torch.arange(0, rows * n + 1, n, **i32), table, torch.full((rows,), own, **i32))
    out, lse = q3s.prefix_attention(q, k, v, *rest, **args)
    for block_of, place, hit in [(int(table[0, 0]), 0, slice(0, n))] + ([(prefix // 2 // block, prefix // 2 % block, slice(None))] if prefix else []):
        w = v.clone()
        w[block_of, :, place, 5] = float("inf")
        w[block_of, :, place, 40] = -float("inf")
        odd, odd_lse = q3s.prefix_attention(q, k, w, *rest, **args)
        want = out.clone()
        want[hit, :, 5] = float("inf")
        want[hit, :, 40] = -float("inf")
        finite = torch.isfinite(want)
        assert torch.equal(odd[~finite], want[~finite])
        # what is taken again key by key has its sums in another order and p in one piece: two roundings of the type apart
        assert bool(((odd - want)[finite].abs().double() <= 2.0 ** (-7 if dtype == torch.bfloat16 else -10) * want[finite].abs().double() + 1e-3).all())
        assert bool(((odd_lse - lse).abs() <= 2.0 ** -15 * (1 + lse.abs())).all())


# ---- reports -------------------------------------------------------------------------

# stands in front of the library's 8-bit products and keeps the error word that they are given
SHIM = r"""
#include "q3s_decode.h"
extern "C" {
const void* seen = 0;
q3s_status q3s_int8_matmul(const q3s_int8_matmul_desc* d, void*) { seen = d->error_word; return Q3S_OK; }
q3s_status q3s_int8_linear(const q3s_quantize_rows_desc*, const q3s_int8_matmul_desc* d, void*) { seen = d->error_word; return Q3S_OK; }
}
"""
SHIM_CALLER = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
import torch, q3s
seen = ctypes.c_void_p.in_dll(shim, "seen")
dev = torch.device("cuda:0")
w, s = torch.ones(32, 64, dtype=torch.int8, device=dev), torch.ones(32, device=dev)
x, err = torch.ones(3, 64, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
q3s.int8_matmul(w[:3], s[:3], w, s, error_word=err)
assert seen.value == err.data_ptr(), "int8_matmul"
q3s.int8_matmul(w[:3], s[:3], w, s)
assert seen.value is None
q3s.int8_linear(x, w, s, error_word=err)
assert seen.value == err.data_ptr(), "int8_linear"
linear = q3s.Int8Linear(torch.randn(32, 64, device=dev))
linear(x)
assert seen.value == linear.error_word.data_ptr() and int(linear.error_word) == 0, "Int8Linear"
"""


def test_error_words_of_8_bit_products_reach_the_library(dev, tmp_path):
    from q3s import build

    src, lib = tmp_path / "shim.cpp", tmp_path / "shim.so"
    src.write_text(SHIM)
    subprocess.run([build.system_cxx(), "-shared", "-fPIC", f"-I{build.INCLUDE}", "-o", str(lib), str(src)], check=True)
    done = subprocess.run([sys.executable, "-c", SHIM_CALLER, str(lib), str(build.PKG_DIR.parent)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_error_word_of_a_product_is_checked_and_left_alone(dev):
    w, s = torch.ones(32, 64, dtype=torch.int8, device=dev), torch.ones(32, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    for rows in (1, 20):
        y = q3s.int8_linear(torch.ones(rows, 64, device=dev), w, s, error_word=err)
        assert int(err) == 0 and bool((y == 64.0).all())
    for bad in (err.long(), err.cpu(), torch.zeros(2, dtype=torch.int32, device=dev)):
        with pytest.raises(RuntimeError, match="error_word"):
            q3s.int8_linear(torch.ones(1, 64, device=dev), w, s, error_word=bad)
        with pytest.raises(RuntimeError, match="error_word"):
            q3s.int8_matmul(w[:3], s[:3], w, s, error_word=bad)


def test_paged_cache_collects_reports(dev):
    def fresh():
        cache = q3s.PagedCache(2, 8, layers=1, kv_heads=1, dim=64, max_blocks=3, device=dev)
        cache.step(torch.ones(2, dtype=torch.int32, device=dev), max_tokens=2)
        return cache

    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device=dev)
    cache = fresh()
    cache.append(0, x, x)
    cache.attend(0, x)
    assert int(cache.error_word) == 0 and int(cache.tables.error_word) == 0
    cache.table[1, 0] = 10 ** 6
    cache.attend(0, x)
    assert int(cache.error_word) == q3s.decode.DECERR_BLOCK_ID
    own = torch.zeros(1, dtype=torch.int32, device=dev)
    cache.error_word.zero_()
    cache.attend(0, x, error_word=own)
    assert int(own) == q3s.decode.DECERR_BLOCK_ID and int(cache.error_word) == 0
    cache = fresh()
    cache.tables.slot_map[0] = 8 * 16
    cache.append(0, x, x)
    assert int(cache.error_word) == q3s.decode.DECERR_BLOCK_ID


# ---- outputs ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 5, 300])
def test_outputs_are_tensors_of_their_own(dev, rows):
    """No two outputs of a call share memory, as their schemas say (an output that is kept keeps nothing else)."""
    from torch._subclasses.schema_check_mode import SchemaCheckMode

    i32 = dict(dtype=torch.int32, device=dev)
    ring, state = torch.arange(rows, **i32), torch.tensor([0, rows], **i32)
    x = torch.ones(rows, 64, device=dev)
    with SchemaCheckMode():
        t = q3s.cache_tables(torch.zeros(rows, **i32), torch.ones(rows, **i32), torch.zeros(rows, 2, **i32), ring, state,
                             block_size=16, max_tokens=rows)
        y = q3s.int8_linear(x, torch.ones(32, 64, dtype=torch.int8, device=dev), torch.ones(32, device=dev), return_quantized=True)
    for outs in (t, y):
        assert len({o.untyped_storage().data_ptr() for o in outs}) == len(outs)
        assert all(o.untyped_storage().nbytes() == o.numel() * o.element_size() for o in outs)


# ---- tables: more tokens than a step has slots for ----------------------------------------

@pytest.mark.parametrize("rows,cap", [(3, 2), (200, 1000), (1500, 300), (40, 0)])
def test_tables_refuse_whole_rows_past_the_last_slot(dev, rows, cap):
    """Rows up to the one whose tokens end past the cap are served as in a step without the others; those keep their length."""
    rng = np.random.RandomState(rows)
    block, width = 16, 12
    context, new = rng.randint(0, 100, rows), rng.randint(0, 30, rows)
    if rows == 3:
        new[:] = 1
    gone = rng.rand(rows) < 0.1
    held = R.ceil_div(context, block)
    ids = rng.permutation(int(held.sum()) + 5 * rows)
    table = np.full((rows, width), -1)
    table[np.arange(width)[None, :] < held[:, None]] = ids[: int(held.sum())]
    ring = np.concatenate([ids[int(held.sum()):], np.full(int(held.sum()), -1)])
    state = [0, len(ids) - int(held.sum())]
    kept = np.where(np.cumsum(new) <= cap, new, 0)
    want = R.cache_tables(context.tolist(), kept.tolist(), table.tolist(), ring.tolist(), state, block_size=block, max_tokens=cap,
                          released=gone.tolist())
    i32 = dict(dtype=torch.int32, device=dev)
    on_gpu = [torch.as_tensor(x, **i32) for x in (context, new, table, ring, state)]
    t = q3s.cache_tables(*on_gpu, block_size=block, max_tokens=cap, released=torch.as_tensor(gone, device=dev), whole_rows=True)
    for name in ("lengths", "free_state", "slot_map"):
        np.testing.assert_array_equal(getattr(t, name).cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(on_gpu[2].cpu().numpy(), want["table"])
    np.testing.assert_array_equal(on_gpu[3].cpu().numpy(), want["ring"])
    np.testing.assert_array_equal(t.query_offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(new)]))
    assert int(t.error_word) == q3s.decode.DECERR_TOKENS
    n = int(kept.sum())
    np.testing.assert_array_equal(t.positions.cpu().numpy()[:n], want["positions"][:n])


def test_paged_cache_after_a_step_with_too_many_tokens(dev):
    """The row that a step had no room for is as before it; the next steps read what was stored, and nothing else."""
    rows, heads, dim, block = 3, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(0)
    cache = q3s.PagedCache(rows, 9, layers=1, kv_heads=heads, dim=dim, max_blocks=3, device=dev)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    stored = [torch.zeros(0, heads, dim, dtype=torch.bfloat16, device=dev) for _ in range(rows)]
    for new, cap, served in (([2, 1, 1], 4, [2, 1, 1]), ([1, 2, 1], 2, [1, 0, 0]), ([17, 1, 1], 19, [17, 1, 1]), ([1, 1, 0], 2, [1, 1, 0])):
        t = cache.step(torch.tensor(new, dtype=torch.int32, device=dev), max_tokens=cap)
        assert int(t.error_word) == (0 if new == served else q3s.decode.DECERR_TOKENS)
        x = torch.randn(cap, heads, dim, device=dev, generator=g).bfloat16()
        cache.append(0, x, x)
        at = 0
        for b in range(rows):
            stored[b] = torch.cat([stored[b], x[at:at + served[b]]])
            at += new[b]
        assert cache.lengths.tolist() == [len(s) for s in stored]
        out = cache.attend(0, x)
        at = 0
        for b in range(rows):
            for i in range(served[b]):
                keys = stored[b][: len(stored[b]) - served[b] + i + 1].double()
                p = (torch.einsum("hd,jhd->hj", x[at + i].double(), keys) * dim ** -0.5).softmax(1)
                want = torch.einsum("hj,jhd->hd", p, keys)
                mass = torch.einsum("hj,jhd->hd", p, keys.abs())
                # out's rounding, and 2^-16 for p in two parts, ex2 and the sums
                assert bool(((out[at + i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * mass).all())
            at += new[b]


# ---- attention of refused rows ---------------------------------------------------------------

@pytest.mark.parametrize("rows,prefix", [(6, 0), (6, 40), (120, 400)])
@pytest.mark.parametrize("why", ["table", "ring", "slots"])
def test_refused_rows_attend_to_nothing(dev, rows, prefix, why):
    """Queries of a row that got no slots: 0 and -inf, in place of what the row's older tokens would give; the others' are as
    without those rows."""
    heads, dim, block, n = 2, 64, 16, 3
    g = torch.Generator(device=dev).manual_seed(rows)
    shared = -(-prefix // block)
    spare = {"ring": 2 * rows - 2, "table": 3 * rows, "slots": 3 * rows}[why]
    cache = q3s.PagedCache(rows, shared + spare, layers=1, kv_heads=heads, dim=dim, max_blocks=2 if why == "table" else 3,
                           prefix_blocks=shared, device=dev)

    def draw(tokens, h=heads):
        return torch.randn(tokens, h, dim, device=dev, generator=g).bfloat16()

    if prefix:
        cache.write_prefix(0, draw(prefix), draw(prefix))
    first = torch.full((rows,), 15, dtype=torch.int32, device=dev)
    first[rows // 2] = 30 if why == "table" else 15
    total = int(first.sum())
    cache.step(first, max_tokens=total)
    cache.append(0, draw(total), draw(total))
    before = cache.lengths.clone()
    cap = n * rows - (2 if why == "slots" else 0)
    t = cache.step(torch.full((rows,), n, dtype=torch.int32, device=dev), max_tokens=cap)
    refused = {"table": [rows // 2], "ring": [rows - 2, rows - 1], "slots": [rows - 1]}[why]
    assert int(t.error_word) == {"table": 2, "ring": 4, "slots": 8}[why]
    served = torch.ones(rows, dtype=torch.bool, device=dev)
    served[refused] = False
    assert torch.equal(cache.lengths, before + n * served)
    x = draw(cap)
    cache.append(0, x, x)
    q = draw(cap, 2 * heads)
    out, lse = cache.attend(0, q, return_lse=True)
    token = served.repeat_interleave(n)[:cap]
    assert not bool(out[~token].any()) and bool((lse[~token] == -float("inf")).all())
    plain, plain_lse = cache.attend(0, q, return_lse=True, slot_map=None)
    assert torch.equal(out[token], plain[token]) and torch.equal(lse[token], plain_lse[token])
    assert bool(plain[~token].any())
    more, more_lse = cache.attend(0, torch.cat([q, q[:5]]), return_lse=True)
    assert torch.equal(more[:cap], out) and not bool(more[cap:].any()) and bool((more_lse[cap:] == -float("inf")).all())


def test_attention_slot_map_is_checked(dev):
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev)
    c = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    for bad in (torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(2, **i32), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(RuntimeError, match="slot_map"):
            q3s.prefix_attention(q, c, c, torch.arange(3, **i32), torch.zeros(2, 1, **i32), torch.ones(2, **i32), slot_map=bad)


# ---- a step of PagedCache in a graph -------------------------------------------------------

def test_paged_cache_step_in_a_cuda_graph(dev):
    """A captured step advances the cache at each replay, as a step that is called does."""
    rows, heads, dim, block, steps = 5, 2, 64, 16, 40
    g = torch.Generator(device=dev).manual_seed(0)
    new = torch.randint(0, 3, (steps, rows), device=dev, generator=g, dtype=torch.int32)
    gone = torch.rand(steps, rows, device=dev, generator=g) < 0.1
    x = torch.randn(steps, 2 * rows, heads, dim, device=dev, generator=g).bfloat16()

    def fresh():
        return q3s.PagedCache(rows, 31, layers=1, kv_heads=heads, dim=dim, block_size=block, max_blocks=6, device=dev)

    def step(cache, n, r, y):
        t = cache.step(n, max_tokens=2 * rows, released=r)
        cache.append(0, y, y)
        return cache.attend(0, y), t

    called = fresh()
    want = []
    for i in range(steps):
        out, t = step(called, new[i], gone[i], x[i])
        want.append((out, t.lengths.clone(), t.slot_map.clone(), t.error_word.clone()))
    cache = fresh()
    n, r, y = new[0].clone(), gone[0].clone(), x[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, t = step(cache, n, r, y)
    for i in range(steps):
        n.copy_(new[i])
        r.copy_(gone[i])
        y.copy_(x[i])
        graph.replay()
        for got, ref in zip((out, t.lengths, t.slot_map, t.error_word), want[i]):
            assert torch.equal(got, ref), i
        assert torch.equal(cache.lengths, t.lengths)
    assert torch.equal(cache.k, called.k) and torch.equal(cache.table, called.table) and torch.equal(cache.ring, called.ring)


def test_tables_with_the_largest_slot_map(dev):
    """2^31 - 1 places (26 GB): the CTAs' shares of them are counted in more than 32 bits."""
    most = 2 ** 31 - 1
    i32 = dict(dtype=torch.int32, device=dev)
    t = q3s.cache_tables(torch.tensor([5, 0], **i32), torch.tensor([2, 1], **i32), torch.tensor([[3, -1], [-1, -1]], **i32),
                         torch.tensor([7, 8], **i32), torch.tensor([0, 2], **i32), block_size=16, max_tokens=most)
    assert t.slot_map[:3].tolist() == [53, 54, 112] and t.positions[:3].tolist() == [5, 6, 0] and int(t.error_word) == 0
    assert int(t.slot_map[3:].amax()) == int(t.slot_map[3:].amin()) == -1
    assert int(t.positions[3:].amax()) == int(t.positions[3:].amin()) == 0
