"""The decode step's operators without a GPU: the C ABI refuses bad arguments
on the host, the torch operators refuse CPU tensors and trace, and the plain
forms that the GPU tests compare with agree with small cases worked by hand."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import decode_reference as R
import q3s
from q3s import _lib

REPO = Path(__file__).resolve().parents[1]
P = 0x7F0000001000  # a pointer that is never followed: every call here is refused first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "q3s_decode.h").read_text(), flags=re.S)
    assert set(re.findall(r"\b(q3s_\w+)\s*\(", text)) == set(_lib.DECODE_EXPORTS)
    for name in _lib.DECODE_EXPORTS:
        assert getattr(lib, name)
    assert lib.q3s_decode_desc_size(99) == 0


GOOD = {
    "q3s_cache_tables": (_lib.CacheTablesDesc, dict(
        batch=4, block_size=16, max_blocks=8, context_lengths=P, new_lengths=P + 64, block_table=P, block_table_stride=8,
        free_blocks=P, free_state=P, free_state_out=P + 64, lengths_out=P + 128, query_offsets=P, slot_map=P, positions=P,
        ring_size=10, max_tokens=5)),
    "q3s_cache_append": (_lib.CacheAppendDesc, dict(
        tokens=3, kv_heads=2, dim=64, block_size=16, blocks=9, elem=1, k=P, v=P, slot_map=P, k_cache=P, v_cache=P)),
    "q3s_prefix_attention": (_lib.PrefixAttentionDesc, dict(
        batch=2, tokens=2, q_heads=8, kv_heads=4, dim=64, block_size=16, blocks=9, elem=1, max_blocks=4, prefix_length=20,
        scale=0.1, q=P, k_cache=P, v_cache=P, query_offsets=P, block_table=P, block_table_stride=4, lengths=P,
        prefix_blocks=P, out=P, workspace=P, workspace_bytes=1 << 40)),
    "q3s_quantize_rows": (_lib.QuantizeRowsDesc, dict(
        rows=2, cols=32, elem=1, x=P, x_row_stride=32, values=P, values_row_stride=32, scales=P)),
    "q3s_int8_matmul": (_lib.Int8MatmulDesc, dict(
        rows=2, inputs=32, outputs=5, elem=1, a=P, a_row_stride=32, a_scales=P, w=P, w_row_stride=32, w_scales=P, y=P,
        y_row_stride=5)),
}


def _call(lib, name, **kw):
    cls, good = GOOD[name]
    d = cls(**{"struct_size": C.sizeof(cls), **good, **kw})
    return getattr(lib, name)(C.byref(d), None), _lib.last_error()


@pytest.mark.parametrize("name,kw,msg", [
    ("q3s_cache_tables", dict(struct_size=8), "struct_size"),
    ("q3s_cache_tables", dict(batch=-1), "batch"),
    ("q3s_cache_tables", dict(batch=65537), "batch"),
    ("q3s_cache_tables", dict(block_size=0), "block_size"),
    ("q3s_cache_tables", dict(max_blocks=0), "max_blocks"),
    ("q3s_cache_tables", dict(max_blocks=1 << 27, block_table_stride=1 << 27), "31 bits"),
    ("q3s_cache_tables", dict(ring_size=0), "ring_size"),
    ("q3s_cache_tables", dict(max_tokens=-1), "max_tokens"),
    ("q3s_cache_tables", dict(free_state=None), "required"),
    ("q3s_cache_tables", dict(new_lengths=None), "required"),
    ("q3s_cache_tables", dict(slot_map=None), "slot_map"),
    ("q3s_cache_tables", dict(block_table_stride=7), "block_table_stride"),
    ("q3s_cache_tables", dict(lengths_out=P), "must not be"),
    ("q3s_cache_tables", dict(free_state_out=P), "must not be"),
    ("q3s_cache_append", dict(struct_size=8), "struct_size"),
    ("q3s_cache_append", dict(tokens=-1), "tokens"),
    ("q3s_cache_append", dict(dim=0), "dim"),
    ("q3s_cache_append", dict(elem=7), "elem"),
    ("q3s_cache_append", dict(slot_map=None), "slot_map"),
    ("q3s_cache_append", dict(kv_heads=1 << 20, dim=1 << 10), "2^24"),
    ("q3s_prefix_attention", dict(struct_size=8), "struct_size"),
    ("q3s_prefix_attention", dict(batch=-1), "batch"),
    ("q3s_prefix_attention", dict(tokens=-1), "tokens"),
    ("q3s_prefix_attention", dict(q_heads=6), "query heads"),
    ("q3s_prefix_attention", dict(q_heads=68), "query heads"),
    ("q3s_prefix_attention", dict(dim=96), "dim"),
    ("q3s_prefix_attention", dict(block_size=8), "block_size"),
    ("q3s_prefix_attention", dict(elem=0), "elem"),
    ("q3s_prefix_attention", dict(blocks=0), "blocks"),
    ("q3s_prefix_attention", dict(prefix_length=-1), "prefix_length"),
    ("q3s_prefix_attention", dict(prefix_length=2 ** 31 - 1), "2^31"),
    ("q3s_prefix_attention", dict(prefix_blocks=None), "prefix_blocks"),
    ("q3s_prefix_attention", dict(out=None), "required"),
    ("q3s_prefix_attention", dict(lengths=None), "lengths"),
    ("q3s_prefix_attention", dict(q=P + 8), "16-byte"),
    ("q3s_prefix_attention", dict(k_place_stride=100), "multiples of 8"),
    ("q3s_prefix_attention", dict(workspace_bytes=100), "workspace of 100"),
    ("q3s_quantize_rows", dict(struct_size=8), "struct_size"),
    ("q3s_quantize_rows", dict(rows=-1), "rows"),
    ("q3s_quantize_rows", dict(cols=0), "cols"),
    ("q3s_quantize_rows", dict(elem=3), "elem"),
    ("q3s_quantize_rows", dict(scales=None), "required"),
    ("q3s_quantize_rows", dict(x_row_stride=31), "strides"),
    ("q3s_int8_matmul", dict(struct_size=8), "struct_size"),
    ("q3s_int8_matmul", dict(rows=-1), "rows"),
    ("q3s_int8_matmul", dict(outputs=0), "outputs"),
    ("q3s_int8_matmul", dict(inputs=40), "multiple of 16"),
    ("q3s_int8_matmul", dict(inputs=131088), "multiple of 16"),
    ("q3s_int8_matmul", dict(elem=9), "elem"),
    ("q3s_int8_matmul", dict(w_scales=None), "required"),
    ("q3s_int8_matmul", dict(a=P + 4), "16 bytes"),
    ("q3s_int8_matmul", dict(w_row_stride=24), "16 bytes"),
    ("q3s_int8_matmul", dict(y_row_stride=4), "y_row_stride"),
])
def test_bad_arguments_are_refused_on_the_host(lib, name, kw, msg):
    status, text = _call(lib, name, **kw)
    assert status in (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED)
    assert msg in text, text


@pytest.mark.parametrize("name,kw", [("q3s_cache_append", dict(tokens=0)), ("q3s_prefix_attention", dict(tokens=0)),
                                     ("q3s_quantize_rows", dict(rows=0)), ("q3s_int8_matmul", dict(rows=0))])
def test_empty_calls_do_nothing(lib, name, kw):
    assert _call(lib, name, **kw)[0] == _lib.OK
    assert getattr(lib, name)(None, None) == _lib.ERR_INVALID_ARGUMENT


def test_attention_workspace_grows_with_the_batch(lib):
    cls, good = GOOD["q3s_prefix_attention"]
    sizes = []
    for tokens in (1, 64, 4096):
        d = cls(struct_size=C.sizeof(cls), **{**good, "batch": tokens, "tokens": tokens})
        n = C.c_int64()
        assert lib.q3s_prefix_attention_workspace(C.byref(d), C.byref(n)) == _lib.OK
        sizes.append(n.value)
    assert 0 < sizes[0] <= sizes[1] < sizes[2]
    assert lib.q3s_prefix_attention_workspace(C.byref(d), None) == _lib.ERR_INVALID_ARGUMENT


def test_python_calls_refuse_cpu_tensors_and_trace_on_meta():
    x = torch.zeros(2, 32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        q3s.quantize_rows(x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        q3s.cache_append(x, x, x, x, x)
    m = dict(device="meta")
    y, v, s = q3s.int8_linear(torch.empty(3, 4, 32, **m), torch.empty(7, 32, dtype=torch.int8, **m), torch.empty(7, **m),
                              return_quantized=True)
    assert y.shape == (3, 4, 7) and v.shape == (3, 4, 32) and v.dtype == torch.int8 and s.shape == (3, 4)
    i = dict(dtype=torch.int32, **m)
    t = q3s.cache_tables(torch.empty(5, **i), torch.empty(5, **i), torch.empty(5, 8, **i), torch.empty(9, **i),
                         torch.empty(2, **i), block_size=16, max_tokens=11)
    assert t.slot_map.shape == (11,) and t.slot_map.dtype == torch.int64 and t.query_offsets.shape == (6,)
    q = torch.empty(6, 8, 64, dtype=torch.bfloat16, **m)
    out, lse = q3s.prefix_attention(q, q, q, torch.empty(6, **i), torch.empty(5, 8, **i), torch.empty(5, **i), return_lse=True)
    assert out.shape == q.shape and lse.shape == (6, 8) and lse.dtype == torch.float32


def test_reference_tables_by_hand():
    """Three rows of blocks of 4: one full and growing, one that ends, one that starts with six tokens."""
    r = R.cache_tables([4, 5, 0], [1, 0, 6], [[7, -1], [3, 2], [-1, -1]], [9, 8, 6, -1, -1], [0, 3], block_size=4,
                       max_tokens=8, released=[0, 1, 0])
    assert r["table"].tolist() == [[7, 9], [3, 2], [8, 6]] and r["ring"].tolist() == [9, 8, 6, 3, 2]
    assert r["free_state"].tolist() == [3, 2] and r["lengths"].tolist() == [5, 0, 6]
    assert r["query_offsets"].tolist() == [0, 1, 1, 7]
    assert r["slot_map"].tolist() == [36, 32, 33, 34, 35, 24, 25, -1] and r["positions"].tolist() == [4, 0, 1, 2, 3, 4, 5, 0]


def test_reference_attention_by_hand():
    """One key: out is its value; two equal keys: their mean, lse = s + log 2."""
    k = torch.zeros(2, 1, 16, 64)
    v = torch.zeros(2, 1, 16, 64)
    v[0, 0, 0], v[1, 0, 0] = 1.0, 3.0
    q = torch.ones(1, 2, 64)
    out, lse, mass = R.prefix_attention(q, k, v, [0, 1], torch.tensor([[0]]), torch.tensor([1]), torch.tensor([1]), 1, 1.0)
    assert torch.allclose(out, torch.full_like(out, 2.0)) and torch.allclose(lse, torch.full_like(lse, float(np.log(2))))
    out, lse, _ = R.prefix_attention(q, k, v, [0, 1], torch.tensor([[0]]), torch.tensor([1]), torch.tensor([1]), 0, 1.0)
    assert torch.equal(out, torch.ones_like(out)) and not lse.any()
