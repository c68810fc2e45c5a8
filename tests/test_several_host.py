"""The operators for steps of several tokens a row without a GPU: the C ABI
refuses bad arguments on the host, the torch operators refuse CPU tensors and
trace, and the plain forms that the GPU tests compare with agree with small
cases worked by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

import several_reference as R
import q3s
from q3s import _lib

P = 0x7F0000001000  # a pointer that is never followed: every call here is refused first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def sections(*x):
    return (C.c_int32 * _lib.MAX_ROTARY_AXES)(*x)


GOOD = {
    "q3s_rotary": (_lib.RotaryDesc, dict(
        tokens=3, q_heads=4, kv_heads=2, dim=64, pairs=32, axes=3, sections=sections(12, 10, 10), scale=1.0, elem=1, block_size=16,
        blocks=9, positions=P, position_stride=3, inv_freq=P, q=P, out=P + 4096, k=P, v=P, slot_map=P, k_cache=P, v_cache=P)),
    "q3s_verify_drafts": (_lib.VerifyDraftsDesc, dict(
        batch=2, tokens=5, vocab=100, elem=1, temperature_default=1.0, logits=P, logits_row_stride=100, ids=P, query_offsets=P,
        uniforms=P, draft_probs=P, draft_row_stride=100, tokens_out=P + 4096, accepted=P, rejected=P, next_ids=P)),
    "q3s_chunk_attention": (_lib.ChunkAttentionDesc, dict(
        batch=2, tokens=20, q_heads=8, kv_heads=4, dim=64, block_size=16, blocks=9, elem=1, max_blocks=4, prefix_length=20, scale=0.1,
        q=P, k_cache=P, v_cache=P, query_offsets=P, block_table=P, block_table_stride=4, lengths=P, prefix_blocks=P, out=P,
        workspace=P, workspace_bytes=1 << 40)),
    "q3s_cache_trim": (_lib.CacheTrimDesc, dict(
        batch=4, block_size=16, max_blocks=8, lengths=P, removed=P + 64, block_table=P, block_table_stride=8, free_blocks=P,
        free_state=P, free_state_out=P + 64, lengths_out=P + 128, ring_size=10)),
}


def _call(lib, name, **kw):
    cls, good = GOOD[name]
    d = cls(**{"struct_size": C.sizeof(cls), **good, **kw})
    return getattr(lib, name)(C.byref(d), None), _lib.last_error()


@pytest.mark.parametrize("name,kw,msg", [
    ("q3s_rotary", dict(struct_size=8), "struct_size"),
    ("q3s_rotary", dict(tokens=-1), "tokens"),
    ("q3s_rotary", dict(q_heads=-1), "q_heads"),
    ("q3s_rotary", dict(kv_heads=-2), "kv_heads"),
    ("q3s_rotary", dict(dim=1, pairs=1), "dim"),
    ("q3s_rotary", dict(dim=1 << 23), "2^24"),
    ("q3s_rotary", dict(pairs=0), "pairs"),
    ("q3s_rotary", dict(pairs=33), "pairs"),
    ("q3s_rotary", dict(dim=2048, pairs=513), "pairs"),
    ("q3s_rotary", dict(flags=4), "flags"),
    ("q3s_rotary", dict(elem=3), "elem"),
    ("q3s_rotary", dict(axes=0), "axes"),
    ("q3s_rotary", dict(axes=5), "axes"),
    ("q3s_rotary", dict(sections=sections(12, 10, 9)), "sections"),
    ("q3s_rotary", dict(sections=sections(33, -1, 0)), "negative"),
    ("q3s_rotary", dict(sections=sections(4, 4, 24), flags=_lib.ROTARY_INTERLEAVED), "interleaved"),
    ("q3s_rotary", dict(block_size=0), "block_size"),
    ("q3s_rotary", dict(blocks=0), "blocks"),
    ("q3s_rotary", dict(positions=None), "positions"),
    ("q3s_rotary", dict(inv_freq=None), "inv_freq"),
    ("q3s_rotary", dict(out=None), "out"),
    ("q3s_rotary", dict(out=P, q_token_stride=256, out_token_stride=512), "same strides"),
    ("q3s_rotary", dict(v_cache=None), "v_cache"),
    ("q3s_rotary", dict(slot_map=None), "slot_map"),
    ("q3s_verify_drafts", dict(struct_size=8), "struct_size"),
    ("q3s_verify_drafts", dict(batch=-1), "batch"),
    ("q3s_verify_drafts", dict(batch=65537), "batch"),
    ("q3s_verify_drafts", dict(tokens=-1), "tokens"),
    ("q3s_verify_drafts", dict(vocab=0), "vocab"),
    ("q3s_verify_drafts", dict(vocab=(1 << 24) + 1), "vocab"),
    ("q3s_verify_drafts", dict(elem=3), "elem"),
    ("q3s_verify_drafts", dict(query_offsets=None), "query_offsets"),
    ("q3s_verify_drafts", dict(next_ids=None), "next_ids"),
    ("q3s_verify_drafts", dict(uniforms=None), "uniforms"),
    ("q3s_verify_drafts", dict(logits_row_stride=99), "strides"),
    ("q3s_verify_drafts", dict(draft_row_stride=99), "strides"),
    ("q3s_verify_drafts", dict(tokens_out=P), "tokens_out"),
    ("q3s_chunk_attention", dict(struct_size=8), "struct_size"),
    ("q3s_chunk_attention", dict(batch=-1), "batch"),
    ("q3s_chunk_attention", dict(batch=65537), "batch"),
    ("q3s_chunk_attention", dict(tokens=-1), "tokens"),
    ("q3s_chunk_attention", dict(q_heads=6), "query heads"),
    ("q3s_chunk_attention", dict(q_heads=129, kv_heads=1), "query heads"),
    ("q3s_chunk_attention", dict(q_heads=65536, kv_heads=65536), "too many"),
    ("q3s_chunk_attention", dict(dim=96), "dim"),
    ("q3s_chunk_attention", dict(block_size=256), "block_size"),
    ("q3s_chunk_attention", dict(elem=0), "elem"),
    ("q3s_chunk_attention", dict(blocks=0), "blocks"),
    ("q3s_chunk_attention", dict(window=-1), "window"),
    ("q3s_chunk_attention", dict(prefix_length=-1), "prefix_length"),
    ("q3s_chunk_attention", dict(scale=0.0), "scale"),
    ("q3s_chunk_attention", dict(scale=-0.1), "scale"),
    ("q3s_chunk_attention", dict(scale=float("nan")), "scale"),
    ("q3s_chunk_attention", dict(scale=float("inf")), "scale"),
    ("q3s_chunk_attention", dict(tokens=1 << 28), "2^31"),
    ("q3s_chunk_attention", dict(prefix_length=(1 << 31) - 65600), "2^31"),
    ("q3s_chunk_attention", dict(prefix_blocks=None), "prefix_blocks"),
    ("q3s_chunk_attention", dict(out=None), "required"),
    ("q3s_chunk_attention", dict(lengths=None), "lengths"),
    ("q3s_chunk_attention", dict(q=P + 8), "16-byte"),
    ("q3s_chunk_attention", dict(k_place_stride=100), "multiples of 8"),
    ("q3s_chunk_attention", dict(workspace_bytes=100), "workspace of 100"),
    ("q3s_cache_trim", dict(struct_size=8), "struct_size"),
    ("q3s_cache_trim", dict(batch=-1), "batch"),
    ("q3s_cache_trim", dict(batch=65537), "batch"),
    ("q3s_cache_trim", dict(block_size=0), "block_size"),
    ("q3s_cache_trim", dict(max_blocks=1 << 27, block_table_stride=1 << 27), "31 bits"),
    ("q3s_cache_trim", dict(ring_size=0), "ring_size"),
    ("q3s_cache_trim", dict(free_state=None), "required"),
    ("q3s_cache_trim", dict(removed=None), "required"),
    ("q3s_cache_trim", dict(block_table_stride=7), "block_table_stride"),
    ("q3s_cache_trim", dict(lengths_out=P + 64), "must not be"),
    ("q3s_cache_trim", dict(free_state_out=P), "must not be"),
])
def test_bad_arguments_are_refused_on_the_host(lib, name, kw, msg):
    status, text = _call(lib, name, **kw)
    assert status in (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED)
    assert msg in text, text


@pytest.mark.parametrize("name,kw", [("q3s_rotary", dict(tokens=0)), ("q3s_rotary", dict(q_heads=0, kv_heads=0)),
                                     ("q3s_verify_drafts", dict(batch=0, tokens=0)), ("q3s_chunk_attention", dict(tokens=0))])
def test_empty_calls_do_nothing(lib, name, kw):
    assert _call(lib, name, **kw)[0] == _lib.OK
    assert getattr(lib, name)(None, None) == _lib.ERR_INVALID_ARGUMENT


def test_python_calls_refuse_cpu_tensors_and_trace_on_meta():
    x = torch.zeros(2, 4, 32)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        q3s.rotary(x, i, torch.zeros(16))
    with pytest.raises((RuntimeError, NotImplementedError)):
        q3s.verify_drafts(x[0], i.long(), i, torch.zeros(2))
    with pytest.raises((RuntimeError, NotImplementedError)):
        q3s.cache_trim(i, i, torch.zeros(2, 3, dtype=torch.int32), i, i, block_size=16)
    m = dict(device="meta")
    n = dict(dtype=torch.int32, **m)
    q = torch.empty(6, 8, 64, dtype=torch.bfloat16, **m)
    assert q3s.rotary(q, torch.empty(3, 6, **n), torch.empty(32, **m), sections=(12, 10, 10)).shape == q.shape
    cache = torch.empty(4, 8, 16, 64, dtype=torch.bfloat16, **m)
    y = q3s.rotary_append(q, q, q, torch.empty(6, **n), torch.empty(32, **m), cache, cache, torch.empty(6, dtype=torch.int64, **m))
    assert y.shape == q.shape and y.dtype == torch.bfloat16
    r = q3s.verify_drafts(torch.empty(6, 50, **m), torch.empty(6, dtype=torch.int64, **m), torch.empty(4, **n), torch.empty(6, **m),
                          temperature=torch.empty(3, **m))
    assert r.tokens.shape == (6,) and r.tokens.dtype == torch.int64 and r.accepted.shape == (3,) and r.accepted.dtype == torch.int32
    assert r.rejected.shape == r.next_ids.shape == (3,) and r.next_ids.dtype == torch.int64
    out, lse = q3s.chunk_attention(q, cache, cache, torch.empty(6, **n), torch.empty(5, 8, **n), torch.empty(5, **n), window=7, return_lse=True)
    assert out.shape == q.shape and lse.shape == (6, 8) and lse.dtype == torch.float32
    t = q3s.cache_trim(torch.empty(5, **n), torch.empty(5, **n), torch.empty(5, 8, **n), torch.empty(9, **n), torch.empty(2, **n), block_size=16)
    assert t.lengths.shape == (5,) and t.free_state.shape == (2,) and t.error_word.shape == (1,)


def test_reference_rotary_by_hand():
    """A quarter turn of the first pair by axis 0, half a turn of the second by axis 1; the last dim is copied."""
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0]]])
    f = torch.tensor([np.pi / 2, np.pi / 2])
    y, _, _ = R.rotary(x, torch.tensor([[1], [2]]), f, sections=(1, 1))
    assert torch.allclose(y, torch.tensor([[[-3.0, -2.0, 1.0, -4.0, 5.0]]]).double(), atol=1e-6)
    y, _, _ = R.rotary(x, torch.tensor([[1], [2]]), f, sections=(1, 1), adjacent=True)
    assert torch.allclose(y, torch.tensor([[[-2.0, 1.0, -3.0, -4.0, 5.0]]]).double(), atol=1e-6)
    assert R.rotary_axes(8, (4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0] and R.rotary_axes(4, (1, 2, 1), False) == [0, 1, 1, 2]


def test_reference_trim_by_hand():
    r = R.cache_trim([9, 4, 8], [2, 4, 1], [[7, 6, 5], [4, -1, -1], [3, 2, -1]], [9, 8, -1, -1, -1], [0, 2], block_size=4)
    assert r["lengths"] == [7, 0, 7] and r["ring"] == [9, 8, 5, 4, -1] and r["free_state"] == [0, 4] and r["error_word"] == [0]


def test_reference_verification_by_hand():
    """p = (1/2, 1/4, 1/4) everywhere, q = (1/4, 1/2, 1/4): draft 1 holds below u = 1/2; a refusal draws 0 for sure."""
    logits = np.log(np.tile(np.float32([0.5, 0.25, 0.25]), (3, 1)))
    q = np.tile(np.float32([0.25, 0.5, 0.25]), (3, 1))
    got = R.verify_drafts(logits, [0, 1, 2], [0, 3], [0.6, 0.49, 0.99], q, [1.0])
    assert got["tokens"] == [1, 2, 1] and got["accepted"] == [2] and got["rejected"] == [0] and got["next_ids"] == [1]
    got = R.verify_drafts(logits, [0, 1, 2], [0, 3], [0.6, 0.51, 0.99], q, [1.0])
    assert got["tokens"] == [0, -1, -1] and got["accepted"] == [0] and got["rejected"] == [2] and got["next_ids"] == [0]
    # a certain draft holds below p = 1/4; what is left, (1/2, 0, 1/4), reaches 0.6 * 3/4 = 0.45 with its first entry
    got = R.verify_drafts(logits, [0, 1, 2], [0, 3], [0.6, 0.3, 0.9], None, [1.0])
    assert got["tokens"] == [0, -1, -1] and got["rejected"] == [2]


def test_verified_tokens_have_the_targets_distribution():
    """The first token of a row, over a grid of the three uniforms, against p (the grid's own step is the tolerance: each
    uniform moves a share of at most vocab steps)."""
    p, q, n = np.float32([0.4, 0.35, 0.2, 0.05]), np.float32([0.1, 0.3, 0.2, 0.4]), 40
    logits, grid, count = np.tile(np.log(p), (2, 1)), (np.arange(n) + 0.5) / n, np.zeros(4)
    for drafted in grid:
        d = int(np.flatnonzero(np.cumsum(q) > drafted)[0])
        for u in grid:
            for w in grid:
                count[R.verify_drafts(logits, [0, d], [0, 2], [w, u], np.stack([q, q]), [1.0])["tokens"][0]] += 1
    assert np.abs(count / n ** 3 - p).max() < 4 * 3 / n


def test_chunk_kernel_shares_no_multiprocessor_with_another_that_takes_tensor_memory(tmp_path):
    """It takes all 512 columns, so no CTA that takes some may fit beside it (228 KB of shared memory)."""
    import subprocess
    from pathlib import Path

    from q3s import build

    src, exe = tmp_path / "chunk.cu", tmp_path / "chunk"
    src.write_text('#include <cstdio>\n#include "q3s_chunk.cuh"\nint main() { printf("%d %d %d", q3s::ChunkTile<64>::SMEM, '
                   'q3s::ChunkTile<128>::SMEM, q3s::TMEM_PART_SMEM); }\n')
    csrc = Path(__file__).resolve().parents[1] / "qwen3tts-streaming_b200" / "csrc"
    subprocess.run([build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", f"-I{csrc}", f"-I{build.INCLUDE}",
                    "-o", str(exe), str(src)], check=True, capture_output=True)
    a, b, part = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert min(a, b) + part > 228 * 1024 and max(a, b) <= 227 * 1024


def test_chunk_operator_takes_an_error_word():
    q3s.load_torch_ops()
    for name in ("chunk_attention", "rotary_append", "verify_drafts"):
        arg = {a.name: a for a in getattr(torch.ops.q3s, name).default._schema.arguments}["error_word"]
        assert arg.alias_info is not None and arg.alias_info.is_write and arg.default_value is None


def test_reference_chunk_attention_by_hand():
    """Two queries of one row on two keys with equal scores: the first sees one, the second both; a window of one, its own."""
    k, v, q = torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, 16, 64), torch.ones(2, 1, 64)
    v[0, 0, 0], v[0, 0, 1] = 1.0, 3.0
    args = ([0, 2], torch.tensor([[0]]), [2], torch.zeros(0, dtype=torch.int32), 0, 1.0)
    out, lse, spread, mass = R.chunk_attention(q, k, v, *args)
    assert out[:, 0, 0].tolist() == [1.0, 2.0] and np.allclose(lse[:, 0], [0.0, np.log(2)])
    assert spread[:, 0, 0].tolist() == [0.0, 1.0] and mass[:, 0, 0].tolist() == [1.0, 2.0]
    assert R.chunk_attention(q, k, v, *args, window=1)[0][:, 0, 0].tolist() == [1.0, 3.0]
