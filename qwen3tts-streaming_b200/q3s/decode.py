"""The decode step's operators beside the sampler: the paged key/value cache's
tables and append, attention over a shared prefix, and 8-bit projections.

A step runs them in this order, from device lengths alone (no host read)::

    t = q3s.cache_tables(lengths, new, table, ring, ring_state, block_size=16, max_tokens=T, whole_rows=True)
    # for every layer:
    q3s.cache_append(k, v, k_cache, v_cache, t.slot_map)
    out = q3s.prefix_attention(q, k_cache, v_cache, t.query_offsets, table, t.lengths,
                               prefix_blocks=voice_blocks, prefix_length=voice_tokens, slot_map=t.slot_map)
    hidden = projection(out)                 # q3s.Int8Linear
    # then the codec head, the sampler and the epilogue (q3s.head_sample, q3s.StepGuard)

``PagedCache`` keeps the state that such a program carries from step to step.
The functions are thin: they call ``torch.ops.q3s.*`` (C++: argument checks,
outputs and workspace from torch's allocator, the current stream), which call
the C ABI of ``include/q3s_decode.h``.  There is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import torch_ops

#: bits of the error words (include/q3s_decode.h)
DECERR_LENGTHS, DECERR_TABLE, DECERR_POOL, DECERR_TOKENS, DECERR_BLOCK_ID, DECERR_WAIT = 1, 2, 4, 8, 16, 32

_bound: dict = {}


def _op(name: str):
    """The operator's CUDA / Meta overload, looked up once."""
    f = _bound.get(name)
    if f is None:
        f = _bound[name] = getattr(torch_ops.load(), name).default
    return f


class CacheTables(NamedTuple):
    """What ``cache_tables`` makes of one step's lengths (device tensors)."""

    query_offsets: torch.Tensor  # int32 [B+1]: row b's new tokens are [offsets[b], offsets[b+1])
    slot_map: torch.Tensor       # int64 [max_tokens]: block * block_size + place; -1: no slot
    positions: torch.Tensor      # int32 [max_tokens]: place of the token in its row
    lengths: torch.Tensor        # int32 [B]: tokens in the cache with the new ones
    free_state: torch.Tensor     # int32 [2]: the ring's first entry and number of entries
    error_word: torch.Tensor     # int32 [1]: DECERR_* bits


def cache_tables(context_lengths: torch.Tensor, new_lengths: torch.Tensor, block_table: torch.Tensor,
                 free_blocks: torch.Tensor, free_state: torch.Tensor, *, block_size: int, max_tokens: int,
                 released: Optional[torch.Tensor] = None, whole_rows: bool = False) -> CacheTables:
    """Give every row the blocks that its new tokens need, and number the
    tokens' slots, in one launch from the lengths on the GPU.

    ``block_table`` (int32 [B, max_blocks]) and the ring ``free_blocks`` are
    updated in place; lengths and ring state come back as new tensors.  Row b
    holds ``context_lengths[b]`` tokens (none where ``released[b]``: its blocks
    go to the back of the ring, for the next step) and gets ``new_lengths[b]``
    more.  A row that its table or the ring cannot serve keeps its length and
    gets slot -1 for its tokens; ``error_word`` says why.  ``max_tokens`` sizes
    the slot map: entries past the last token are -1 (positions 0), so a
    captured graph can keep one size.  With ``whole_rows`` a row whose new
    tokens end past it is refused like one that its table cannot serve; without,
    ``lengths`` counts all of its tokens, and a caller that sees
    ``DECERR_TOKENS`` must not go on from them."""
    return tuple.__new__(CacheTables, _op("cache_tables")(context_lengths, new_lengths, block_table, free_blocks,
                                                          free_state, block_size, max_tokens, released, whole_rows))


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slot_map: torch.Tensor, *, error_word: Optional[torch.Tensor] = None) -> None:
    """Write the step's keys and values ([T, kv_heads, dim], any strides with
    unit last one) into the caches ([blocks, kv_heads, block_size, dim], any
    such strides) at ``slot_map`` (int64 [T], distinct; negative: not
    stored)."""
    _op("cache_append")(k, v, k_cache, v_cache, slot_map, error_word)


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, query_offsets: torch.Tensor,
                     block_table: torch.Tensor, lengths: torch.Tensor, *,
                     prefix_blocks: Optional[torch.Tensor] = None, prefix_length: int = 0,
                     scale: Optional[float] = None, return_lse: bool = False,
                     error_word: Optional[torch.Tensor] = None, slot_map: Optional[torch.Tensor] = None):
    """Attention of a batch whose rows share a prefix, which is read and
    computed once for all of them.

    ``q`` bf16 or f16 [T, q_heads, dim] (dim 64 or 128); row b's queries are
    tokens [query_offsets[b], query_offsets[b+1]), n of them.  Query i sees
    the ``prefix_length`` tokens in ``prefix_blocks`` and the row's own tokens
    up to and including number ``lengths[b] - n + i``, in ``block_table[b]``
    (so the step's own keys are appended first).  ``scale`` defaults to
    1 / sqrt(dim).  Returns ``out`` like ``q``, and with ``return_lse`` the
    log-sum-exp of the scaled scores (fp32 [T, q_heads]), with which the
    result joins others over further keys.  A query that sees nothing gets 0
    and -inf; so does one whose entry in ``slot_map`` (int64 [T], the step's) is
    negative: a row that ``cache_tables`` refused has queries, but their keys
    were not stored, and without the slot map the row's older tokens would be
    taken for them."""
    out, lse = _op("prefix_attention")(q, k_cache, v_cache, query_offsets, block_table, lengths, prefix_blocks,
                                       prefix_length, scale, error_word, slot_map)
    return (out, lse) if return_lse else out


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """8-bit values and a scale per row (over the last dimension) of a bf16,
    f16 or fp32 tensor: scale = max|x| / 127, values = round(x * (127 /
    max|x|)), to nearest even.  A row whose largest magnitude is below 2^-100
    gets values and scale 0; one with an infinity or NaN gets values 0 and
    scale NaN."""
    return _op("quantize_rows")(x)


def int8_matmul(values: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
                dtype: torch.dtype = torch.bfloat16, bias: Optional[torch.Tensor] = None,
                error_word: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(values @ weight^T) * scales[:, None] * weight_scales (+ bias)``:
    int8 [M, K] and [N, K] (K a multiple of 16), exact 32-bit sums, fp32
    scales, bias and arithmetic after them, rounded to ``dtype`` at the end.
    ``error_word`` (int32 [1]) gets ``DECERR_WAIT`` if a device wait gave up, which leaves the result
    incomplete."""
    return _op("int8_matmul")(values, scales, weight, weight_scales, dtype, bias, error_word)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
                bias: Optional[torch.Tensor] = None, return_quantized: bool = False,
                error_word: Optional[torch.Tensor] = None):
    """``quantize_rows(x)`` times an int8 weight [N, K] with a scale per
    output: y [..., N] in x's type.  ``return_quantized`` also returns the
    values and scales of x, for another product of the same activations
    (``int8_matmul``); ``error_word`` as there."""
    y, values, scales = _op("int8_linear")(x, weight, weight_scales, bias, error_word)
    return (y, values, scales) if return_quantized else y


class Int8Linear:
    """A Linear whose weight is held as int8 with a scale per output channel,
    quantised once from ``weight`` [N, K] (``nn.Linear.weight``; K a multiple
    of 16).  ``error_word`` collects ``DECERR_*`` bits of its calls."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None):
        self.weight, self.scales = quantize_rows(weight)
        self.bias = None if bias is None else bias.float().contiguous()
        self.error_word = torch.zeros(1, dtype=torch.int32, device=self.weight.device)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return int8_linear(x, self.weight, self.scales, bias=self.bias, error_word=self.error_word)


class PagedCache:
    """The state of a paged key/value cache of ``layers`` layers for ``batch``
    rows, and the three calls of a step on it.

    ``blocks`` blocks of ``block_size`` tokens; the first ``prefix_blocks`` of
    them are set aside for a prefix that all rows share (``prefix``), the rest
    are the ring that rows draw from.  ``step`` leaves the row lengths, the
    ring and the step's tables on the device and reads nothing back.
    ``tables.error_word`` reports on the step, ``error_word`` collects the
    ``DECERR_*`` bits of ``append`` and ``attend``."""

    def __init__(self, batch: int, blocks: int, *, layers: int, kv_heads: int, dim: int, block_size: int = 16,
                 max_blocks: int, prefix_blocks: int = 0, dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dev.type != "cuda":
            raise ValueError("PagedCache lives on a CUDA device")
        if not 0 <= prefix_blocks < blocks:
            raise ValueError(f"{prefix_blocks} prefix blocks of {blocks}")
        i32 = dict(dtype=torch.int32, device=dev)
        self.block_size, self.batch = block_size, batch
        self.k = torch.zeros(layers, blocks, kv_heads, block_size, dim, dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.prefix = torch.arange(prefix_blocks, **i32)
        self.prefix_length = 0
        self.ring = torch.arange(prefix_blocks, blocks, **i32)
        self.ring_state = torch.tensor([0, blocks - prefix_blocks], **i32)
        self.table = torch.full((batch, max_blocks), -1, **i32)
        self.lengths = torch.zeros(batch, **i32)
        self.error_word = torch.zeros(1, **i32)
        self.tables: Optional[CacheTables] = None

    def write_prefix(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The shared prefix's keys and values of one layer ([P, kv_heads, dim])."""
        if k.shape[0] > self.prefix.numel() * self.block_size:
            raise ValueError(f"a prefix of {k.shape[0]} tokens in {self.prefix.numel()} blocks of {self.block_size}")
        self.prefix_length = k.shape[0]
        # the prefix's blocks are the cache's first ones, in order: token p has slot p
        cache_append(k, v, self.k[layer], self.v[layer], torch.arange(k.shape[0], device=k.device), error_word=self.error_word)

    def step(self, new_lengths: torch.Tensor, max_tokens: int, released: Optional[torch.Tensor] = None) -> CacheTables:
        """Start a step that adds ``new_lengths`` tokens to the rows.  A row
        that its table or the ring cannot serve, or whose tokens end past
        ``max_tokens``, is refused: it keeps its length and its new tokens get
        slot -1; ``error_word`` of the result says why."""
        t = cache_tables(self.lengths, new_lengths, self.table, self.ring, self.ring_state,
                         block_size=self.block_size, max_tokens=max_tokens, released=released, whole_rows=True)
        self.lengths.copy_(t.lengths)  # in place: a captured step goes on from what the last replay left
        self.ring_state.copy_(t.free_state)
        self.tables = t
        return t

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Store this step's keys and values of one layer ([max_tokens, kv_heads, dim])."""
        cache_append(k, v, self.k[layer], self.v[layer], self.tables.slot_map, error_word=self.error_word)

    def attend(self, layer: int, q: torch.Tensor, **kw):
        """This step's queries of one layer ([max_tokens, q_heads, dim]) over
        prefix and rows; those of a refused row get 0 (and a log-sum-exp of -inf)."""
        slots = self.tables.slot_map
        if q.shape[0] != slots.shape[0]:  # queries past the step's tokens have no slot
            slots = torch.nn.functional.pad(slots, (0, q.shape[0] - slots.shape[0]), value=-1)
        return prefix_attention(q, self.k[layer], self.v[layer], self.tables.query_offsets, self.table, self.lengths,
                                prefix_blocks=self.prefix, prefix_length=self.prefix_length,
                                **{"error_word": self.error_word, "slot_map": slots, **kw})
