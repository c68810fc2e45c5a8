"""The decode step's operators beside the sampler: the paged key/value cache's
tables and append, attention over a shared prefix, 8-bit projections, and what a
step of several tokens a row needs: rotary positions, attention of chunks,
drafts verified, rows cut back.

A step runs them in this order, from device lengths alone (no host read)::

    t = q3s.cache_tables(lengths, new, table, ring, ring_state, block_size=16, max_tokens=T, whole_rows=True)
    # for every layer:
    q3s.cache_append(k, v, k_cache, v_cache, t.slot_map)
    out = q3s.prefix_attention(q, k_cache, v_cache, t.query_offsets, table, t.lengths,
                               prefix_blocks=voice_blocks, prefix_length=voice_tokens, slot_map=t.slot_map)
    hidden = projection(out)                 # q3s.Int8Linear
    # then the codec head, the sampler and the epilogue (q3s.head_sample, q3s.StepGuard)

A step whose rows bring several tokens (drafts, a prompt in chunks)::

    t = q3s.cache_tables(...)                # new: 1 + drafts, or the chunk's length
    # for every layer:
    q = q3s.rotary_append(q, k, v, t.positions + voice_tokens, inv_freq, k_cache, v_cache, t.slot_map)
    out = q3s.chunk_attention(q, k_cache, v_cache, t.query_offsets, table, t.lengths,
                              prefix_blocks=voice_blocks, prefix_length=voice_tokens, slot_map=t.slot_map)
    # then the head's logits, and
    r = q3s.verify_drafts(logits, ids, t.query_offsets, uniforms, draft_probs=proposed, slot_map=t.slot_map)
    c = q3s.cache_trim(t.lengths, r.rejected, table, ring, t.free_state, block_size=16)

``PagedCache`` keeps the state that such a program carries from step to step.
The functions are thin: they call ``torch.ops.q3s.*`` (C++: argument checks,
outputs and workspace from torch's allocator, the current stream), which call
the C ABI of ``include/q3s_decode.h``.  There is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import torch_ops

#: bits of the error words (include/q3s_decode.h)
DECERR_LENGTHS, DECERR_TABLE, DECERR_POOL, DECERR_TOKENS, DECERR_BLOCK_ID, DECERR_WAIT = 1, 2, 4, 8, 16, 32
DECERR_VALUES = 64

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


class CacheTrim(NamedTuple):
    """What ``cache_trim`` leaves (device tensors)."""

    lengths: torch.Tensor     # int32 [B]: tokens that stay in the cache
    free_state: torch.Tensor  # int32 [2]: the ring's first entry and number of entries
    error_word: torch.Tensor  # int32 [1]: DECERR_* bits


def cache_trim(lengths: torch.Tensor, removed: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
               free_state: torch.Tensor, *, block_size: int) -> CacheTrim:
    """Take the last ``removed[b]`` tokens of every row back out of the cache,
    in one launch: the blocks that a row no longer needs go to the back of the
    ring ``free_blocks`` (updated in place) in row order.  ``block_table`` is
    only read: entries past a row's blocks mean nothing.  ``removed`` outside
    [0, lengths[b]] is cut to it (``DECERR_LENGTHS``)."""
    return tuple.__new__(CacheTrim, _op("cache_trim")(lengths, removed, block_table, free_blocks, free_state, block_size))


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections: Optional[Sequence[int]] = None,
           interleaved: bool = False, adjacent: bool = False, scale: float = 1.0) -> torch.Tensor:
    """Rotary positions of ``x`` [T, heads, dim] (bf16, f16 or fp32, any
    strides with unit last one): a new tensor in which pair i of every head is
    turned by ``positions[axis(i)][t] * inv_freq[i]``.

    ``inv_freq`` fp32 [P] turns the first 2 P dims (2 P <= dim; the others are
    copied), as pairs (i, i + P), or (2 i, 2 i + 1) with ``adjacent``.
    ``positions`` int32 [T], or [axes, T] for several axes (time, height, width),
    whose pairs ``sections`` counts (``sum(sections) == P``): the first
    sections[0] pairs turn with axis 0 and so on, or with ``interleaved`` pair i
    with axis i % axes while i < axes * sections[i % axes], else with axis 0.
    The angle is exact to 64 bits, far positions included; cos and sin are
    multiplied by ``scale``."""
    return _op("rotary")(x, positions, inv_freq, sections or (), interleaved, adjacent, scale)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, slot_map: torch.Tensor, *,
                  sections: Optional[Sequence[int]] = None, interleaved: bool = False, adjacent: bool = False,
                  scale: float = 1.0, error_word: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rotary`` of the step's queries and keys and ``cache_append`` of the
    turned keys and the values, in one launch that reads and writes each once.
    Returns the queries."""
    return _op("rotary_append")(q, k, v, positions, inv_freq, k_cache, v_cache, slot_map, sections or (), interleaved,
                                adjacent, scale, error_word)


class Rotary:
    """Rotary positions of one model: frequencies base^(-i / P) of P pairs
    (``pairs``, by default dim / 2) and how the pairs lie.  ``inv_freq`` may be given
    instead of ``base`` (scaled variants), with their factor as ``scale``."""

    def __init__(self, dim: int, *, base: float = 10000.0, pairs: Optional[int] = None,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False, adjacent: bool = False,
                 scale: float = 1.0, inv_freq: Optional[torch.Tensor] = None, device: Optional[torch.device] = None):
        pairs = dim // 2 if pairs is None else pairs
        if not 1 <= pairs <= dim // 2:
            raise ValueError(f"{pairs} pairs of {dim} elements")
        if inv_freq is None:
            inv_freq = (float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()
        elif inv_freq.shape != (pairs,):
            raise ValueError(f"inv_freq of shape {tuple(inv_freq.shape)} for {pairs} pairs")
        if sections is not None and sum(sections) != pairs:
            raise ValueError(f"sections {list(sections)} of {pairs} pairs")
        self.inv_freq = inv_freq.float().contiguous().to(device if device is not None else "cuda")
        self.how = dict(sections=None if sections is None else tuple(sections), interleaved=interleaved, adjacent=adjacent, scale=scale)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        return rotary(x, positions, self.inv_freq, **self.how)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor, slot_map: torch.Tensor, *, error_word: Optional[torch.Tensor] = None) -> torch.Tensor:
        return rotary_append(q, k, v, positions, self.inv_freq, k_cache, v_cache, slot_map, error_word=error_word, **self.how)


def chunk_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, query_offsets: torch.Tensor,
                    block_table: torch.Tensor, lengths: torch.Tensor, *, prefix_blocks: Optional[torch.Tensor] = None,
                    prefix_length: int = 0, window: int = 0, scale: Optional[float] = None, return_lse: bool = False,
                    error_word: Optional[torch.Tensor] = None, slot_map: Optional[torch.Tensor] = None):
    """Attention of every row's chunk of new tokens over the shared prefix and
    its own pages: ``prefix_attention`` for rows of many query tokens (a prompt
    in chunks, drafts), with an optional sliding window.

    Arguments and results as there, up to 128 query heads for a key/value head,
    ``scale`` positive.  With ``window`` a query sees the ``window`` keys up to
    its own, counted over prefix and own tokens together.  Every row's query
    tokens are taken in tiles of 128 (tokens times heads of a group); where they
    are too few for that (at most 112, or 20 a row of the batch), without a
    window, the call is ``prefix_attention``'s, whose tiles are 16.  Rows without
    tokens count there: leave them out of a call for one long chunk, or give a
    window that leaves nothing out (2**31 - 1), which always takes tiles of 128.
    These round probabilities to the type of ``q`` once, as ``prefix_attention``
    does over a large batch's prefix."""
    out, lse = _op("chunk_attention")(q, k_cache, v_cache, query_offsets, block_table, lengths, prefix_blocks,
                                      prefix_length, window, scale, error_word, slot_map)
    return (out, lse) if return_lse else out


class VerifiedDrafts(NamedTuple):
    """What ``verify_drafts`` decides (device tensors)."""

    tokens: torch.Tensor    # int64 [T]: from each row's first place on its accepted drafts, then what it drew; -1 elsewhere
    accepted: torch.Tensor  # int32 [B]: drafts accepted
    rejected: torch.Tensor  # int32 [B]: drafts not accepted (their tokens are in the cache: cache_trim takes them out)
    next_ids: torch.Tensor  # int64 [B]: what the row drew, its next settled token; -1 for a row without tokens


def verify_drafts(logits: torch.Tensor, ids: torch.Tensor, query_offsets: torch.Tensor, uniforms: torch.Tensor, *,
                  draft_probs: Optional[torch.Tensor] = None, temperature: Union[float, torch.Tensor] = 1.0,
                  slot_map: Optional[torch.Tensor] = None, error_word: Optional[torch.Tensor] = None) -> VerifiedDrafts:
    """Speculative sampling's decision, from given random numbers: which
    drafted tokens of a step hold against the target's probabilities, and what
    every row draws behind them, so that the tokens are distributed as the
    target's alone.

    Row b's tokens are [query_offsets[b], query_offsets[b+1]) of the step: one
    that is settled, then drafts.  ``logits`` [T, V] (bf16, f16 or fp32) are the
    target's for the token after each; ``ids`` int64 [T] the tokens;
    ``draft_probs`` fp32 [T, V] the distributions that they were drawn from
    (without: each was certain, as from a lookup); ``uniforms`` fp32 [T] in
    [0, 1).  With p = softmax(logits / temperature), a draft d at token t holds
    if ``uniforms[t] * draft_probs[t, d] < p[t - 1, d]``; behind the last that
    does the row draws from max(p - draft_probs, 0), or from p after all of them,
    by the inverse of the cumulative sum at the uniform of the row's first token.
    ``temperature`` is a number or fp32 [B]; 0 is greedy (ties: the lowest
    index).  Logits of -inf (what top-k or a mask left out) have no probability.
    A row with a negative entry in ``slot_map`` (refused by ``cache_tables``) is
    treated like one without tokens.  ``error_word``: ``DECERR_VALUES``,
    ``DECERR_LENGTHS``."""
    heat = (temperature, 1.0) if isinstance(temperature, torch.Tensor) else (None, temperature)
    return tuple.__new__(VerifiedDrafts, _op("verify_drafts")(logits, ids, query_offsets, uniforms, draft_probs, *heat, slot_map,
                                                              error_word))


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
    rows, and the calls of a step on it: ``step``, ``append`` or
    ``append_rotary``, ``attend`` or ``attend_chunk``, and ``trim``.

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

    @property
    def positions(self) -> torch.Tensor:
        """Places of the step's tokens behind the prefix (int32 [max_tokens]): what a rotary turns them by."""
        return self.tables.positions + self.prefix_length

    def append_rotary(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rotary: Rotary,
                      positions: torch.Tensor) -> torch.Tensor:
        """``append`` of keys that ``rotary`` turns by ``positions`` (``self.positions``, or [axes, max_tokens]), and the
        queries turned likewise, in one launch."""
        return rotary.append(q, k, v, positions, self.k[layer], self.v[layer], self.tables.slot_map, error_word=self.error_word)

    def attend_chunk(self, layer: int, q: torch.Tensor, *, window: int = 0, **kw):
        """``attend`` for rows that bring many tokens (a prompt, drafts), with an optional sliding window over prefix and row."""
        slots = self.tables.slot_map
        if q.shape[0] != slots.shape[0]:
            slots = torch.nn.functional.pad(slots, (0, q.shape[0] - slots.shape[0]), value=-1)
        return chunk_attention(q, self.k[layer], self.v[layer], self.tables.query_offsets, self.table, self.lengths,
                               prefix_blocks=self.prefix, prefix_length=self.prefix_length, window=window,
                               **{"error_word": self.error_word, "slot_map": slots, **kw})

    def trim(self, removed: torch.Tensor) -> None:
        """Take the last ``removed[b]`` tokens of every row back out (``verify_drafts``' rejected ones): lengths and the ring
        go on without them.  ``error_word`` collects what ``cache_trim`` reports."""
        t = cache_trim(self.lengths, removed, self.table, self.ring, self.ring_state, block_size=self.block_size)
        self.lengths.copy_(t.lengths)  # in place, as step does
        self.ring_state.copy_(t.free_state)
        self.error_word.bitwise_or_(t.error_word)
