"""Decode steps with drafted tokens, of a small random model on one GPU: every
row brings its last token and a few drafts, which are turned by their
positions, stored, attended to, verified against the target's logits from given
random numbers, and taken out of the cache again where they were refused.

    python examples/draft_step.py [--rows 16] [--steps 8] [--drafts 3]

The prompt goes through the same path first, as one chunk a row.  The drafter
is the model without its layers, so some of its drafts hold and some do not.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qwen3tts-streaming_b200"))
import q3s  # noqa: E402

HIDDEN, LAYERS, Q_HEADS, KV_HEADS, DIM, VOCAB, BLOCK = 512, 2, 8, 4, 64, 1024, 16


class Layer:
    """Attention with 8-bit projections; the rotary turns by three axes, as the talker's does."""

    def __init__(self, gen, dev):
        self.qkv = q3s.Int8Linear(torch.randn((Q_HEADS + 2 * KV_HEADS) * DIM, HIDDEN, device=dev, generator=gen) / HIDDEN ** 0.5)
        self.out = q3s.Int8Linear(torch.randn(HIDDEN, Q_HEADS * DIM, device=dev, generator=gen) / (Q_HEADS * DIM) ** 0.5)

    def __call__(self, cache, i, x, rotary, positions, window=0):
        y = self.qkv(norm(x)).view(x.shape[0], -1, DIM)
        q = cache.append_rotary(i, y[:, :Q_HEADS], y[:, Q_HEADS:Q_HEADS + KV_HEADS], y[:, Q_HEADS + KV_HEADS:], rotary, positions)
        return x + 0.3 * self.out(cache.attend_chunk(i, q, window=window).reshape(x.shape[0], -1))


def norm(x):
    return torch.nn.functional.rms_norm(x, x.shape[-1:])


def draw(probs, u):
    """The inverse of the cumulative sum, a row each."""
    return (probs.double().cumsum(1) <= u.double()[:, None]).sum(1).clamp(max=probs.shape[1] - 1)


def main(rows=16, steps=8, drafts=3, prompt=40, seed=0, temperature=0.7):
    """Runs the steps; returns each row's tokens, how many drafts held, and the cache."""
    dev = torch.device("cuda:0")
    q3s.load_library()
    gen = torch.Generator(device=dev).manual_seed(seed)
    layers = [Layer(gen, dev) for _ in range(LAYERS)]
    embed = torch.randn(VOCAB, HIDDEN, device=dev, generator=gen).bfloat16()
    head = q3s.Int8Linear(torch.randn(VOCAB, HIDDEN, device=dev, generator=gen) * (3 / HIDDEN ** 0.5))
    rotary = q3s.Rotary(DIM, base=1e6, sections=(12, 10, 10), interleaved=True, device=dev)
    per_row = -(-(prompt + steps * (drafts + 1)) // BLOCK) + 1
    cache = q3s.PagedCache(rows, rows * per_row, layers=LAYERS, kv_heads=KV_HEADS, dim=DIM, block_size=BLOCK, max_blocks=per_row, device=dev)

    def forward(ids, new):
        t = cache.step(new, max_tokens=ids.shape[0])
        positions = cache.positions
        x = embed[ids]
        for i, layer in enumerate(layers):
            x = layer(cache, i, x, rotary, positions)
        return t, head(norm(x))

    def uniforms(n, step):
        return q3s.philox_rows(seed, n, 1, step=step, device=dev).reshape(-1)

    # the prompt: nothing to verify but its last token's draw
    ids = torch.randint(0, VOCAB, (rows, prompt), device=dev, generator=gen)
    _, logits = forward(ids.reshape(-1), torch.full((rows,), prompt, dtype=torch.int32, device=dev))
    last = logits.view(rows, prompt, VOCAB)[:, -1].contiguous()
    each = torch.arange(rows + 1, dtype=torch.int32, device=dev)
    settled = q3s.verify_drafts(last, ids[:, -1].contiguous(), each, uniforms(rows, 0), temperature=temperature).next_ids
    tokens, held = [settled[:, None]], []
    new = torch.full((rows,), 1 + drafts, dtype=torch.int32, device=dev)
    for step in range(1, steps + 1):
        ids, proposed = [settled], [torch.zeros(rows, VOCAB, device=dev)]
        for i in range(drafts):
            proposed.append(torch.softmax(head(norm(embed[ids[-1]])).float() / temperature, 1))
            ids.append(draw(proposed[-1], uniforms(rows, 1000 * step + i)))
        t, logits = forward(torch.stack(ids, 1).reshape(-1), new)
        r = q3s.verify_drafts(logits, torch.stack(ids, 1).reshape(-1), t.query_offsets, uniforms(rows * (1 + drafts), step),
                              draft_probs=torch.stack(proposed, 1).reshape(-1, VOCAB), temperature=temperature, slot_map=t.slot_map,
                              error_word=cache.error_word)
        cache.trim(r.rejected)
        settled = r.next_ids
        tokens.append(r.tokens.view(rows, 1 + drafts))
        held.append(r.accepted)
    if int(cache.error_word) or int(t.error_word):
        raise RuntimeError(f"the decode operators reported {int(cache.error_word)}, {int(t.error_word)}")
    return torch.cat(tokens, 1), torch.stack(held), cache


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=3)
    a = ap.parse_args()
    tokens, held, cache = main(a.rows, a.steps, a.drafts)
    print("first row", [x for x in tokens[0].tolist() if x >= 0])
    print(f"drafts that held: {held.float().mean():.2f} of {a.drafts} a step; cache lengths {cache.lengths.tolist()}")
