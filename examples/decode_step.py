"""A few decode steps of a small random model on one GPU: paged cache, shared
voice prefix, 8-bit projections, codec head, sampler and step epilogue.

    python examples/decode_step.py [--rows 48] [--steps 20]

Every step runs from device state alone -- row lengths, block tables, the free
ring and the rows' histories stay on the GPU; the host reads the epilogue's
event count.  Rows whose stream ends (EOS) give their blocks back and start
again as a new request in the next step.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qwen3tts-streaming_b200"))
import q3s  # noqa: E402

HIDDEN, LAYERS, Q_HEADS, KV_HEADS, DIM, VOCAB, BLOCK = 1024, 2, 8, 4, 128, 2048, 16


class Layer:
    """Attention and a gated feed-forward block with 8-bit weights."""

    def __init__(self, gen, dev):
        def weight(n, k):
            return torch.randn(n, k, device=dev, generator=gen) / k ** 0.5

        self.qkv = q3s.Int8Linear(weight((Q_HEADS + 2 * KV_HEADS) * DIM, HIDDEN))
        self.out = q3s.Int8Linear(weight(HIDDEN, Q_HEADS * DIM))
        self.up = q3s.Int8Linear(weight(4 * HIDDEN, HIDDEN))
        self.down = q3s.Int8Linear(weight(HIDDEN, 2 * HIDDEN))

    def split(self, x):
        """[T, hidden] -> queries, keys and values as views of one product."""
        y = self.qkv(norm(x)).view(x.shape[0], -1, DIM)
        return y[:, :Q_HEADS], y[:, Q_HEADS:Q_HEADS + KV_HEADS], y[:, Q_HEADS + KV_HEADS:]

    def finish(self, x, attended):
        x = x + self.out(attended.reshape(x.shape[0], -1))
        gate, up = self.up(norm(x)).chunk(2, -1)
        return x + self.down(torch.nn.functional.silu(gate) * up)


def norm(x):
    return torch.nn.functional.rms_norm(x, x.shape[-1:])


def main(rows=48, steps=20, voice_tokens=200, max_tokens_per_row=256, seed=0):
    """Runs the steps; returns what each row drew and the final cache lengths."""
    dev = torch.device("cuda:0")
    q3s.load_library()
    gen = torch.Generator(device=dev).manual_seed(seed)
    layers = [Layer(gen, dev) for _ in range(LAYERS)]
    embed = torch.randn(VOCAB, HIDDEN, device=dev, generator=gen).bfloat16()
    head = (torch.randn(VOCAB, HIDDEN, device=dev, generator=gen) * (3 / HIDDEN ** 0.5)).bfloat16()
    per_row = max_tokens_per_row // BLOCK
    voice_blocks = -(-voice_tokens // BLOCK)
    cache = q3s.PagedCache(rows, voice_blocks + rows * per_row, layers=LAYERS, kv_heads=KV_HEADS, dim=DIM, block_size=BLOCK,
                           max_blocks=per_row, prefix_blocks=voice_blocks, device=dev)
    eos = 7
    guard = q3s.StepGuard(rows, eos_id=eos, token_loop_abort_frames=0, device=dev)
    history = q3s.RowHistory(rows, max_tokens_per_row, device=dev)

    # the voice prompt, once for all rows: its tokens attend to themselves
    x = torch.randn(voice_tokens, HIDDEN, device=dev, generator=gen).bfloat16()
    for i, layer in enumerate(layers):
        q, k, v = layer.split(x)
        cache.write_prefix(i, k, v)
        one_row = torch.tensor([0, voice_tokens], dtype=torch.int32, device=dev)
        x = layer.finish(x, q3s.prefix_attention(q, cache.k[i], cache.v[i], one_row, cache.prefix[None],
                                                 torch.tensor([voice_tokens], dtype=torch.int32, device=dev)))

    ids = torch.randint(0, VOCAB, (rows,), device=dev, generator=gen)
    one = torch.ones(rows, dtype=torch.int32, device=dev)
    ended = torch.zeros(rows, dtype=torch.bool, device=dev)
    drawn = []
    for step in range(steps):
        t = cache.step(one, max_tokens=rows, released=ended)
        x = embed[ids]
        for i, layer in enumerate(layers):
            q, k, v = layer.split(x)
            cache.append(i, k, v)
            x = layer.finish(x, cache.attend(i, q))
        u = q3s.philox_rows(seed, rows, 1, step=step, device=dev)
        ids, _ = q3s.head_sample(norm(x), head, mode="icdf", uniforms=u, temperature=0.9, topk=50, top_p=0.95, penalty=1.05,
                                 eos_id=eos, **history.sampler_kwargs())
        guard.step(ids, rows=history)
        ended = ids == eos
        events = guard.read_events()
        done = [r for r, bits in events if bits & q3s._lib.EVT_EOS]
        if done:
            history.reset_rows(done)
            guard.reset_rows(done)
        drawn.append(ids)
    words = [t.error_word, cache.error_word] + [p.error_word for x in layers for p in (x.qkv, x.out, x.up, x.down)]
    if int(torch.stack(words).max()):
        raise RuntimeError(f"the decode operators reported {[int(w) for w in words]}")
    return torch.stack(drawn), cache.lengths


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=48)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    tokens, lengths = main(a.rows, a.steps)
    print("drawn", tuple(tokens.shape), "first row", tokens[:, 0].tolist())
    print("cache lengths", lengths.tolist())
