"""Clips to token sequences: the features and the model operators as one path.

    python -m scriptrs_amd.recognizer --clips 16 --beams 4

A small encoder and a text decoder of random weights (the reference's networks
are closed bundles, src/model.rs, so there is nothing to load) show how a
program runs ``ModelOps`` behind ``ParakeetFeatureExtractor``:

  * features of a ragged batch, 8 frames stacked to an encoder frame;
  * encoder blocks over the packed frames: rotary positions, attention
    with one plan for all blocks, each sub-block's residual and the next one's norm in one call;
  * decoder steps of single tokens: grouped heads over a cache of fixed rows (a key
    mask hides what is not written yet) or over a paged cache of 16 or 8 bits (``cache``), attention of a
    stream's beams over its encoder frames, penalties and a grammar's mask on the logits, beam selection, and
    the beams' caches and tokens reordered in place;
  * a tree of drafted tokens of each clip scored in one pass over the paged cache (``draft_logits``).
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass

import numpy as np

from .frontend import ParakeetFeatureExtractor
from .model_ops import KvCache, ModelOps, RotaryTable

STACK = 8  # feature frames in an encoder frame


@dataclass
class RecognizerConfig:
    width: int = 512
    heads: int = 8
    kv_heads: int = 2  # of the decoder's self-attention
    encoder_blocks: int = 4
    decoder_blocks: int = 2
    hidden: int = 2048
    vocab: int = 1025  # pieces, then the end of a transcript
    left: int = -1  # encoder frames that a frame sees before it, and after it
    right: int = -1
    seed: int = 0
    head_norm: bool = False  # of the decoder's queries and keys, before they are turned
    cache: str | None = None  # type of a paged cache of the decoder's (KvCache); None: dense rows
    page: int = 16  # tokens of a page


class Recognizer:
    """Encoder, decoder and beam search on one device."""

    def __init__(self, config: RecognizerConfig | None = None, device: int = 0):
        import torch
        self.config = c = config or RecognizerConfig()
        self.extractor = ParakeetFeatureExtractor(device=device)
        self.ops = ModelOps(extractor=self.extractor)
        self.device = torch.device("cuda", device)
        self.dim = c.width // c.heads
        self.rotary = RotaryTable(self.dim)
        self.end = c.vocab - 1
        g = torch.Generator(device=self.device).manual_seed(c.seed)

        def matrix(rows, columns, gain=1.0):
            w = torch.randn(rows, columns, device=self.device, generator=g) * (gain * rows ** -0.5)
            return w.to(torch.bfloat16)

        def weight():
            return 1.0 + 0.1 * torch.randn(c.width, device=self.device, generator=g)

        kv = c.kv_heads * self.dim
        self.encoder_in = matrix(STACK * 128, c.width)
        self.encoder = [{"norm": weight(), "qkv": matrix(c.width, 3 * c.width), "out": matrix(c.width, c.width),
                         "norm_ff": weight(), "up": matrix(c.width, c.hidden), "down": matrix(c.hidden, c.width)}
                        for _ in range(c.encoder_blocks)]
        self.encoder_norm = weight()
        self.embedding = matrix(c.vocab, c.width, gain=c.vocab ** 0.5)
        self.decoder = [{"norm": weight(), "qkv": matrix(c.width, c.width + 2 * kv), "out": matrix(c.width, c.width),
                         "norm_cross": weight(), "q": matrix(c.width, c.width), "kv": matrix(c.width, 2 * c.width),
                         "cross_out": matrix(c.width, c.width),
                         "norm_ff": weight(), "up": matrix(c.width, c.hidden), "down": matrix(c.hidden, c.width)}
                        for _ in range(c.decoder_blocks)]
        self.decoder_norm = weight()
        self.head = matrix(c.width, c.vocab, gain=2.0)
        if c.head_norm:
            for b in self.decoder:
                b["head_q"], b["head_k"] = (1.0 + 0.1 * torch.randn(self.dim, device=self.device, generator=g) for _ in range(2))

    def close(self) -> None:
        self.extractor.close()

    def frames(self, samples, offsets):
        """Stacked feature frames [sum of frames, 1024] of clips ``samples[offsets[i]:offsets[i + 1]]``, and where each
        clip's begin."""
        import torch
        feats, at = self.extractor.extract_batch(samples, offsets, dtype="bf16")
        parts, out = [], [0]
        for a, b in zip(at[:-1], at[1:]):
            n = int(b - a) // STACK
            x = feats[128 * int(a):128 * int(b)].view(128, int(b - a))[:, :n * STACK]
            parts.append(x.reshape(128, n, STACK).transpose(0, 1).reshape(n, 128 * STACK))
            out.append(out[-1] + n)
        return torch.cat(parts), np.asarray(out, np.int64)

    def encode(self, frames, offsets):
        """Encoder output [sum of frames, width] of packed stacked frames."""
        import torch
        c, ops = self.config, self.ops
        positions = torch.from_numpy(np.concatenate([np.arange(b - a) for a, b in zip(offsets[:-1], offsets[1:])]
                                                    ).astype(np.int32)).to(self.device)
        plan = ops.attention_plan(offsets, offsets, c.heads, c.heads, self.dim, left=c.left, right=c.right)
        x = torch.zeros(len(frames), c.width, device=self.device)  # (the residual stream stays in 32 bits)
        x, y = ops.residual_norm(x, frames @ self.encoder_in, pre="rms", pre_weight=self.encoder[0]["norm"], out=x)
        for i, b in enumerate(self.encoder):
            after = self.encoder[i + 1]["norm"] if i + 1 < len(self.encoder) else self.encoder_norm
            qkv = (y @ b["qkv"]).view(-1, 3, c.heads, self.dim)
            q, k, v = qkv.unbind(1)
            ops.rotary(self.rotary, positions, q, k, inplace=True)
            y = ops.attention(plan, q, k, v).view(-1, c.width) @ b["out"]
            x, y = ops.residual_norm(x, y, pre="rms", pre_weight=b["norm_ff"], out=x, norm_out=y)
            y = torch.nn.functional.silu(y @ b["up"]) @ b["down"]
            x, y = ops.residual_norm(x, y, scale=0.5, pre="rms", pre_weight=after, out=x, norm_out=y)
        plan.close()
        return y

    def _turn(self, block, positions, q, k):
        """Queries and keys normed (if the decoder does) and turned, in place."""
        if self.config.head_norm:
            self.ops.norm_rotary(self.rotary, positions, q, k, q_weight=block["head_q"], k_weight=block["head_k"],
                                 inplace=True)
        else:
            self.ops.rotary(self.rotary, positions, q, k, inplace=True)

    def _pages(self, sequences, tokens):
        """Paged caches of the decoder's blocks for ``tokens`` of each sequence, and the table of their pages: a sequence's
        lie side by side, so that a cache's rows are the sequences'."""
        import torch
        c = self.config
        each = -(-tokens // c.page)
        caches = [KvCache(sequences * each, c.page, c.kv_heads, self.dim, dtype=c.cache or "bf16", device=self.device.index)
                  for _ in self.decoder]
        table = torch.arange(sequences * each, dtype=torch.int32, device=self.device).view(sequences, each)
        return caches, table

    def _decoder(self, x, y, positions, attend, cross_plan, cross):
        """The decoder's blocks: ``attend(i, q, kv)`` is block i's attention over its own tokens."""
        import torch
        c, ops, rows = self.config, self.ops, len(x)
        kv = c.kv_heads * self.dim
        for i, b in enumerate(self.decoder):
            after = self.decoder[i + 1]["norm"] if i + 1 < len(self.decoder) else self.decoder_norm
            qkv = y @ b["qkv"]
            q = qkv[:, :c.width].view(rows, c.heads, self.dim)
            k = qkv[:, c.width:c.width + kv].view(rows, c.kv_heads, self.dim)
            self._turn(b, positions, q, k)
            y = attend(i, q, qkv[:, c.width:].view(rows, 2, c.kv_heads, self.dim)).view(rows, c.width) @ b["out"]
            x, y = ops.residual_norm(x, y, pre="rms", pre_weight=b["norm_cross"], out=x, norm_out=y)
            q = (y @ b["q"]).view(rows, c.heads, self.dim)
            y = ops.attention(cross_plan, q, *cross[i]).view(rows, c.width) @ b["cross_out"]
            x, y = ops.residual_norm(x, y, pre="rms", pre_weight=b["norm_ff"], out=x, norm_out=y)
            y = torch.nn.functional.silu(y @ b["up"]) @ b["down"]
            x, y = ops.residual_norm(x, y, pre="rms", pre_weight=after, out=x, norm_out=y)
        return y

    def decode(self, encoded, offsets, beams: int = 4, steps: int = 32, repetition: float = 1.0, frequency: float = 0.0,
               allowed=None):
        """Beam search over each clip's encoder frames; returns (scores, tokens) of
        [clips, beams] and [clips, beams, steps], best first, ended beams filled with ``end``.
        ``repetition``, ``frequency``: penalties for the beam's own tokens; ``allowed`` [1, words] int32: the
        tokens that may be chosen (``ModelOps.adjust_logits``)."""
        import torch
        c, ops, device = self.config, self.ops, self.device
        streams = len(offsets) - 1
        rows = streams * beams
        # one plan for all steps of each attention: a beam's token over its own cache, a clip's beams over its frames
        cross_plan = ops.attention_plan(np.arange(streams + 1) * beams, offsets, c.heads, c.heads, self.dim)
        cross = [(encoded @ b["kv"]).view(-1, 2, c.heads, self.dim).unbind(1) for b in self.decoder]
        tokens = torch.full((rows, steps), self.end, dtype=torch.int32, device=device)
        lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        if c.cache is None:
            self_plan = ops.attention_plan(np.arange(rows + 1), np.arange(rows + 1) * steps, c.heads, c.kv_heads, self.dim)
            cache = [torch.zeros(rows, steps, 2, c.kv_heads, self.dim, dtype=torch.bfloat16, device=device)
                     for _ in self.decoder]
            written = torch.zeros(rows, steps, dtype=torch.bool, device=device)
            states = [*cache, tokens]

            def attend(i, q, kv):
                cache[i][:, t] = kv
                keys, values = cache[i].view(rows * steps, 2, c.kv_heads, self.dim).unbind(1)
                return ops.attention(self_plan, q, keys, values, key_mask=written.view(-1))
        else:
            self_plan = ops.cache_plan(np.arange(rows + 1), c.heads, c.kv_heads, self.dim)
            paged, table = self._pages(rows, steps)
            states = [*(p.data.view(rows, -1) for p in paged), tokens]

            def attend(i, q, kv):
                ops.cache_write(self_plan, paged[i], table, lengths, *kv.unbind(1))
                return ops.cache_attention(self_plan, paged[i], table, lengths, q)
        steered = repetition != 1.0 or frequency != 0.0 or allowed is not None
        every = None if allowed is None else torch.zeros(rows, dtype=torch.int32, device=device)
        # a clip's beams begin alike: only the first counts
        scores = torch.full((streams, beams), -float("inf"), device=device)
        scores[:, 0] = 0.0
        finished = torch.zeros(streams, beams, dtype=torch.bool, device=device)
        token = torch.full((rows,), self.end, dtype=torch.int64, device=device)
        first = self.decoder[0]["norm"]
        for t in range(steps):
            positions = torch.full((rows,), t, dtype=torch.int32, device=device)
            if c.cache is None:
                written[:, t] = True
            x = torch.zeros(rows, c.width, device=device)
            x, y = ops.residual_norm(x, self.embedding[token], pre="rms", pre_weight=first, out=x)
            lengths.fill_(t + 1)
            logits = self._decoder(x, y, positions, attend, cross_plan, cross) @ self.head
            if steered:
                ops.adjust_logits(logits, history=tokens, lengths=lengths - 1, repetition=repetition, frequency=frequency,
                                  allowed=allowed, states=every, out=logits)
            scores, parents, chosen, finished = ops.beam_select(logits, scores, finished, self.end)
            ops.beam_reorder(parents, states, out=states)
            token = chosen.view(-1).long().clamp(min=0)  # (a beam without a candidate has token -1 and score -inf)
            tokens[:, t] = token
        self_plan.close()
        cross_plan.close()
        return scores, tokens.view(streams, beams, steps)

    def draft_logits(self, encoded, offsets, tokens, parents):
        """Logits [clips, drafts, vocab] that each of ``tokens`` [clips, drafts] (at most 64) of a tree is chosen from:
        ``parents`` (a list) has the draft before it, an earlier one, or -1 for those that begin a transcript.  One pass
        over a paged cache (of bf16 without ``cache``)."""
        import torch
        c, ops, device = self.config, self.ops, self.device
        clips, n = tokens.shape
        depth, seen = [], []
        for i, p in enumerate(parents):
            depth.append(depth[p] + 1 if p >= 0 else 0)
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        tree = torch.tensor([s - (s >> 63 << 64) for s in seen], dtype=torch.int64, device=device).repeat(clips)
        positions = torch.tensor(depth, dtype=torch.int32, device=device).repeat(clips)
        previous = torch.tensor([p if p >= 0 else n for p in parents], device=device)
        # (a draft's row comes from the token before it)
        before = torch.cat([tokens.long(), tokens.new_full((clips, 1), self.end).long()], 1)[:, previous].reshape(-1)
        plan = ops.cache_plan(np.arange(clips + 1) * n, c.heads, c.kv_heads, self.dim)
        cross_plan = ops.attention_plan(np.arange(clips + 1) * n, offsets, c.heads, c.heads, self.dim)
        cross = [(encoded @ b["kv"]).view(-1, 2, c.heads, self.dim).unbind(1) for b in self.decoder]
        paged, table = self._pages(clips, n)
        lengths = torch.full((clips,), n, dtype=torch.int32, device=device)

        def attend(i, q, kv):
            ops.cache_write(plan, paged[i], table, lengths, *kv.unbind(1))
            return ops.cache_attention(plan, paged[i], table, lengths, q, tree=tree)
        x = torch.zeros(clips * n, c.width, device=device)
        x, y = ops.residual_norm(x, self.embedding[before], pre="rms", pre_weight=self.decoder[0]["norm"], out=x)
        logits = self._decoder(x, y, positions, attend, cross_plan, cross) @ self.head
        plan.close()
        cross_plan.close()
        return logits.view(clips, n, c.vocab)

    def transcribe(self, samples, offsets, beams: int = 4, steps: int = 32, **steering):
        """(scores, tokens) of the clips ``samples[offsets[i]:offsets[i + 1]]`` of a device tensor (``steering``: as for
        ``decode``)."""
        frames, at = self.frames(samples, offsets)
        return self.decode(self.encode(frames, at), at, beams, steps, **steering)


def main() -> None:
    import torch

    from .synth import ragged_batch
    p = argparse.ArgumentParser(description="features, encoder and beam search over synthetic clips, random weights")
    p.add_argument("--clips", type=int, default=16)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--cache", choices=["bf16", "e4m3", "int8"], help="a paged cache of this type for the decoder's tokens")
    p.add_argument("--head-norm", action="store_true", help="norms of the decoder's queries and keys")
    p.add_argument("--repetition", type=float, default=1.0, help="penalty for tokens said before")
    a = p.parse_args()
    flat, offsets = ragged_batch(a.clips, 1)
    samples = torch.from_numpy(flat).cuda()
    r = Recognizer(RecognizerConfig(cache=a.cache, head_norm=a.head_norm))

    def timed(f, *args, **named):
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = f(*args, **named)
        torch.cuda.synchronize()
        return out, 1e3 * (time.perf_counter() - t)

    for name in ("first", "second"):
        (frames, at), features_ms = timed(r.frames, samples, offsets)
        encoded, encode_ms = timed(r.encode, frames, at)
        (scores, tokens), decode_ms = timed(r.decode, encoded, at, a.beams, a.steps, repetition=a.repetition)
        print(f"{name} pass: {a.clips} clips, {len(samples) / 16_000:.1f} s, {int(at[-1])} encoder frames: features "
              f"{features_ms:.2f} ms, encoder {encode_ms:.2f} ms, {a.steps} steps of {a.beams} beams {decode_ms:.2f} ms")
    for i in range(min(4, a.clips)):
        print(f"clip {i}: score {scores[i, 0].item():.2f}, tokens {tokens[i, 0, :8].tolist()} ...")
    r.close()


if __name__ == "__main__":
    main()
