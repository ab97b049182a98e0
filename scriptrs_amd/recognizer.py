"""Clips to token sequences: the features and the model operators as one path.

    python -m scriptrs_amd.recognizer --clips 16 --beams 4

A small encoder and a text decoder of random weights (the reference's networks
are closed bundles, src/model.rs, so there is nothing to load) show how a
program runs ``ModelOps`` behind ``ParakeetFeatureExtractor``:

  * features of a ragged batch, 8 frames stacked to an encoder frame;
  * encoder blocks over the packed frames: rotary positions, attention
    with one plan for all blocks, each sub-block's residual and the next one's norm in one call;
  * decoder steps of single tokens: grouped heads over a cache of fixed rows (a key
    mask hides what is not written yet), attention of a stream's beams over its encoder
    frames, beam selection, and the beams' caches and tokens reordered in place.
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass

import numpy as np

from .frontend import ParakeetFeatureExtractor
from .model_ops import ModelOps, RotaryTable

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

    def decode(self, encoded, offsets, beams: int = 4, steps: int = 32):
        """Beam search over each clip's encoder frames; returns (scores, tokens) of
        [clips, beams] and [clips, beams, steps], best first, ended beams filled with ``end``."""
        import torch
        c, ops, device = self.config, self.ops, self.device
        streams = len(offsets) - 1
        rows, kv = streams * beams, c.kv_heads * self.dim
        # one plan for all steps of each attention: a beam's token over its own cache, a clip's beams over its frames
        self_plan = ops.attention_plan(np.arange(rows + 1), np.arange(rows + 1) * steps, c.heads, c.kv_heads, self.dim)
        cross_plan = ops.attention_plan(np.arange(streams + 1) * beams, offsets, c.heads, c.heads, self.dim)
        cross = [(encoded @ b["kv"]).view(-1, 2, c.heads, self.dim).unbind(1) for b in self.decoder]
        cache = [torch.zeros(rows, steps, 2, c.kv_heads, self.dim, dtype=torch.bfloat16, device=device)
                 for _ in self.decoder]
        written = torch.zeros(rows, steps, dtype=torch.bool, device=device)
        tokens = torch.full((rows, steps), self.end, dtype=torch.int32, device=device)
        # a clip's beams begin alike: only the first counts
        scores = torch.full((streams, beams), -float("inf"), device=device)
        scores[:, 0] = 0.0
        finished = torch.zeros(streams, beams, dtype=torch.bool, device=device)
        token = torch.full((rows,), self.end, dtype=torch.int64, device=device)
        first = self.decoder[0]["norm"]
        for t in range(steps):
            positions = torch.full((rows,), t, dtype=torch.int32, device=device)
            written[:, t] = True
            x = torch.zeros(rows, c.width, device=device)
            x, y = ops.residual_norm(x, self.embedding[token], pre="rms", pre_weight=first, out=x)
            for i, b in enumerate(self.decoder):
                after = self.decoder[i + 1]["norm"] if i + 1 < len(self.decoder) else self.decoder_norm
                qkv = y @ b["qkv"]
                q = qkv[:, :c.width].view(rows, c.heads, self.dim)
                k = qkv[:, c.width:c.width + kv].view(rows, c.kv_heads, self.dim)
                ops.rotary(self.rotary, positions, q, k, inplace=True)
                cache[i][:, t] = qkv[:, c.width:].view(rows, 2, c.kv_heads, self.dim)
                keys, values = cache[i].view(rows * steps, 2, c.kv_heads, self.dim).unbind(1)
                y = ops.attention(self_plan, q, keys, values, key_mask=written.view(-1)).view(rows, c.width) @ b["out"]
                x, y = ops.residual_norm(x, y, pre="rms", pre_weight=b["norm_cross"], out=x, norm_out=y)
                q = (y @ b["q"]).view(rows, c.heads, self.dim)
                y = ops.attention(cross_plan, q, *cross[i]).view(rows, c.width) @ b["cross_out"]
                x, y = ops.residual_norm(x, y, pre="rms", pre_weight=b["norm_ff"], out=x, norm_out=y)
                y = torch.nn.functional.silu(y @ b["up"]) @ b["down"]
                x, y = ops.residual_norm(x, y, pre="rms", pre_weight=after, out=x, norm_out=y)
            scores, parents, chosen, finished = ops.beam_select(y @ self.head, scores, finished, self.end)
            ops.beam_reorder(parents, [*cache, tokens], out=[*cache, tokens])
            token = chosen.view(-1).long().clamp(min=0)  # (a beam without a candidate has token -1 and score -inf)
            tokens[:, t] = token
        self_plan.close()
        cross_plan.close()
        return scores, tokens.view(streams, beams, steps)

    def transcribe(self, samples, offsets, beams: int = 4, steps: int = 32):
        """(scores, tokens) of the clips ``samples[offsets[i]:offsets[i + 1]]`` of a device tensor."""
        frames, at = self.frames(samples, offsets)
        return self.decode(self.encode(frames, at), at, beams, steps)


def main() -> None:
    import torch

    from .synth import ragged_batch
    p = argparse.ArgumentParser(description="features, encoder and beam search over synthetic clips, random weights")
    p.add_argument("--clips", type=int, default=16)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--steps", type=int, default=32)
    a = p.parse_args()
    flat, offsets = ragged_batch(a.clips, 1)
    samples = torch.from_numpy(flat).cuda()
    r = Recognizer()

    def timed(f, *args):
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = f(*args)
        torch.cuda.synchronize()
        return out, 1e3 * (time.perf_counter() - t)

    for name in ("first", "second"):
        (frames, at), features_ms = timed(r.frames, samples, offsets)
        encoded, encode_ms = timed(r.encode, frames, at)
        (scores, tokens), decode_ms = timed(r.decode, encoded, at, a.beams, a.steps)
        print(f"{name} pass: {a.clips} clips, {len(samples) / 16_000:.1f} s, {int(at[-1])} encoder frames: features "
              f"{features_ms:.2f} ms, encoder {encode_ms:.2f} ms, {a.steps} steps of {a.beams} beams {decode_ms:.2f} ms")
    for i in range(min(4, a.clips)):
        print(f"clip {i}: score {scores[i, 0].item():.2f}, tokens {tokens[i, 0, :8].tolist()} ...")
    r.close()


if __name__ == "__main__":
    main()
