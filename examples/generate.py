"""Text from frames: an attention decoder that reads the encoder's output as its
prompt and writes tokens, one step for the whole batch at a time.

    python examples/generate.py [--utterances 4] [--seconds 30] [--tokens 64]

The encoder (two 4-bit blocks) and the decoder have random weights, so the
tokens mean nothing; the calls are those of a real program:

  prompt   frames of all utterances, ragged: append() fills the pages of each,
           attend() over the prompt's own tokens (causal), layer by layer
  step     one token an utterance: append(), attend(), sample(); the lengths
           stay on the GPU, and a step is captured once as a CUDA graph

Linears are the library's f16 kernel (Encoder.linear_f16); everything runs on
the encoder context's stream.
"""
from __future__ import annotations

import argparse
import importlib
import pathlib
import sys

import numpy as np
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
from __graft_entry__ import load_package  # noqa: E402

WIDTH, HEAD_DIM, HEADS, KV_HEADS, FFN = 640, 64, 10, 5, 2560
VOCAB, VOCAB_ROWS = 8193, 8320   # the head's rows are a multiple of 128


class TextDecoder:
    """Pre-norm transformer decoder over frames (WIDTH channels, the encoder's
    output) and tokens, its keys and values in one KvCache a layer."""

    def __init__(self, pkg, enc, layers: int, seqs: int, max_tokens: int, page_tokens: int = 32, seed: int = 0):
        self.pkg, self.enc, self.seqs = pkg, enc, seqs
        self.dev = torch.device("cuda", enc.device)
        g = torch.Generator(device=self.dev).manual_seed(seed)

        def weight(rows, cols):
            w = torch.randn(rows, cols, generator=g, device=self.dev) * cols ** -0.5
            return w.half().view(torch.int16)

        qkv = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.layers = [dict(qkv=weight(qkv, WIDTH), out=weight(WIDTH, WIDTH), gate=weight(FFN, WIDTH), up=weight(FFN, WIDTH),
                            down=weight(WIDTH, FFN), q_norm=torch.ones(HEAD_DIM, device=self.dev),
                            k_norm=torch.ones(HEAD_DIM, device=self.dev)) for _ in range(layers)]
        self.embed = torch.randn(VOCAB, WIDTH, generator=g, device=self.dev)
        self.head = weight(VOCAB_ROWS, WIDTH)
        pages = -(-max_tokens // page_tokens)
        self.caches = [pkg.KvCache(seqs * pages, KV_HEADS, HEAD_DIM, page_tokens, enc.device) for _ in range(layers)]
        self.table = torch.arange(seqs * pages, device=self.dev, dtype=torch.int32).reshape(seqs, pages)
        angle = torch.arange(max_tokens, device=self.dev)[:, None] * 10000.0 ** (
            -torch.arange(0, HEAD_DIM, 2, device=self.dev) / HEAD_DIM)
        self.cos, self.sin = angle.cos().contiguous(), angle.sin().contiguous()
        self.lens = torch.zeros(seqs, device=self.dev, dtype=torch.int32)
        self.one_each = torch.arange(seqs + 1, device=self.dev, dtype=torch.int32)

    def _linear(self, x, w):
        return self.enc.linear_f16(x.float().contiguous(), w)

    @staticmethod
    def _norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def forward(self, x, cu_q, max_q: int):
        """x (tokens, WIDTH) f32, the last tokens of their sequences (self.lens
        counts them); returns the hidden states."""
        for w, cache in zip(self.layers, self.caches):
            qkv = self._linear(self._norm(x), w["qkv"]).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM)
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], dim=1)
            q = cache.append(q, k, v, cu_q, self.lens, self.table, q_norm=w["q_norm"], k_norm=w["k_norm"], cos=self.cos,
                             sin=self.sin)
            a = cache.attend(q, cu_q, self.lens, self.table, max_q=max_q)
            x = x + self._linear(a.view(-1, WIDTH), w["out"])
            y = self._norm(x)
            y = torch.nn.functional.silu(self._linear(y, w["gate"])) * self._linear(y, w["up"])
            x = x + self._linear(y, w["down"])
        return x

    def logits(self, x):
        return self._linear(self._norm(x), self.head)[:, :VOCAB]

    def prompt(self, frames, lengths):
        """frames (sum of lengths, WIDTH): fills the caches, returns the logits after each sequence's last frame."""
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), device=self.dev, dtype=torch.int32)
        self.lens.copy_(cu[1:] - cu[:-1])
        return self.logits(self.forward(frames, cu, int(max(lengths)))[cu[1:].long() - 1])

    def step(self, ids):
        """One token a sequence: ids (seqs,) int32 -> logits (seqs, VOCAB)."""
        self.lens.add_(1)
        return self.logits(self.forward(self.embed[ids.long()], self.one_each, 1))

    def check(self):
        for cache in self.caches:
            cache.check()


def generate(dec: TextDecoder, frames, lengths, tokens: int, temperature=0.8, top_k=50, top_p=0.95, seed=0, graph=True):
    """tokens new tokens for every sequence: (seqs, tokens) ids and log-probabilities."""
    dev, n = dec.dev, dec.seqs
    settings = dict(temperature=torch.full((n,), temperature, device=dev),
                    top_k=torch.full((n,), top_k, device=dev, dtype=torch.int32), top_p=torch.full((n,), top_p, device=dev))
    uniform = torch.rand(tokens, n, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)
    u = torch.empty(n, device=dev)
    ids, logprob = dec.pkg.sample(dec.prompt(frames, lengths), uniform[0], **settings)
    out = [(ids.clone(), logprob.clone())]

    def step():
        return dec.pkg.sample(dec.step(ids), u, **settings)

    captured = None
    for i in range(1, tokens):
        u.copy_(uniform[i])
        if captured is None:
            new = step()                # the first step runs as it is (and does every kernel's set-up)
            if graph and i + 1 < tokens:
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=torch.cuda.current_stream()):
                    result = step()
        else:
            captured.replay()
            new = result
        ids.copy_(new[0])
        out.append((ids.clone(), new[1].clone()))
    dec.check()
    return torch.stack([a for a, _ in out], 1), torch.stack([b for _, b in out], 1)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--utterances", type=int, default=4)
    ap.add_argument("--seconds", type=float, default=30.0)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args()
    pkg = load_package()
    syn = importlib.import_module("bark3_b200.synthetic")
    enc = pkg.Encoder(0)
    enc.load(syn.encoder_weights(seed=7, n_layers=2, layout="lut4"))
    enc.finalize(2)
    rng = np.random.default_rng(1)
    lengths = [pkg.frames_for_seconds(a.seconds * s) for s in rng.uniform(0.4, 1.0, a.utterances)]
    with torch.cuda.stream(torch.cuda.ExternalStream(enc.stream)):
        sub = torch.from_numpy(np.concatenate([syn.sub_features(rng, t) for t in lengths])).cuda()
        frames = enc.encode_batch(sub, np.concatenate([[0], np.cumsum(lengths)]))
        dec = TextDecoder(pkg, enc, a.layers, a.utterances, max(lengths) + a.tokens)
        generate(dec, frames, lengths, 4)      # set-up
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        ids, logprob = generate(dec, frames, lengths, a.tokens)
        t1.record()
        t1.synchronize()
    for i, t in enumerate(lengths):
        print(f"utterance {i}: {t} frames -> {ids[i, :8].tolist()} ..., mean log-probability {logprob[i].mean():.2f}")
    print(f"{a.utterances} prompts and {a.tokens} tokens each in {t0.elapsed_time(t1):.1f} ms")
    enc.close()


if __name__ == "__main__":
    main()
