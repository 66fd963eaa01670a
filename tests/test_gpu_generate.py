"""examples/generate.py: the cached decode step against prompts that hold the same tokens.

The hidden state after step i has to be what a fresh prompt of all tokens up
to i gives: the same keys and values go through the cache one by one and in one
call.  The stored codes can differ only where a page's scale grew after a
value was rounded below e4m3's normal range (2^-6 of a scale that fits the
page's largest value to 448), at most 2^-9 of the scale: 2^-17 of the largest value
in the page.  Sums run in another order (f32) and the linears round activations
to f16 (2^-11) in both, of values that differ by as little; through 3 layers
the logits, sums of 640 products of unit size, stay within 2^-7 of their largest.
"""
import importlib.util
import pathlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("generate_example", ROOT / "examples" / "generate.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_steps_match_prompts(pkg, example):
    enc = pkg.Encoder(0)
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(enc.stream)):
            lengths, steps = [75, 1, 40], 12
            g = torch.Generator(device="cuda").manual_seed(3)
            frames = torch.randn(sum(lengths), example.WIDTH, generator=g, device="cuda")
            a = example.TextDecoder(pkg, enc, 3, len(lengths), 128)
            b = example.TextDecoder(pkg, enc, 3, len(lengths), 128)
            logits = a.prompt(frames, lengths)
            parts = list(frames.split(lengths))
            for _ in range(steps):
                ids = logits.argmax(-1).to(torch.int32)
                logits = a.step(ids)
                parts = [torch.cat([p, a.embed[i:i + 1]]) for p, i in zip(parts, ids.tolist())]
                want = b.prompt(torch.cat(parts), [p.shape[0] for p in parts])
                d = (logits - want).abs().max().item()
                assert d <= 2.0 ** -7 * want.abs().max().item()
            a.check(), b.check()
    finally:
        enc.close()


def test_graph_and_eager_steps_agree(pkg, example):
    enc = pkg.Encoder(0)
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(enc.stream)):
            lengths = [33, 70]
            frames = torch.randn(sum(lengths), example.WIDTH, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
            runs = []
            for graph in (True, False):
                dec = example.TextDecoder(pkg, enc, 2, 2, 128)
                runs.append(example.generate(dec, frames, lengths, 20, graph=graph))
            assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
            assert (runs[0][0] >= 0).all() and (runs[0][0] < example.VOCAB).all() and (runs[0][1] <= 0).all()
    finally:
        enc.close()
