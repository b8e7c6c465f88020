"""The example decoder over the 8-bit paged cache: prompt in chunks, decode steps and sampling together.

The logits of a decode step are compared with those of the same weights when the whole text is given as one prompt (its
attention then sees unquantised rows of the last chunk).  The codes' rounding is 1 / 254 (int8) or 1 / 32 (e4m3) of a row's
largest value at most, uniformly distributed: about 0.3 % and 2.6 % of a value's size; two layers of residual stream keep
the logits' relative error within a few of those: 3 % and 15 % of their norm."""

from __future__ import annotations

import os
import sys

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_paged_q8

    return decode_paged_q8


def _cfg(example):
    return example.DecoderConfig(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=2000, max_seq=512)


@pytest.mark.parametrize("code,limit", [("int8", 0.03), ("e4m3", 0.15)])
def test_decode_matches_one_prompt(example, code, limit):
    cfg = _cfg(example)
    g = torch.Generator(device="cuda").manual_seed(0)
    text = torch.randint(0, cfg.vocab, (2, 90), device="cuda", generator=g)
    whole = example.PagedQ8Decoder(cfg, 2, 128, code=code)
    want = torch.stack([whole.prompt(b, text[b], chunk=128) for b in range(2)]).float()
    model = example.PagedQ8Decoder(cfg, 2, 128, code=code)
    for b in range(2):
        model.prompt(b, text[b, :80 - 7 * b], chunk=33)  # uneven lengths, several chunks
    logits = torch.empty_like(want)
    for t in range(17):  # sequence 0 is done after 10 of them
        at = (model.past.long()).clamp(max=89)
        out = model.step(text[torch.arange(2), at.cpu()]).float()
        for b in range(2):
            if int(model.past[b]) == 90:
                logits[b] = out[b]
    err = (logits - want).norm(dim=1) / want.norm(dim=1)
    assert (err < limit).all(), err


def test_generate_is_reproducible_and_greedy_at_zero(example):
    cfg = _cfg(example)
    prompts = torch.randint(0, cfg.vocab, (3, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    runs = [example.generate(example.PagedQ8Decoder(cfg, 3, 64), prompts, 8, seed=5) for _ in range(2)]
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert runs[0][0].shape == (3, 8) and (runs[0][0] >= 0).all() and (runs[0][1] <= 0).all()
    model = example.PagedQ8Decoder(cfg, 3, 64)
    ids, _ = example.generate(model, prompts, 1, temperature=0.0)
    again = example.PagedQ8Decoder(cfg, 3, 64)
    logits = torch.stack([again.prompt(b, prompts[b]) for b in range(3)])
    assert torch.equal(ids[:, 0], logits.float().argmax(1))
