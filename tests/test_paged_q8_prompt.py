"""A prompt taken in chunks over the 8-bit paged cache, and a decode step after it, against attention in 64 bits.

Per chunk: the past is read back (fp16), GroupQueryAttention appends the chunk's rows there and attends, and the rows are
quantised into the pages.  The values that the cache stands for are exact in the comparison (they are read from it); the
chunk's own rows are rotated here and rounded to fp16 by GroupQueryAttention, one place of the row's largest element.

GroupQueryAttention holds q, the new keys and P in 11 bits: with R and sg as in test_paged_q8_precision.py a score is off
by 2^-10 sg and an element by b = 2^-10 ((1 + sg) R + |o|); an element is allowed half a last place and 4 b.  The decode
step has the bounds of that file."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_q8 import Case, _device_error_clean, cache_of, ops, rotate, run_attention  # noqa: E402,F401
from test_paged_q8_precision import exact, last_place, excess  # noqa: E402

H, HK, D, S = 8, 2, 64, 51
CHUNKS = ((0, 7), (7, 8), (8, 40), (40, 50))


def attend(q, k, v):
    """(o, b) of rows q [n, H, D] that see keys 0 .. len(k) - n + i: k, v [t, HK, D] in 64 bits."""
    n, t = len(q), len(k)
    o, b = np.zeros((n, H, D)), np.zeros((n, H, D))
    for i in range(n):
        seen = t - n + i + 1
        qi = q[i].reshape(HK, H // HK, D)
        s = np.einsum("hgd,nhd->hgn", qi, k[:seen]) * D ** -0.5
        sg = np.sqrt(np.einsum("hgd,nhd->hgn", qi ** 2, k[:seen] ** 2).max(-1)) * D ** -0.5
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        o[i] = np.einsum("hgn,nhd->hgd", p, v[:seen]).reshape(H, D)
        r = np.sqrt(np.einsum("hgn,nhd->hgd", p ** 2, v[:seen] ** 2))
        b[i] = 2.0 ** -10 * ((1 + sg[..., None]) * r + np.abs(o[i].reshape(r.shape))).reshape(H, D)
    return o, b


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_prompt_in_chunks_and_a_decode_step(ops, code):
    c = Case(np.random.default_rng(17), H=H, HK=HK, D=D, bs=16, new=[S], past=[0], dt="f16", code=code)
    t = c.cuda()
    pages = [t[n] for n in ("kc", "vc", "ks", "vs")]
    i32 = dict(dtype=torch.int32, device="cuda")
    cos, sin = (x.double().numpy() for x in (c.cos, c.sin))
    q, k = (rotate(x, cos, sin, c.pos, 0) for x in (c.q, c.k))
    qkv = c.qkv.cuda()
    for lo, hi in CHUNKS:
        before, rows, last = torch.tensor([lo], **i32), torch.tensor([0, hi - lo], **i32), torch.tensor([hi - 1], **i32)
        keys, values = ops.paged_kv_dequantize(*pages, before, t["bt"], cap=hi)
        past = [x[0, :, :lo].double().cpu().numpy().transpose(1, 0, 2) for x in (keys, values)]
        c.codes = cache_of(t, c)
        for which in (0, 1):  # what the pages stand for, rounded to fp16
            np.testing.assert_array_equal(past[which], c.values(which, 0, lo).astype(np.float16).astype(np.float64))
        out = ops.group_query_attention(qkv[lo:hi][None], None, None, keys, values, last, t["cos"], t["sin"],
                                        num_heads=H, kv_heads=HK)[0]
        ops.paged_kv_quantize(t["k"][lo:hi], t["v"][lo:hi], *pages, rows, before, t["bt"], t["cos"], t["sin"])
        new = keys[0, :, lo:hi].double().cpu().numpy().transpose(1, 0, 2)
        assert (np.abs(new - k[lo:hi]) <= np.abs(k[lo:hi]).max(-1, keepdims=True) * 2.0 ** -10).all()
        o, b = attend(q[lo:hi], np.concatenate([past[0], k[lo:hi]]), np.concatenate([past[1], c.v[lo:hi]]))
        got = out.double().cpu().numpy().reshape(hi - lo, H, D)
        over = (np.abs(got - o) / (last_place(o, "f16") / 2 + 4 * b)).max()
        assert over <= 1, (lo, hi, over)
    got = ops.paged_attention_quantized(t["q"][50:], t["k"][50:], t["v"][50:], *pages, torch.tensor([0, 1], **i32),
                                        torch.tensor([50], **i32), t["bt"], t["cos"], t["sin"], num_heads=H, kv_heads=HK)
    c.codes = cache_of(t, c)
    o, b = exact(c)
    over, _ = excess(got.double().cpu().numpy().reshape(1, H, D), o[50:], b[50:], "f16")
    assert over <= 1, over


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_the_bounds_see_a_chunk_that_is_lost(code):
    """On the formula: keys of the chunk before that are left out, or not quantised, exceed the bounds."""
    c = Case(np.random.default_rng(17), H=H, HK=HK, D=D, bs=16, new=[S], past=[0], dt="f16", code=code)
    cos, sin = (x.double().numpy() for x in (c.cos, c.sin))
    q, k = (rotate(x, cos, sin, c.pos, 0) for x in (c.q, c.k))
    c.put(c.written())
    kq, vq = (np.concatenate([c.values(w, 0, 40), x[40:50]]) for w, x in ((0, k), (1, c.v)))
    o, b = attend(q[40:50], kq, vq)
    step = last_place(o, "f16")
    for kk, vv in ((np.delete(kq, slice(8, 24), 0), np.delete(vq, slice(8, 24), 0)), (k[:50], c.v[:50])):
        wrong, _ = attend(q[40:50], kk, vv)
        assert (np.abs(wrong - o) / (step / 2 + 4 * b)).max() > 1
