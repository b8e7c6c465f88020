"""Attention over the 8-bit paged cache, element by element, against the formula in 64 bits.

What an element o = sum_j p_j v_j of a head may be off, apart from its rounding to the output's type: with
R = sqrt(sum_j p_j^2 v_j^2) (errors of single keys are independent) and sg = the largest scale * |q * k_j|_2,
  * a score: q to 22 bits (two fp16 numbers; 24 bits below its largest element over int8 codes) and a sum of D products
    in fp32, 2^-19 sg at most, which moves p_j by that share;
  * exp2, the products with the value's scale and P in two fp16 numbers: 2^-22 of each p_j v_j;
  * sums over the keys in fp32, up to 16 additions one after the other: 2^-19 (R + |o|);
  * P's smallest step, 2^-31 of the head's largest p_j max |v_j| (call it M): n 2^-31 M for n keys.
Together b = 2^-18 ((1 + sg) R + |o|) + n 2^-31 M.  An element is allowed half a last place of its type and 8 b (b is
the size of a sum of many roundings), and the share of elements that are not the exact one's nearest number is allowed
2 b over a last place, in the mean, and five standard deviations of that count."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_q8 import DT, Case, _device_error_clean, cache_of, ops, rotate, run_attention  # noqa: E402,F401

BITS = {"f16": 11, "bf16": 8, "f32": 24}


def last_place(x, dt):
    """The step between numbers of the type at x."""
    _, e = np.frexp(np.abs(x))
    return np.exp2(np.maximum(e - BITS[dt], {"f16": -24, "bf16": -133, "f32": -149}[dt]).astype(np.float64))


def nearest(x, dt):
    step = last_place(x, dt)
    return np.rint(x / step) * step


def exact(c, scale=None, p_bits=None, q_bits=None, drop=None):
    """(o, b), each [T, H, D].  `p_bits` / `q_bits` round P / q to that many bits and `drop` leaves these keys out: the
    mistakes that the bounds have to catch."""
    q = c.q
    if c.cos is not None:
        q = rotate(q, c.cos.double().numpy(), c.sin.double().numpy(), c.pos, c.inter)

    def cut(x, bits):
        m, e = np.frexp(x)
        return np.ldexp(np.rint(m * 2.0 ** bits), e - bits)

    q = q if q_bits is None else cut(q, q_bits)
    G, scale = c.H // c.HK, scale or c.D ** -0.5
    out, b = np.zeros((c.T, c.H, c.D)), np.zeros((c.T, c.H, c.D))
    for i in range(c.T):
        n = int(c.pos[i]) + 1
        k, v = (c.values(w, c.seq[i], n) for w in (0, 1))
        qi = q[i].reshape(c.HK, G, c.D)
        s = np.einsum("hgd,nhd->hgn", qi, k) * scale
        sg = np.sqrt(np.einsum("hgd,nhd->hgn", qi ** 2, k ** 2).max(-1)) * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        if drop is not None:
            p[..., drop[0]:drop[1]] = 0
        if p_bits is not None:
            p = cut(p, p_bits)
        o = np.einsum("hgn,nhd->hgd", p, v)
        r = np.sqrt(np.einsum("hgn,nhd->hgd", p ** 2, v ** 2))
        out[i] = o.reshape(c.H, c.D)
        m = (p * np.abs(v).max(-1).T[:, None]).max(-1)
        b[i] = (2.0 ** -18 * ((1 + sg[..., None]) * r + np.abs(o)) + n * 2.0 ** -31 * m[..., None]).reshape(c.H, c.D)
    return out, b


def excess(got, o, b, dt):
    """(most that an element is off over what it may be, flipped elements over what they may be)"""
    step = last_place(o, dt)
    over = (np.abs(got - o) / (step / 2 + 8 * b + 1e-300)).max()
    few = np.minimum(1.0, 2 * b / step)
    most = few.sum() + 5 * np.sqrt(few.sum()) + 5
    return over, (got != nearest(o, dt)).sum() / most


SHAPES = [
    # H, HK, D, bs, new, past
    (32, 8, 128, 16, [1, 1], [15, 400]),
    (64, 8, 128, 32, [1, 1], [900, 63]),          # groups of 8
    (12, 4, 64, 24, [1, 1], [300, 70]),           # groups of 3, pages of 24
    (8, 8, 32, 16, [1], [200]),
    (32, 2, 64, 16, [1], [130]),                  # 16 heads to a CTA
    (8, 2, 256, 16, [1], [333]),
]


def made(H, HK, D, bs, new, past, dt, code, seed=0, **kw):
    return Case(np.random.default_rng(H * 131 + D + sum(past) + seed), H=H, HK=HK, D=D, bs=bs, new=new, past=past, dt=dt,
                code=code, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_elements(ops, code, dt, shape):
    c = made(*shape, dt, code)
    t = c.cuda()
    got = run_attention(ops, t, c, True).double().cpu().numpy().reshape(c.T, c.H, c.D)
    c.codes = cache_of(t, c)
    o, b = exact(c)
    over, flips = excess(got, o, b, dt)
    assert over <= 1, over
    if dt != "f32":  # (32-bit outputs have no room below their own rounding)
        assert flips <= 1, flips


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_the_bounds_see_mistakes(code, dt, shape):
    """A unit of keys left out, and q or P in 11 bits: on the formula, without a GPU."""
    c = made(*shape, dt, code)
    c.put(c.written())
    o, b = exact(c)
    assert max(excess(nearest(o, dt), o, b, dt)) <= 1
    n = max(c.total)
    for mistake in (dict(drop=(n - 16, n)), dict(q_bits=11), dict(p_bits=11)):
        assert max(excess(nearest(exact(c, **mistake)[0], dt), o, b, dt)) > 1, mistake


def outlier(dt, code, power):
    """One value row 2^power times the others, seen by heads 0 to 3 alone: heads 4 to 7 give its key e^-40 and less."""
    c = Case(np.random.default_rng(power), H=8, HK=1, D=64, bs=16, new=[1], past=[90], dt=dt, code=code, rotary=False)
    at = 37
    page, off = c.bt[0, at // 16], at % 16
    big = np.rint(8 * np.sign(np.random.default_rng(1).standard_normal(64)))
    c.codes[0][0][page, 0, off] = big * (8 if code == "int8" else 16)  # its key: a row of +-64 (+-128) codes
    row = c.values(0, 0, 91 - 1)[at, 0]
    q = c.q.copy()
    for h in range(8):  # scores of +40 and of -60 and less, on top of the others'
        q[0, h] = np.float16(0.25) * q[0, h] + (40.0 if h < 4 else -70.0) * 8 / (row @ row) * row
    c.qkv[:, :8 * 64] = torch.from_numpy(q.reshape(1, -1)).to(DT[dt])
    c.q = c.qkv.double().numpy()[:, :8 * 64].reshape(1, 8, 64)
    c.codes[1][1][page, 0, off] *= 2.0 ** power
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("power", [12, 24, 34])
def test_a_value_scale_that_other_heads_do_not_see(ops, code, dt, power):
    """The heads that give the large row no weight lose no bits to it (and those that do hold it)."""
    c = outlier(dt, code, power)
    t = c.cuda()
    got = run_attention(ops, t, c, True).double().cpu().numpy().reshape(1, 8, 64)
    c.codes = cache_of(t, c)
    o, b = exact(c)
    assert np.abs(o[:, 4:]).max() < 8 < 2.0 ** 12 < np.abs(o[:, :4]).max()
    if dt == "f16":  # (larger than the type's largest number)
        got, o, b = got[:, 4:], o[:, 4:], b[:, 4:]
    over, _ = excess(got, o, b, dt)
    assert over <= 1, over


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,HK,D", [(8, 1, 128), (8, 1, 256), (16, 1, 64), (4, 1, 32), (24, 1, 128)])
def test_elements_of_a_long_sequence(ops, code, dt, H, HK, D):
    """One sequence over every CTA: hundreds of parts a row, more than are joined at a time."""
    c = made(H, HK, D, 16, [1], [20011], dt, code)
    t = c.cuda()
    got = run_attention(ops, t, c, True).double().cpu().numpy().reshape(c.T, c.H, c.D)
    c.codes = cache_of(t, c)
    o, b = exact(c)
    over, _ = excess(got, o, b, dt)
    assert over <= 1, over


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_elements_of_many_new_rows(ops, dt):
    """More new rows of one sequence than a CTA has threads, between two others."""
    c = made(8, 2, 64, 16, [3, 150, 1], [10, 61, 0], dt, "int8")
    t = c.cuda()
    got = run_attention(ops, t, c, True).double().cpu().numpy().reshape(c.T, c.H, c.D)
    c.codes = cache_of(t, c)
    o, b = exact(c)
    over, flips = excess(got, o, b, dt)
    assert over <= 1 and flips <= 1, (over, flips)
