"""Token sampling against the definition in 64 bits, row by row.

Tokens are compared for equality.  The draw is a race of w_j / noise_j, so a rounding of 2^-22 in w decides a row only
where the two best quotients lie that close; a row whose two best differ by less than 1e-5 (or whose filters have a
token within 1e-5 of their border) is allowed either of the two outcomes.  logprob: fp32 sums of at most 2^18 terms,
1e-5 of 1 + |logprob|."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from onnxruntime_ep_b200 import ops as _ops

    return _ops


def race(x, e, t, k, p, m, slack=0.0):
    """(token, how near another outcome is) of one row in 64 bits; `slack` moves the borders of top-p and min-p."""
    V = x.size
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, math.inf
    if t <= 0:
        return int(order[0]), math.inf
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    k = V if k <= 0 or k > V else k
    order = order[:k]
    ws = w[order]
    keep = np.ones(k, bool)
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        keep = before < p * ws.sum() * (1 + slack)
        keep[0] = True
    keep &= (ws >= min(m, 1.0) * (1 - slack)) & (x[order] > -np.inf)
    kept = np.sort(order[keep])
    key = w[kept] / e[kept]
    best = int(np.argmax(key))
    rest = np.delete(key, best)
    gap = math.inf if not rest.size or key[best] == 0 else 1 - rest.max() / key[best]
    return int(kept[best]), gap


def check(ops, x, e, t=None, k=None, p=None, m=None, xs=None, es=None):
    """x, e: cuda tensors; xs / es: what is passed instead (strided forms of the same)."""
    B, V = x.shape
    dev = dict(device="cuda")
    args = [None if a is None else torch.tensor(a, dtype=d, **dev)
            for a, d in ((t, torch.float32), (k, torch.int32), (p, torch.float32), (m, torch.float32))]
    tok, lp = ops.sample(x if xs is None else xs, e if es is None else es, *args)
    tok2, lp2 = ops.sample(x, e, *args)
    assert torch.equal(tok, tok2) and torch.equal(lp, lp2)  # equal inputs, equal tokens
    xh, eh = x.double().cpu().numpy(), e.double().cpu().numpy()
    tok, lp = tok.cpu().numpy(), lp.double().cpu().numpy()
    near = 0
    for b in range(B):
        a = [1.0 if t is None else float(np.float32(t[b])), 0 if k is None else k[b],
             1.0 if p is None else float(np.float32(p[b])), 0.0 if m is None else float(np.float32(m[b]))]
        want, gap = race(xh[b], eh[b], *a)
        if tok[b] != want:
            other = {race(xh[b], eh[b], *a, slack=s)[0] for s in (1e-5, -1e-5)}
            assert gap < 1e-5 or tok[b] in other, (b, tok[b], want, gap, a)
            near += 1
        if tok[b] < 0:
            assert lp[b] == -math.inf
            continue
        xb = np.where(np.isnan(xh[b]), -np.inf, xh[b])
        with np.errstate(invalid="ignore"):
            z = np.log(np.where(xb == xb.max(), 1.0, np.exp(xb - xb.max())).sum())
            ref = (0.0 if xb[tok[b]] == xb.max() else xb[tok[b]] - xb.max()) - z
        assert ref == lp[b] or abs(lp[b] - ref) <= 1e-5 * (1 + abs(ref)), (b, lp[b], ref)
    assert near <= 1 + B // 50
    return tok


def inputs(B, V, dt, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(B, V, device="cuda", generator=g) * scale).to(DT[dt])
    e = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_(min=1e-10)
    return x, e


FILTERS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.05),
           (1.0, 200, 0.8, 0.02), (0.7, 40, 1.0, 0.0), (0.6, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (2.0, 0, 1.0, 1.0),
           (0.3, 10 ** 6, 0.5, 0.5), (5.0, 777, 0.999, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (12, 7), (24, 1000), (1, 128256), (12, 50257), (48, 32000),
                                 (160, 4099), (2, 262144)])
def test_filters(ops, dt, B, V):
    """Every filter, over vocabularies from one token to the largest, odd ones among them."""
    x, e = inputs(B, V, dt, V + B)
    f = [FILTERS[(b + V) % len(FILTERS)] for b in range(B)]
    check(ops, x, e, *(list(c) for c in zip(*f)))


@pytest.mark.gpu
@pytest.mark.parametrize("B,V", [(3, 33), (2, 70001)])
def test_no_filters(ops, B, V):
    x, e = inputs(B, V, "f32", 1)
    check(ops, x, e)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("V", [5, 4096, 40000])
def test_equal_logits(ops, dt, V):
    """All logits equal (and two values only): ties are cut by index, exactly."""
    x, e = inputs(6, V, dt, 9)
    x[:3] = 1.25
    x[3:] = (x[3:] > 0).to(x.dtype)
    ks = [3, 0, 0, V // 2, 0, 5]
    ps = [1.0, 0.5, 0.0, 1.0, 0.75, 0.4]
    tok = check(ops, x, e, [1.0] * 6, ks, ps, [0.0] * 6)
    assert tok[0] < 3 and tok[1] <= V // 2 and tok[2] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_masked_logits(ops, dt):
    """-inf, NaN, +inf and the type's lowest value among the logits; rows with nothing left."""
    V = 3001
    x, e = inputs(8, V, dt, 4)
    low = torch.finfo(DT[dt]).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 1234] = -5.0
    x[3, ::2] = -math.inf
    x[3, 1::4] = math.nan
    x[4] = low
    x[4, 77] = 0
    x[5] = low
    x[6, 10] = x[6, 2000] = math.inf
    x[7, :3000] = -math.inf
    n = 8
    for t, k, p, m in FILTERS[:6]:
        tok = check(ops, x, e, [t] * n, [k] * n, [p] * n, [m] * n)
        assert tok[0] == tok[1] == -1 and tok[2] == 1234 and tok[4] == 77 and tok[6] in (10, 2000) and tok[7] == 3000


@pytest.mark.gpu
def test_zeros_of_both_signs_are_one_value(ops):
    x = torch.zeros(1, 64, device="cuda")
    x[0, ::2] = -0.0
    e = torch.ones(1, 64, device="cuda")
    e[0, 40] = 0.5
    assert ops.sample(x, e, top_k=torch.tensor([41], dtype=torch.int32, device="cuda"))[0].item() == 40
    assert ops.sample(x, e, top_k=torch.tensor([40], dtype=torch.int32, device="cuda"))[0].item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_strides_and_alignment(ops, dt):
    """Rows that are slices of wider ones, at addresses that are not 16-byte aligned."""
    wide, ew = inputs(9, 5003, dt, 3)
    for off, V in ((0, 5000), (1, 4999), (3, 1777), (5, 6)):
        xs, es = wide[:, off:off + V], ew[:, off:off + V]
        check(ops, xs.contiguous(), es.contiguous(), [0.9] * 9, [20] * 9, [0.9] * 9, None, xs=xs, es=es)


@pytest.mark.gpu
def test_draws_follow_the_distribution(ops):
    """Frequencies of many draws against the kept tokens' probabilities: a chi-square of 7 degrees of freedom
    stays below 40 (its probability of not doing so is 1e-6; the noise is seeded)."""
    V, B = 50, 20000
    g = torch.Generator(device="cuda").manual_seed(0)
    row = torch.randn(V, device="cuda", generator=g)
    x = row.expand(B, V).contiguous()
    e = torch.empty(B, V, device="cuda").exponential_(generator=g)
    k = torch.full((B,), 8, dtype=torch.int32, device="cuda")
    t = torch.full((B,), 0.9, device="cuda")
    tok, _ = ops.sample(x, e, t, k)
    top = row.topk(8)
    p = torch.softmax(top.values.double() / 0.9, 0).cpu().numpy()
    n = np.array([(tok == i).sum().item() for i in top.indices])
    assert n.sum() == B
    assert ((n - B * p) ** 2 / (B * p)).sum() < 40


@pytest.mark.gpu
def test_side_stream_and_given_outputs(ops):
    x, e = inputs(4, 32000, "f16", 8)
    k = torch.full((4,), 30, dtype=torch.int32, device="cuda")
    want = ops.sample(x, e, top_k=k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ids = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
        lp = torch.zeros(4, device="cuda")
        ops.sample(x, e, top_k=k, tokens=ids, logprobs=lp)
    s.synchronize()
    assert torch.equal(ids[:, 0], want[0]) and torch.equal(lp, want[1])


def test_no_rows(ops):
    assert ops._lib().b200ep_sample(*([None] * 8), 0, 10, 0, 0, 1, None) == 0


@pytest.mark.parametrize("kw,match", [
    (dict(noise=torch.ones(2, 9)), "both be"),
    (dict(noise=torch.ones(2, 8, dtype=torch.float16)), "float32"),
    (dict(logits=torch.zeros(2, 16)[:, ::2]), "contiguous"),
    (dict(temperature=torch.ones(3)), "temperature"),
    (dict(top_k=torch.ones(2)), "top_k"),
    (dict(top_p=torch.ones(2, dtype=torch.float64)), "top_p"),
    (dict(min_p=torch.ones(4)[::2]), "min_p"),
    (dict(tokens=torch.zeros(2, dtype=torch.int32)), "tokens"),
    (dict(logprobs=torch.zeros(3)), "logprobs"),
])
def test_refusals_of_the_binding(ops, kw, match):
    a = dict(logits=torch.zeros(2, 8), noise=torch.ones(2, 8))
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        ops.sample(a.pop("logits"), a.pop("noise"), **a)


def test_refusals_of_the_entry_point(ops):
    import ctypes

    L = ops._lib()
    one = ctypes.c_void_p(16)
    for rows, vocab, ls, ns, dtype, word in ((1, 0, 0, 0, 1, "vocab"), (1, 262145, 0, 0, 1, "vocab"),
                                             (-1, 5, 0, 0, 1, "rows"), (1, 5, 4, 0, 1, "strides"),
                                             (1, 5, 0, 4, 1, "strides"), (1, 5, 0, 0, 7, "dtype")):
        assert L.b200ep_sample(*([one] * 8), rows, vocab, ls, ns, dtype, None) == 1
        assert word in L.b200ep_last_error().decode()
    assert L.b200ep_sample(None, *([one] * 7), 1, 5, 0, 0, 1, None) == 1
