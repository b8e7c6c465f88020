"""Token sampling at the ends of its filters' ranges, against the definition in 64 bits (tokens equal, as in
test_sample.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_sample import DT, check, inputs, ops  # noqa: E402,F401

TINY = [1e-45, 1e-39, 4.2e-39, 1e-38, 1e-30]  # (1.44 / T is beyond fp32 for the first three)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (50, 0.9, 0.1),
                                   (0, 1.0, 0.05), (0, 0.0, 1.0), (900, 0.5, 0.0)])
def test_temperatures_near_zero(ops, dt, k, p, m):
    """The largest logit is taken, and where several are equal the race decides between them."""
    B = 2 * len(TINY)
    x, e = inputs(B, 3001, dt, 11)
    x[1::2, 100:2000:90] = 20.0
    t = [TINY[b // 2] for b in range(B)]
    tok = check(ops, x, e, t, [k] * B, [p] * B, [m] * B)
    assert all(x[b, int(tok[b])] == x[b].max() for b in range(B))
    if k == 0 and p == 1.0:  # all 22 of the equal ones race
        assert len(set(tok[1::2].tolist())) > 1


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [7, 3001, 50257])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.25, 0.0), (600, 0.5, 0.0), (0, 1.0, 1.0)])
@pytest.mark.parametrize("scale", [2.5, 2500.0])
def test_infinite_temperature(ops, dt, V, k, p, m, scale):
    """All logits above -infinity weigh the same: of the first k in order, the first p of them, then the least noise."""
    x, e = inputs(4, V, dt, V, scale)
    x[1, ::2] = -math.inf
    x[2, 1:] = -math.inf
    f = [torch.full((4,), v, dtype=d, device="cuda") for v, d in (
        (math.inf, torch.float32), (k, torch.int32), (p, torch.float32), (m, torch.float32))]
    tok, _ = ops.sample(x, e, *f)
    for b in range(4):
        xb, eb = x[b].double().cpu().numpy(), e[b].cpu().numpy()
        order = np.argsort(-xb, kind="stable")
        order = order[xb[order] > -math.inf][:k or V]
        if p < 1:  # (equal weights: exact sums, but for the border itself)
            order = order[:max(1, math.ceil(p * order.size))]
        assert int(tok[b]) == np.sort(order)[np.argmin(eb[np.sort(order)])]
