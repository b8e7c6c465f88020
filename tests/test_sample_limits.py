"""Token sampling at the ends of its filters' ranges, against the definition in 64 bits (tokens equal, as in
test_sample.py)."""

from __future__ import annotations

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
