"""The oracles of the routing and of the 8-bit blocks, pinned on the CPU: the
routing's gradient against differences, e4m3 against torch's conversion, the
reference's softmax router as a special case."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import ops_oracle as O


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_against_differences(score, renorm):
    rng = np.random.default_rng(0)
    l = rng.normal(size=(3, 12))
    l[1, 4] = -np.inf
    kw = dict(score=score, renormalize=renorm, scale=1.7)
    inds, gates = O.route(l, 4, **kw)
    dg = rng.normal(size=gates.shape)
    got = O.route_backward(l, inds, gates, dg, **kw)
    h = 1e-6
    for r in range(3):
        for e in range(12):
            if not np.isfinite(l[r, e]):
                assert got[r, e] == 0
                continue
            d = []
            for sgn in (1, -1):
                m = l.copy()
                m[r, e] += sgn * h
                i2, g2 = O.route(m, 4, **kw)
                assert (i2 == inds).all()
                d.append((g2 * dg).sum())
            # (central differences in 64 bits: h² of the third derivative, and 2^-52 / h)
            assert abs((d[0] - d[1]) / (2 * h) - got[r, e]) < 1e-8


def test_route_equals_softmax_over_the_selected():
    rng = np.random.default_rng(1)
    l = rng.normal(size=(5, 8))
    inds, gates = O.route(l, 2)
    for r in range(5):
        top = np.argsort(-l[r], kind="stable")[:2]
        assert (inds[r] == top).all()
        w = np.exp(l[r, top] - l[r, top].max())
        np.testing.assert_allclose(gates[r], w / w.sum(), rtol=1e-14)


def test_route_of_rows_with_nothing_left():
    l = np.full((2, 8), -np.inf)
    l[1, 5] = 0.0
    inds, gates = O.route(l, 3, score="sigmoid", n_groups=2, top_groups=1, group_score="top2")
    assert inds.tolist() == [[0, 1, 2], [5, 4, 6]]
    assert gates.tolist() == [[0, 0, 0], [1, 0, 0]]


def test_e4m3_is_torchs():
    v = np.concatenate([np.linspace(-448, 448, 20011), np.linspace(-0.1, 0.1, 20011), [2.0 ** -10, 3 * 2.0 ** -10]])
    v = v.astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert (O.e4m3(v) == want).all()


def test_block_rounding_is_within_half_a_step():
    rng = np.random.default_rng(2)
    x = (rng.normal(size=(7, 300)) * np.exp(rng.normal(size=(7, 1)) * 20)).astype(np.float32)
    got = O.held_rows(*O.quantize_rows(x))
    a = np.stack([np.abs(x[:, i:i + 128]).max(1) for i in (0, 128, 256)], 1).repeat(128, 1)[:, :300]
    # e4m3's half step: 2^-4 of a value, 2^-10 where its exponent is the least; a few fp32 roundings
    tol = np.maximum(np.abs(x) * 2.0 ** -4, a / 448 * 2.0 ** -10) * (1 + 2.0 ** -18)
    assert (np.abs(got - x) <= tol).all()
