"""The oracle of the paged 4-bit cache, pinned by closed forms (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged as orc


def test_rotation_closed_forms():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 3, 2, 16))
    f = [0.7, 0.1, 0.01]
    pos = np.array([[0, 1, 5], [7, -3, 1000]])
    for inter in (False, True):
        y = orc.rotate(x, pos, f, interleaved=inter)
        assert np.allclose(y[0, 0], x[0, 0])                       # position 0
        assert np.array_equal(y[..., 6:], x[..., 6:])              # the rest of the head
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
        assert np.allclose(orc.rotate(y, pos, f, interleaved=inter, inverse=True), x)
    # scores depend on the distance of two positions alone
    q, k = rng.standard_normal((1, 1, 1, 8)), rng.standard_normal((1, 1, 1, 8))
    dots = [float((orc.rotate(q, [[p]], f) * orc.rotate(k, [[p - 4]], f)).sum())
            for p in (4, 90, 3000)]
    assert np.allclose(dots, dots[0])


@pytest.mark.parametrize("value,held", [(0.25, 0.0), (0.2500001, 0.5), (0.75, 1.0), (1.25, 1.0),
                                        (1.75, 2.0), (2.5, 2.0), (3.5, 4.0), (5.0, 4.0),
                                        (5.0000001, 6.0), (7.9, 6.0), (-3.5, -4.0)])
def test_nearest_code(value, held):
    # beside a 4, the block's power of two is 1
    x = np.zeros(32)
    x[0], x[5] = 4.0, value
    assert orc.stored(x, True)[5] == held


def test_block_scales():
    x = np.zeros((1, 64))
    x[0, 0], x[0, 40] = 96.0, 3.0 / 1024
    y = orc.stored(x, False)
    assert y[0, 0] == 96.0 and y[0, 40] == 3.0 / 1024     # 6 * 16, 6 / 2048: a block each
    x[0, 1] = np.inf
    assert np.isfinite(orc.stored(x, True)).all() and orc.stored(x, True)[0, 1] == 6 * 2.0 ** 13
    x[0, 1] = np.nan
    assert orc.stored(x, True)[0, 1] == 0.0


def test_attend_against_a_dense_softmax():
    rng = np.random.default_rng(1)
    m = orc.PagedModel(5, 16, 2, 32, False)
    table = np.array([[3, 1], [4, 9]])                    # 9: no page
    k, v = rng.standard_normal((2, 20, 2, 32)), rng.standard_normal((2, 20, 2, 32))
    m.store(k, v, table, [0, 0])
    q = rng.standard_normal((2, 3, 4, 32))
    out, lse, *_ = orc.attend(q, m, table, [20, 20])
    ks, vs = orc.stored(k, False), orc.stored(v, False)
    for b, keys in ((0, 20), (1, 16)):
        for i in range(3):
            for h in range(4):
                n = min(18 + i, keys)
                s = ks[b, :n, h // 2] @ q[b, i, h] / np.sqrt(32)
                p = np.exp(s)
                assert np.allclose(out[b, i, h], p @ vs[b, :n, h // 2] / p.sum())
                assert np.isclose(lse[b, h, i], np.log(p.sum()))
    out, lse, *_ = orc.attend(q, m, table, [2, 0])
    assert (out[0, 0] == 0).all() and np.isinf(lse[0, :, 0]).all() and np.isinf(lse[1]).all()
    assert np.isfinite(lse[0, :, 1:]).all()
