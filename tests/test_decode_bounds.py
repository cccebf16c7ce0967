"""The bounds the decode over the 8-bit cache is held to are tight enough to see what
could go wrong in a split: mistakes planted in the oracle's result exceed them."""
import math

import numpy as np
import pytest

from oracle import cache_oracle as co
from tests._decode_bounds import expected, gather, marked
from tests.test_decode_fp8_gpu import make


def _case(n, D, flat):
    q, codes, sc, bt = make([n], 1, 4, D, 64, 701 + D)
    if flat:
        marked(codes, sc, bt, [n])
    _, k, _ = gather(codes, sc, bt, 0, n, 0)
    vc, v, ev = gather(codes, sc, bt, 0, n, 1)
    return q[0].double().numpy(), k, v, vc, ev, 1 / math.sqrt(D)


def _outside(o, lse, wo, wl, tol_o, tol_l):
    return bool(np.any(np.abs(o - wo) > tol_o)) or bool(np.any(np.abs(lse - wl) > tol_l))


@pytest.mark.parametrize("n,D,tile", [(9000, 128, 128), (20000, 128, 128), (12000, 64, 256)])
@pytest.mark.parametrize("flat", [True, False])
def test_planted_mistakes_exceed_the_bounds(n, D, tile, flat):
    q, k, v, vc, ev, scale = _case(n, D, flat)
    wo, wl, tol_o, tol_l = expected(q, k, v, vc, ev, scale)
    assert not _outside(wo, wl, wo, wl, tol_o, tol_l)
    assert np.any(np.abs(0.01 * wo) > tol_o)                                        # O one per cent off
    t0 = 3 * tile
    left = np.r_[0:t0, t0 + tile:n]
    assert _outside(*co.decode(q, k[left], v[left], scale)[:2], wo, wl, tol_o, tol_l)        # a tile lost
    twice = np.r_[0:n, t0:t0 + tile]
    assert _outside(*co.decode(q, k[twice], v[twice], scale)[:2], wo, wl, tol_o, tol_l)      # a tile taken twice
    if flat:
        for mistake in ("no values", "another tile's values"):
            bad = v.copy()
            bad[t0:t0 + tile] = 0 if mistake == "no values" else v[0:tile]
            assert np.any(np.abs(co.decode(q, k, bad, scale)[0] - wo) > tol_o), mistake
        # a sequence's last segment merged with half its weight
        a, b = co.decode(q, k[:t0], v[:t0], scale), co.decode(q, k[t0:], v[t0:], scale)
        w = 0.5 * np.exp(a[1] - wl)[:, None]
        assert np.any(np.abs((w * a[0] + (1 - w) * b[0]) - wo) > tol_o)
