"""Decode over the paged 8-bit cache at the ends of its number range: keys and queries
of opposite extremes, values near bf16's largest."""
import math

import numpy as np
import pytest
import torch

from oracle import cache_oracle as co
from tests._decode_bounds import check
from tests.test_decode_fp8_gpu import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("k_pow,q_pow", [(121, -124), (126, -126), (-105, 110), (100, -90)])
def test_decode_fp8_keys_and_queries_of_opposite_extremes(D, k_pow, q_pow):
    """Scores of ordinary size from keys near the ends of the scale range and queries that make up for them, and
    (100, -90) scores of about 2^10 that one token takes."""
    import blackwell_b200 as bw
    lens, ps = [150, 64], 16
    q, codes, sc, bt = make(lens, 1, 4, D, ps, 351, spread=0)
    rng = np.random.default_rng(1)
    q = (torch.from_numpy(rng.choice([-1.0, 1.0, 1.5], (2, 4, D))) * 2.0 ** q_pow).bfloat16()
    for b, n in enumerate(lens):
        x = rng.uniform(-1.5, 1.5, (n, 1, D)) * 2.0 ** (k_pow if b == 0 else k_pow - 1)
        c, byte = co.quantise_rows(x.astype(np.float32))
        t = np.arange(n)
        codes[0, bt[b, t // ps], t % ps] = c
        sc[bt[b, t // ps], :, 0, t % ps] = byte
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


def test_decode_fp8_orthogonal_keys_at_the_top_of_the_range():
    """Products that are all zero times scales whose product is beyond fp32: scores of 0, not NaN."""
    import blackwell_b200 as bw
    lens = [100]
    q, codes, sc, bt = make(lens, 1, 2, 64, 16, 361, spread=0)
    q[:] = 0
    q[..., 0] = 2.0 ** 100
    codes[0, ..., 0] = 0
    t = np.arange(100)
    sc[bt[0, t // 16], :, 0, t % 16] = 127 + 110
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


def test_decode_fp8_largest_values_one_segment():
    """Values of 1.875 * 2^127: the references of the weights and of the denominator are 2^128 apart (tokens 0..127:
    score 0 and small values, tokens 128..255: score 8 in powers of two, which moves one reference and not the other)."""
    import blackwell_b200 as bw
    lens, ps, D = [256], 16, 128
    q, codes, sc, bt = make(lens, 1, 4, D, ps, 371, spread=0, width_extra=0)
    q[:] = 0
    q[..., 0] = 1.0
    codes[0] = 0
    codes[1] = co.to_e4m3(np.array(240.0))
    t = np.arange(256)
    sc[bt[0, t // ps], :, :, t % ps] = 127
    far = t[128:]
    codes[0, bt[0, far // ps], far % ps, :, 0] = co.to_e4m3(np.array(8.0))
    sc[bt[0, t // ps], :, 1, t % ps] = np.where(t < 128, 127 + 100, 127 + 120)[:, None]
    scale = float(np.float32(math.log(2.0)))
    o, lse = run(q, codes, sc, bt, lens, scale=scale)
    assert bw.stream_status() == 0
    assert torch.all(torch.isfinite(o))
    check(o, lse, q, codes, sc, bt, lens, scale=scale)


@pytest.mark.parametrize("lens,Hkv,width_extra", [([9000], 2, 1), ([40000], 1, 1), ([130] * 600, 1, 40)])
def test_decode_fp8_largest_values_joined(lens, Hkv, width_extra):
    """Parts of a sequence whose values are all about 1.5 * 2^127: their weighted sum is beyond fp32, their mean is not."""
    import blackwell_b200 as bw
    q, codes, sc, bt = make(lens, Hkv, 4, 128, 64, 381, spread=0, width_extra=width_extra)
    own = sc == 120
    codes[1] = np.where(own[:, :, 1].transpose(0, 2, 1)[..., None], (codes[1] & 7) | co.to_e4m3(np.array(128.0)), codes[1])
    own[:, :, 0] = False
    sc[own] = 127 + 120
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    assert torch.all(torch.isfinite(o))
    check(o, lse, q, codes, sc, bt, lens)
