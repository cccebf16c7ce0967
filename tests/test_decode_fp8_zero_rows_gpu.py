"""Decode over the paged 8-bit cache where some value rows are all zeros (padding or
sink tokens): the other rows carry the output and keep their relative weights."""
import math

import numpy as np
import pytest
import torch

from oracle import cache_oracle as co
from tests._decode_bounds import check
from tests.test_decode_fp8_gpu import make, run

pytestmark = pytest.mark.gpu


def _raise_logit(codes, sc, bt, q, b, t, head, over):
    """Token t's key of `head` becomes a multiple of the group's first query row that lifts its logit to about `over`."""
    ps, D = codes.shape[2], codes.shape[4]
    G = q.shape[1] // codes.shape[3]
    row = q[b, head * G].double().numpy()
    want = row * (over * math.sqrt(D) / (row @ row))
    c, byte = co.quantise_rows(want[None].astype(np.float32))
    codes[0, bt[b, t // ps], t % ps, head] = c[0]
    sc[bt[b, t // ps], head, 0, t % ps] = byte[0]


def _zero_value(codes, sc, bt, b, t, head):
    """A row of zeros as bw_kv_cache_write stores it: codes 0, scale byte 127."""
    ps = codes.shape[2]
    codes[1, bt[b, t // ps], t % ps, head] = 0
    sc[bt[b, t // ps], head, 1, t % ps] = 127


@pytest.mark.parametrize("G,Hkv,D,ps,lens", [
    (4, 2, 128, 16, [4096, 200]), (12, 1, 128, 64, [700, 90]), (8, 2, 64, 16, [3000, 250]), (16, 2, 64, 8, [130, 600]),
])
@pytest.mark.parametrize("over", [10.0, 14.0])
def test_decode_fp8_row_of_zeros_in_v(G, Hkv, D, ps, lens, over):
    """A token that takes the softmax's weight and has no value (a sink): the other tokens carry the output and keep
    their relative weights.  First, middle and last tokens, and a warp's worth of them side by side."""
    import blackwell_b200 as bw
    q, codes, sc, bt = make(lens, Hkv, G, D, ps, 300 + G + D, spread=1)
    for b, n in enumerate(lens):
        for head in range(Hkv):
            for t in [0, n // 2, n - 1] if head == 0 else range(n // 3, n // 3 + 18):
                _raise_logit(codes, sc, bt, q, b, t, head, over)
                _zero_value(codes, sc, bt, b, t, head)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


def test_decode_fp8_only_zeros_and_few_values():
    """A sequence whose values are all zeros gives zeros; one with a single value row among zeros gives that row's."""
    import blackwell_b200 as bw
    lens = [300, 300, 17]
    q, codes, sc, bt = make(lens, 1, 4, 128, 16, 331)
    for b, n in enumerate(lens):
        for t in range(n):
            if not (b == 1 and t == 211):
                _zero_value(codes, sc, bt, b, t, 0)
    sc[bt[1, 211 // 16], 0, 1, 211 % 16] = 127 - 40
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)
    assert torch.all(o[0] == 0) and torch.all(o[2] == 0) and torch.any(o[1] != 0)


def test_decode_fp8_nan_in_a_row_of_zeros():
    """A row that holds one NaN and zeros (scale byte 127): its column is NaN, the other columns are as exact as with
    a row of zeros."""
    lens = [400]
    q, codes, sc, bt = make(lens, 1, 4, 64, 16, 341, spread=1)
    _raise_logit(codes, sc, bt, q, 0, 100, 0, 12.0)
    _zero_value(codes, sc, bt, 0, 100, 0)
    clean, lse0 = run(q, codes, sc, bt, lens)
    check(clean, lse0, q, codes, sc, bt, lens)
    codes[1, bt[0, 100 // 16], 100 % 16, 0, 9] = 0x7f
    o, lse = run(q, codes, sc, bt, lens)
    assert torch.all(torch.isnan(o[0, :, 9])) and torch.equal(lse, lse0)
    keep = [d for d in range(64) if d != 9]
    assert torch.equal(o[..., keep], clean[..., keep])
