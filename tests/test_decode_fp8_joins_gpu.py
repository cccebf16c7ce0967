"""The joins of the decode over the 8-bit cache, each at both head dimensions, held to
bounds that see a lost, doubled or misplaced tile (tests/test_decode_bounds.py)."""
import numpy as np
import pytest

from tests._decode_bounds import check, marked
from tests.test_decode_fp8_gpu import make, run

pytestmark = pytest.mark.gpu


def _run(lens, Hkv, G, D, ps, seed, flat, width_extra, some=None):
    import blackwell_b200 as bw
    q, codes, sc, bt = make(lens, Hkv, G, D, ps, seed, width_extra=width_extra)
    if flat:
        marked(codes, sc, bt, lens)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    some = list(range(len(lens))) if some is None else some
    check(o[some], lse[some], q[some], codes, sc, bt[some], [lens[i] for i in some])


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,Hkv,G", [([9000], 2, 4), ([20000], 1, 16), ([12345, 9000], 1, 3), ([40000], 8, 1)])
def test_wide_join(lens, Hkv, G, D, flat):
    """Few long sequences, a table of more than 32 tiles (heads of 64: 8192 tokens)."""
    _run(lens, Hkv, G, D, 64, 801, flat, 140)


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_join_of_many_rows(D, flat):
    """2048 rows and more of cut sequences: a warp a row; heads of 64 have two segments side by side."""
    lens = [int(n) for n in np.random.default_rng(D).integers(0, 1500, 128)]
    lens[:4] = [0, 4000, 1, 2500]
    _run(lens, 2, 8, D, 16, 811, flat, 40, list(range(0, 128, 5)) + [1, 2, 3])


@pytest.mark.parametrize("D", [64, 128])
def test_join_of_many_rows_with_more_than_32_segments(D):
    """One long sequence among many of one token: its segments take several rounds of a warp."""
    lens = [3] * 128
    lens[77] = 60000
    _run(lens, 1, 16, D, 64, 821, True, 1, [0, 76, 77, 78, 127])


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,Hkv,G", [([517], 8, 4), ([3000, 0, 700, 1], 2, 9), ([1] * 9 + [5000, 4999], 4, 2)])
def test_small_join(lens, Hkv, G, D, flat):
    _run(lens, Hkv, G, D, 16, 831, flat, 1)


@pytest.mark.parametrize("B,D", [(700, 64), (700, 128), (4096, 64)])
def test_many_short_sequences_with_a_wide_table(B, D):
    """As a server's table is: of fixed width, whatever the sequences have."""
    lens = [int(n) for n in np.random.default_rng(B).integers(0, 90, B)]
    _run(lens, 1, 4, D, 16, 841, False, 40, list(range(0, B, B // 25)) + [B - 1])


@pytest.mark.parametrize("D", [64, 128])
def test_many_kv_heads_with_a_wide_table(D):
    _run([700, 3], 700, 1, D, 8, 851, False, 100)
