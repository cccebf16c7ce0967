"""Bounded waits of the decode over the 8-bit cache that run out in the middle of
things: runs longer than the ring of stages, several segments a block, runs that fit
the ring.  A test hook withholds the first K tile of every block."""
import contextlib

import pytest

from tests._decode_bounds import check
from tests.test_decode_fp8_gpu import make, run

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def withheld(ns):
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    old = bw.get_option(_ffi.BW_OPT_TIMEOUT_NS)
    try:
        bw.set_option(_ffi.BW_OPT_TIMEOUT_NS, ns)
        bw.set_option(_ffi.BW_OPT_DEBUG_FLAGS, 1)
        yield
    finally:
        bw.set_option(_ffi.BW_OPT_DEBUG_FLAGS, 0)
        bw.set_option(_ffi.BW_OPT_TIMEOUT_NS, old)


@pytest.mark.parametrize("D,Hkv,lens,width_extra", [
    # 9 groups, 12 to 13 tiles a run (7 of 256): producers are refused a stage; cut sequences, several segments a block
    (128, 32, [3000, 600, 0, 1500, 2222, 700, 1999, 3, 2900], 1),
    (64, 32, [3000, 600, 0, 1500, 2222, 700, 1999, 3, 2900], 1),
    # tables of two tiles: no sequence is cut, many short segments a block
    (128, 32, [250, 1, 0, 130, 128, 17] * 12, 0),
    (64, 32, [500, 1, 0, 300, 256, 17] * 12, 0),
    # one to three tiles a run: they fit the ring, and the producers leave while copies are under way
    (128, 4, [3000, 0, 700], 1),
    (64, 16, [3000, 2500, 0, 700], 1),
])
def test_waits_that_run_out_unwind(D, Hkv, lens, width_extra):
    """The calls report BW_ERR_TIMEOUT, end, and the calls after them are right, several times in turn (a block that
    left copies under way would write into the next call's shared memory)."""
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    q, codes, sc, bt = make(lens, Hkv, 2, D, 16, 501, width_extra=width_extra)
    for ns in (5_000_000, 1_000_000, 200_000):
        with withheld(ns):
            run(q, codes, sc, bt, lens)
            assert bw.stream_status() == _ffi.BW_ERR_TIMEOUT
        o, lse = run(q, codes, sc, bt, lens)
        assert bw.stream_status() == 0
    some = list(range(min(len(lens), 9)))
    check(o[some], lse[some], q[some], codes, sc, bt[some], [lens[i] for i in some])
