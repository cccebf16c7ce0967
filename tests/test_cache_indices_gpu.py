"""Indices of the cache calls at the ends of their types: skipped and reported, and
the other sequences are done."""
import pytest
import torch

from tests._util import seeded_bf16
from tests.test_cache_gpu import make_cache, raw

pytestmark = pytest.mark.gpu
TOP = (1 << 63) - 1


@pytest.mark.parametrize("fp8", [True, False])
def test_read_offsets_whose_end_passes_64_bits(fp8):
    """An offset of 2^63 - 1 plus a length is negative in 64 bits: such a span is outside the output."""
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    kc, vc, sc = make_cache(4, 16, 2, 64, fp8, fill=0x38)            # e4m3 1.0 times 2^(7 - 127)
    bt = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [0, 1]], dtype=torch.int32).cuda()
    lens = torch.tensor([20, 1, 32, 5, 7], dtype=torch.int32).cuda()
    offs = torch.tensor([TOP, TOP, TOP - 31, 1 << 62, 3]).cuda()
    ko = torch.full((10, 2, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    bw.kv_cache_read(kc, vc, bt, lens, offs, scales=sc, k_out=ko, v_out=vo)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    one = 2.0 ** -120 if fp8 else 3.0
    assert torch.all(ko[3:] == one) and torch.all(vo[3:] == one) and torch.all(ko[:3] == 9) and torch.all(vo[:3] == 9)


def test_read_starts_and_lengths_at_the_ends_of_32_bits():
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    kc, vc, sc = make_cache(4, 16, 1, 128, False)
    top = (1 << 31) - 1
    bt = torch.tensor([[0, 1]] * 5, dtype=torch.int32).cuda()
    lens = torch.tensor([top, 1, top, -top - 1, 4], dtype=torch.int32).cuda()
    starts = torch.tensor([top, top, -top - 1, top, 28], dtype=torch.int32).cuda()
    offs = torch.tensor([0, 0, 0, 0, 1]).cuda()
    ko = torch.full((6, 1, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    bw.kv_cache_read(kc, vc, bt, lens, offs, kv_starts=starts, k_out=ko, v_out=vo)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    for t in (ko, vo):
        assert torch.all(t[1:5] == 3) and torch.all(t[0] == 9) and torch.all(t[5] == 9)


def test_write_slots_and_positions_at_the_ends_of_their_types():
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    kc, vc, sc = make_cache(2, 8, 1, 64, True)
    before = raw(kc).copy()
    k = seeded_bf16((5, 1, 64), 1).cuda()
    tab = bw.rope_table(4, 64)
    slots = torch.tensor([TOP, -TOP - 1, 1 << 32, 16, 3]).cuda()
    pos = torch.tensor([0, 0, 0, 0, (1 << 31) - 1], dtype=torch.int32).cuda()
    bw.kv_cache_write(k, k, kc, vc, slots, scales=sc, cos_sin_cache=tab, positions=pos)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    now = raw(kc)
    assert (now[0, 3] != before[0, 3]).any() and (now[0, 3] == raw(vc)[0, 3]).all()   # a position outside the table: as it is
    now[0, 3] = before[0, 3]
    assert (now == before).all()


def test_rope_positions_and_offsets_at_the_ends_of_32_bits():
    """Position plus offset is formed in 64 bits: none wraps into the table."""
    import blackwell_b200 as bw
    top = (1 << 31) - 1
    tab = bw.rope_table(8, 16)
    x = torch.randn(4, 2, 16, device="cuda")
    for pos, off in (([top, -top - 1, 1, 2], top), ([top, -top - 1, -1, -2], -top - 1)):
        y = bw.rope(x, None, tab, positions=torch.tensor(pos, dtype=torch.int32).cuda(), pos_offset=off)[0]
        for t in range(4):
            p = pos[t] + off
            want = bw.rope(x[t:t + 1], None, tab, pos_offset=p)[0][0] if 0 <= p < 8 else x[t]
            assert torch.equal(y[t], want)
