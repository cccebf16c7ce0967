"""Head counts of ``bw_rope`` at the limit of a launch: more are refused as a shape,
before anything touches the device (the launch itself would fail)."""
import pytest
import torch

from blackwell_b200 import _ffi

P = 0x100000


@pytest.mark.parametrize("Hq,Hkv", [(65536, 65536), (65536, 65535), (65535, 65536), (65537, 0)])
def test_rope_refuses_more_head_groups_than_a_grid_has(Hq, Hkv):
    k = P if Hkv else None
    rc = _ffi.lib().bw_rope(P, P, k, k, 0, 1, Hq, Hkv, 1, 64, None, None, None, None, P, 10, 64, P, 0, 0, 0, None)
    assert rc == _ffi.BW_ERR_SHAPE


@pytest.mark.gpu
def test_rope_of_the_most_heads():
    import blackwell_b200 as bw
    tab = bw.rope_table(4, 16)
    q, k = torch.randn(2, 65536, 16, device="cuda"), torch.randn(2, 65534, 16, device="cuda")
    pos = torch.tensor([1, 3], dtype=torch.int32).cuda()
    qo, ko = bw.rope(q, k, tab, positions=pos)
    assert bw.stream_status() == 0
    assert torch.equal(qo[:, :65534], bw.rope(q[:, :65534], None, tab, positions=pos)[0])
    assert torch.equal(ko, bw.rope(k, None, tab, positions=pos)[0])
    assert torch.equal(qo[:, -9:], bw.rope(q[:, -9:].contiguous(), None, tab, positions=pos)[0])
