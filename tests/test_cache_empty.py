"""Empty batches through the rotary and cache calls: nothing to do is no error, and
nothing is left unwritten without one."""
import pytest
import torch

import blackwell_b200 as bw


def test_rope_refuses_keys_beside_no_queries():
    """k_out would be left as it was allocated."""
    tab = torch.zeros(4, 64)
    for q, k in ((torch.zeros(3, 0, 64), torch.zeros(3, 2, 64)), (torch.zeros(2, 0, 5, 64), torch.zeros(2, 1, 5, 64))):
        with pytest.raises(ValueError, match="no heads"):
            bw.rope(q.bfloat16(), k.bfloat16(), tab)


@pytest.mark.gpu
def test_an_empty_step():
    """Rotation, write, read-back and decode of a step without sequences."""
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    kc = z(2, 8, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc, tab, none = z(2, 2, 2, 8, dtype=torch.uint8), bw.rope_table(4, 64), z(0, dtype=torch.int32)
    q, k = bw.rope(z(0, 8, 64), z(0, 2, 64), tab, positions=none)
    assert q.shape == (0, 8, 64) and k.shape == (0, 2, 64)
    bw.kv_cache_write(k, k, kc, kc, z(0, dtype=torch.int64), scales=sc, cos_sin_cache=tab, positions=none)
    for kw in ({}, dict(workspace=z(0, dtype=torch.uint8)), dict(out=q, lse=z(0, 8, dtype=torch.float32))):
        o, lse = bw.gqa_decode_paged_fp8(q, kc, kc, sc, z(0, 3, dtype=torch.int32), none, **kw)
        assert o.shape == (0, 8, 64) and lse.shape == (0, 8)
    # keys without heads beside queries: the queries alone
    x = torch.randn(3, 2, 64, device="cuda").bfloat16()
    y, none_out = bw.rope(x, x[:, :0], tab)
    assert torch.equal(y, bw.rope(x, None, tab)[0]) and none_out.shape == (3, 0, 64)
    assert bw.stream_status() == 0
