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
