"""What ``rope`` refuses under gradients, without a GPU."""
import pytest
import torch

import blackwell_b200 as bw


def test_rope_refuses_outputs_and_tables_that_gradients_would_miss():
    x, tab = torch.zeros(3, 2, 16), torch.zeros(8, 16)
    w = x.clone().requires_grad_()
    for call in (lambda: bw.rope(w, None, tab, q_out=torch.zeros_like(x)),
                 lambda: bw.rope(x, w, tab, k_out=torch.zeros_like(x)),
                 lambda: bw.rope(x, None, tab, q_out=w),
                 lambda: bw.rope(w, None, tab, q_out=w),
                 lambda: bw.rope(x, None, tab.clone().requires_grad_())):
        with pytest.raises(ValueError, match="gradient"):
            call()
    # without gradients the calls come as far as the check of the device
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        bw.rope(w, None, tab, q_out=torch.zeros_like(x))
    with pytest.raises(ValueError, match="CUDA"):
        bw.rope(w, None, tab)
