"""Decode over a bf16 cache whose pages held something else before: what lies behind
a sequence's end, infinities and NaN included, does not reach its output."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as orc
from tests._util import LSE_TOL, O_TOL, seeded_bf16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.0])
@pytest.mark.parametrize("ps,D,G", [(8, 64, 4), (16, 128, 8), (64, 128, 1), (256, 64, 16), (32, 128, 12)])
def test_paged_decode_over_recycled_pages(ps, D, G, bad):
    """Every row that no sequence owns (the rest of last pages, free pages) holds `bad`."""
    import blackwell_b200 as bw
    rng = np.random.default_rng(ps + D)
    Hkv = 2
    lens = [1, 63, 64, 65, 130, 0, 1025, ps + 3]
    need = [(n + ps - 1) // ps for n in lens]
    pages = sum(need) + 3
    perm = rng.permutation(pages)
    bt = -np.ones((len(lens), max(need) + 1), np.int32)
    kc = torch.full((pages, ps, Hkv, D), bad, dtype=torch.bfloat16)
    vc = torch.full((pages, ps, Hkv, D), bad, dtype=torch.bfloat16)
    at, rows = 0, []
    for b, n in enumerate(lens):
        bt[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        k, v = seeded_bf16((n, Hkv, D), 2 * b), seeded_bf16((n, Hkv, D), 2 * b + 1)
        kc[bt[b, t // ps], t % ps], vc[bt[b, t // ps], t % ps] = k, v
        rows.append((k, v))
    q = seeded_bf16((len(lens), Hkv * G, D), 77)
    o, lse = bw.gqa_decode_paged(q.cuda(), kc.cuda(), vc.cuda(), torch.from_numpy(bt).cuda(),
                                 torch.tensor(lens, dtype=torch.int32).cuda(), chunk=128)
    assert bw.stream_status() == 0
    offs = np.concatenate([[0], np.cumsum(lens)[:-1]])
    some = [b for b, n in enumerate(lens) if n]
    ro, rl = orc.decode_reference(q[some].float(), torch.cat([r[0] for r in rows]).float(), torch.cat([r[1] for r in rows]).float(),
                                  np.array(lens)[some], offs[some], 1 / math.sqrt(D))
    assert np.abs(o[some].float().cpu().numpy() - ro).max() <= O_TOL
    assert np.abs(lse[some].cpu().numpy() - rl).max() <= LSE_TOL
    assert torch.all(o[5] == 0) and torch.all(torch.isneginf(lse[5]))


def test_packed_decode_beside_a_neighbour_of_nan():
    """Sequences of one packed tensor: the next one's values are not this one's business."""
    import blackwell_b200 as bw
    lens, Hkv, G, D = [37, 200, 64], 2, 4, 128
    offs = np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.int64)
    q, k, v = seeded_bf16((3, Hkv * G, D), 1), seeded_bf16((sum(lens), Hkv, D), 2), seeded_bf16((sum(lens), Hkv, D), 3)
    v[37:237] = float("nan")
    o, lse = bw.gqa_decode(q.cuda(), k.cuda(), v.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.from_numpy(offs).cuda())
    assert bw.stream_status() == 0
    assert torch.all(torch.isnan(o[1]))
    ok = [0, 2]
    v[37:237] = 0
    ro, rl = orc.decode_reference(q[ok].float(), k.float(), v.float(), np.array(lens)[ok], offs[ok], 1 / math.sqrt(D))
    assert np.abs(o[ok].float().cpu().numpy() - ro).max() <= O_TOL
    assert np.abs(lse[ok].cpu().numpy() - rl).max() <= LSE_TOL
