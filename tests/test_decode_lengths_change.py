"""Decode over the 8-bit cache while the caller changes kv_lens (an error: the results
mean nothing then).  The kernel must stay inside the tables and come to an end, and
later calls must be right."""
import numpy as np
import pytest
import torch

from tests._decode_bounds import check
from tests.test_decode_fp8_gpu import make


@pytest.mark.parametrize("kTile", [128, 256])
@pytest.mark.parametrize("clamped", [True, False])
def test_segments_of_lengths_that_change(kTile, clamped):
    """The segment rule of decode_fp8.cu restated: the tiles come from one reading of the lengths, the length of a
    segment from another.  Clamped to the last of its tiles, every segment has tokens, is inside the table and has the
    same number of tiles for any reading; without the clamp there are segments that end at or before token 0, whose last
    page would be in front of the table."""
    rng = np.random.default_rng(kTile)
    most, bad = 1500, 0
    for _ in range(300):
        B = int(rng.integers(1, 9))
        first = rng.integers(0, most + 1, B)
        tiles = (first + kTile - 1) // kTile
        prefix = np.concatenate([[0], np.cumsum(tiles)]).astype(int)
        total, groups = int(prefix[-1]), int(rng.integers(1, 40))
        per = max((total + groups - 1) // groups, 1)
        for g in range(groups):
            t0, t1 = min(g * per, total), min(g * per + per, total)
            while t0 < t1:
                b = int(np.searchsorted(prefix[:-1], t0, side="right")) - 1
                end = min(t1, prefix[b + 1])
                assert end > t0
                n_tiles = []
                for again in rng.integers(0, most + 1, 3):            # three warps read the length
                    n = int(prefix[b + 1] - prefix[b])
                    length = min(max(int(again), (n - 1) * kTile + 1), n * kTile) if clamped else int(again)
                    tok0, tok1 = (t0 - prefix[b]) * kTile, min((end - prefix[b]) * kTile, length)
                    bad += tok1 <= tok0
                    if clamped:
                        assert 0 <= tok0 < tok1 <= most
                    n_tiles.append(len(range(tok0, tok1, kTile)))
                bad += len(set(n_tiles)) > 1
                t0 = end
    assert (bad == 0) == clamped


@pytest.mark.gpu
@pytest.mark.parametrize("D,width_extra", [(64, 0), (64, 60), (128, 0), (128, 60)])
def test_lengths_that_change_under_the_call(D, width_extra):
    """Lengths overwritten on another stream while decodes run: every call ends without an error of the device, and
    the calls after it are right."""
    import blackwell_b200 as bw
    F8 = torch.float8_e4m3fn
    lens = [200, 0, 17, 230, 1, 128] * 20
    q, codes, sc, bt = make(lens, 2, 4, D, 16, 401, width_extra=width_extra)
    bt = np.clip(bt, 0, codes.shape[1] - 1)                           # any length within the table has pages
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    kc, vc, s, t, qd = cu(codes[0]).view(F8), cu(codes[1]).view(F8), cu(sc), cu(bt), q.cuda()
    good = torch.tensor(lens, dtype=torch.int32).cuda()
    others = [torch.randint(-5, 300, (len(lens),), generator=torch.Generator().manual_seed(i)).int().cuda() for i in range(8)]
    live = good.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(200):
        bw.gqa_decode_paged_fp8(qd, kc, vc, s, t, live)
        with torch.cuda.stream(side):
            for j in range(4):
                live.copy_(others[(i + j) % 8])
    torch.cuda.synchronize()
    assert bw.stream_status() == 0
    o, lse = bw.gqa_decode_paged_fp8(qd, kc, vc, s, t, good)
    assert bw.stream_status() == 0
    some = list(range(12))
    check(o[some], lse[some], q[some], codes, sc, bt[some], [lens[i] for i in some])
