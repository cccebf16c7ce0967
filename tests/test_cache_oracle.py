"""The cache oracle against independent statements of the same things (CPU):
torch's e4m3 cast, a search for the row's exponent, torch softmax in fp64; and
the decode's split of the token tiles, restated."""
import math

import numpy as np
import pytest
import torch

from oracle import cache_oracle as co


def test_e4m3_values_and_rounding_match_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(co.e4m3_values(), want)
    y = np.random.default_rng(0).standard_normal(20000) * 2.0 ** np.random.default_rng(1).integers(-12, 8, 20000)
    y = np.clip(y.astype(np.float32), -448, 448)
    y[:4] = [0.0, -0.0, 448.0, -448.0]
    got = co.to_e4m3(y)
    np.testing.assert_array_equal(got, torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    # every midpoint between neighbours goes to the even code
    v = co.e4m3_values()[:127]
    mid = co.to_e4m3((v[:-1] + v[1:]) / 2)
    np.testing.assert_array_equal(mid % 2, 0)


@pytest.mark.parametrize("power", [-140, -120, -101, -91, -10, 0, 7, 100, 127])
def test_row_exponent_is_the_smallest(power):
    rng = np.random.default_rng(abs(power))
    x = (rng.uniform(-1, 1, (50, 16)) * 2.0 ** power).astype(np.float32)
    x[0] = 0
    x[1, 3], x[2, 5] = np.nan, np.inf
    x[3, :] = np.float32(1.75 * 2.0 ** power)          # exactly 448 * 2^e
    x[4, :] = np.nextafter(x[3, 0], np.float32(np.inf))
    codes, byte = co.quantise_rows(x)
    for r in range(50):
        top = max([abs(float(t)) for t in x[r] if np.isfinite(t)])
        e = int(byte[r]) - 127
        if top == 0:
            assert e == 0
            continue
        assert top <= 448.0 * 2.0 ** e or e == 120
        assert top > 448.0 * 2.0 ** (e - 1) or e == -100
    back = co.cache_values(codes, byte)
    fine = np.isfinite(x)
    assert np.all(np.isnan(back[~fine]))
    # half a step of e4m3: 2^-4 of the value, or half of the smallest step 2^-9 2^e
    step = np.maximum(np.abs(x.astype(np.float64)) * 2.0 ** -4, (2.0 ** (byte.astype(float) - 127 - 10))[:, None])
    assert np.all(np.abs(back - x)[fine] <= step[fine])


def test_decode_oracle_matches_torch():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((6, 64)), rng.standard_normal((37, 2, 64)), rng.standard_normal((37, 2, 64))
    o, lse, mean_abs, size = co.decode(q, k, v, 0.125)
    t = lambda a: torch.from_numpy(a)  # noqa: E731
    x = torch.einsum("hd,lhd->hl", t(q), t(k).repeat_interleave(3, 1)) * 0.125
    np.testing.assert_allclose(lse, torch.logsumexp(x, -1).numpy(), rtol=1e-12)
    np.testing.assert_allclose(o, torch.einsum("hl,lhd->hd", x.softmax(-1), t(v).repeat_interleave(3, 1)).numpy(),
                               rtol=1e-10, atol=1e-14)
    assert np.all(mean_abs >= np.abs(o)) and np.all(size >= np.abs(x.numpy()).max(-1) - 1e-12)


def test_table_matches_plain_formula():
    t = co.table(5, 7, 16)
    for p in range(5, 12):
        for i in range(8):
            a = p * 10000.0 ** (-i / 8)
            assert abs(t[p - 5, i] - math.cos(a)) < 1e-14 and abs(t[p - 5, 8 + i] - math.sin(a)) < 1e-14


@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("Hkv,blocks", [(1, 296), (8, 296), (12, 444), (16, 1024), (700, 296)])
def test_decode_split_covers_every_tile_once(Hkv, blocks, tile):
    """Segments of the decode (decode_fp8.cu: equal runs of tiles, whole tiles of a
    sequence): every tile belongs to one segment, a segment's partial index (group +
    sequence) is its own and within (groups + B), and the join's range of groups is
    the segments'."""
    rng = np.random.default_rng(Hkv)
    groups = max(blocks // Hkv, 1)
    for lens in ([0], [1], [517], [64, 0, 65, 0, 0, 4096], list(rng.integers(0, 9000, 70)), [131072], [0, 0]):
        tiles = [(n + tile - 1) // tile for n in lens]
        prefix = np.concatenate([[0], np.cumsum(tiles)]).astype(int)
        total = prefix[-1]
        per = max((total + groups - 1) // groups, 1)
        seen, parts, by_seq = set(), set(), {}
        for g in range(groups):
            t0, t1 = min(g * per, total), min(g * per + per, total)
            while t0 < t1:
                b = int(np.searchsorted(prefix[:-1], t0, side="right")) - 1
                end = min(t1, prefix[b + 1])
                assert end > t0
                for t in range(t0, end):
                    assert t not in seen
                    seen.add(t)
                assert g + b not in parts and g + b < groups + len(lens)
                parts.add(g + b)
                by_seq.setdefault(b, []).append(g)
                t0 = end
        assert len(seen) == total
        for b, gs in by_seq.items():
            assert gs == list(range(prefix[b] // per, (prefix[b + 1] - 1) // per + 1))


@pytest.mark.parametrize("groups", [1, 4, 37, 74, 296])
def test_decode_runs_of_whole_sequences(groups):
    """Short tables: a run begins and ends with a sequence, so every sequence with
    tokens is in exactly one run, whole."""
    rng = np.random.default_rng(groups)
    for tiles in ([1], [0], [2, 0, 1, 2, 2, 0], list(rng.integers(0, 5, 300)), [0, 0, 4], [4] * 40):
        prefix = np.concatenate([[0], np.cumsum(tiles)]).astype(int)
        total, B = prefix[-1], len(tiles)
        per = max((total + groups - 1) // groups, 1)
        start = lambda t: prefix[np.searchsorted(prefix, t)]   # noqa: E731
        seen = []
        for g in range(groups):
            t0, t1 = start(min(g * per, total)), start(min(g * per + per, total))
            while t0 < t1:
                b = int(np.searchsorted(prefix[:-1], t0, side="right")) - 1
                assert prefix[b] == t0 and prefix[b + 1] <= t1
                seen.append(b)
                t0 = prefix[b + 1]
        assert seen == [b for b in range(B) if tiles[b]]
        # the sequences without tokens, by groups
        assert sorted(b for g in range(groups) for b in range(g, B, groups) if not tiles[b]) == \
            [b for b in range(B) if not tiles[b]]
