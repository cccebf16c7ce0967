"""Writes into the paged cache and reads back, bit for bit against the oracle."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as co
from tests._util import seeded_bf16

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def make_cache(pages, ps, Hkv, D, fp8, fill=0x55):
    if fp8:
        kc = torch.full((pages, ps, Hkv, D), fill, dtype=torch.uint8, device="cuda")
        return kc.view(F8), kc.clone().view(F8), torch.full((pages, Hkv, 2, ps), 7, dtype=torch.uint8, device="cuda")
    kc = torch.full((pages, ps, Hkv, D), 3.0, dtype=torch.bfloat16, device="cuda")
    return kc, kc.clone(), None


def raw(t):
    return t.view(torch.uint8 if t.dtype == F8 else torch.int16).cpu().numpy()


def expect_write(cache, sc, which, x32, slots, ps):
    """The oracle's cache after the write of fp32 rows x32 [T, Hkv, D]."""
    c = raw(cache).copy()
    s = sc.cpu().numpy().copy() if sc is not None else None
    if sc is None:
        bits = torch.from_numpy(x32).bfloat16().view(torch.int16).numpy()
    else:
        bits, byte = co.quantise_rows(x32)
    for t, slot in enumerate(slots):
        if 0 <= slot < c.shape[0] * ps:
            c[slot // ps, slot % ps] = bits[t]
            if sc is not None:
                s[slot // ps, :, which, slot % ps] = byte[t]
    return c, s


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("ps,Hkv,D,T,R,interleaved", [
    (16, 8, 128, 64, 128, False), (8, 1, 64, 1, 64, True), (64, 3, 64, 37, 16, False), (256, 2, 128, 300, 48, True),
    (128, 5, 128, 19, 0, False),
])
def test_write(ps, Hkv, D, T, R, interleaved, fp8):
    """Rotated and plain K, padding slots, positions outside the table, rows of other
    slots untouched; K and V as strided slices of one projection."""
    import blackwell_b200 as bw
    rng = np.random.default_rng(T + R)
    pages = (T + 40) // ps + 3
    kv = seeded_bf16((T, 2 * Hkv * D), 1)
    kv[:, ::7] *= 30.0
    kv = kv.cuda()
    k, v = kv[:, :Hkv * D].view(T, Hkv, D), kv[:, Hkv * D:].view(T, Hkv, D)
    slots = rng.permutation(pages * ps)[:T].astype(np.int64)
    if T > 3:
        slots[2] = -1
    pos = rng.integers(-2, 60, T).astype(np.int32)
    tab = co.table(0, 50, R).astype(np.float32) if R else None
    kc, vc, sc = make_cache(pages, ps, Hkv, D, fp8)
    x = k.float().cpu().numpy()
    if R:
        x = np.asarray(co.rotate(x.transpose(1, 0, 2), pos, tab, interleaved, dtype=np.float32)).transpose(1, 0, 2)
    want_k, s1 = expect_write(kc, sc, 0, x, slots, ps)
    want_v, _ = expect_write(vc, sc, 1, v.float().cpu().numpy(), slots, ps)
    rot = dict(cos_sin_cache=torch.from_numpy(tab).cuda(), positions=torch.from_numpy(pos).cuda()) if R else {}
    bw.kv_cache_write(k, v, kc, vc, torch.from_numpy(slots).cuda(), scales=sc, interleaved=interleaved, **rot)
    assert bw.stream_status() == 0
    np.testing.assert_array_equal(raw(kc), want_k)
    np.testing.assert_array_equal(raw(vc), want_v)
    if fp8:
        want_s = s1
        _, byte = co.quantise_rows(v.float().cpu().numpy())
        for t, slot in enumerate(slots):
            if slot >= 0:
                want_s[slot // ps, :, 1, slot % ps] = byte[t]
        np.testing.assert_array_equal(sc.cpu().numpy(), want_s)


def test_write_rows_at_the_edges_of_the_range():
    """Rows of zeros, subnormals, bf16's largest, exactly 448 * 2^e and just above,
    infinities and NaN among finite elements."""
    import blackwell_b200 as bw
    D = 64
    rows = torch.zeros(10, 1, D)
    rows[1, 0, 3] = 2.0 ** -133
    rows[2] = torch.randn(D, generator=torch.Generator().manual_seed(0)) * 2.0 ** -110
    rows[3] = torch.finfo(torch.bfloat16).max
    rows[4, 0, :5] = torch.tensor([448.0, -448.0, 1.0, 2.0 ** -7, -0.0])
    rows[5, 0, :2] = torch.tensor([450.0, 1.0])
    rows[6, 0, :4] = torch.tensor([float("inf"), 2.0, float("nan"), -float("inf")])
    rows[7] = float("nan")
    rows[8] = 1.75 * 2.0 ** -92                       # smallest rows above the lowest scale
    rows[9] = torch.arange(D) * 0.37
    rows = rows.bfloat16()
    kc, vc, sc = make_cache(2, 8, 1, D, True)
    slots = torch.arange(10).cuda()
    bw.kv_cache_write(rows.cuda(), rows.flip(0).cuda(), kc, vc, slots, scales=sc)
    assert bw.stream_status() == 0
    for which, cache, x in ((0, kc, rows), (1, vc, rows.flip(0))):
        codes, byte = co.quantise_rows(x.float().numpy())
        got = raw(cache).reshape(-1, 1, D)[:10]
        np.testing.assert_array_equal(got & 127, codes & 127)
        np.testing.assert_array_equal(np.where((got & 127) == 127, 0, got), np.where((codes & 127) == 127, 0, codes))
        np.testing.assert_array_equal(sc.cpu().numpy()[:, 0, which].reshape(-1)[:10], byte[:, 0])


def _paged(lens, ps, extra, seed):
    rng = np.random.default_rng(seed)
    need = [(n + ps - 1) // ps for n in lens]
    pages = sum(need) + extra
    perm = rng.permutation(pages)
    width = max(max(need), 1) + 2
    bt = -np.ones((len(lens), width), np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at:at + n]
        at += n
    return bt, pages


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("ps,Hkv,D,lens,starts", [
    (16, 8, 128, [100, 0, 1, 33], None), (8, 1, 64, [7], [0]), (64, 3, 64, [130, 65, 64], [1, 64, 0]),
    (256, 2, 128, [300, 900], [299, 17]), (16, 4, 128, [5000], [1234]),
])
def test_read(ps, Hkv, D, lens, starts, fp8):
    """Spans of sequences into given rows: values exact, other rows as they were."""
    import blackwell_b200 as bw
    rng = np.random.default_rng(ps)
    bt, pages = _paged(lens, ps, 3, 5)
    st = np.zeros(len(lens), int) if starts is None else np.array(starts)
    n = np.array(lens) - st                                   # tokens to read
    kc, vc, sc = make_cache(pages, ps, Hkv, D, fp8)
    if fp8:
        kc.view(torch.uint8).random_(0, 256)
        vc.view(torch.uint8).random_(0, 256)
        sc.random_(60, 200)
        val = [co.cache_values(raw(c), sc.cpu().numpy()[:, :, w].transpose(0, 2, 1)) for w, c in enumerate((kc, vc))]
    else:
        kc.normal_()
        vc.normal_()
        val = [c.float().cpu().numpy() for c in (kc, vc)]
    gaps = np.array([3, 0, 5, 1, 2])[:len(lens)]              # rows between the spans
    offs = np.cumsum(n + gaps) - n
    total = int((n + gaps).sum()) + 4
    ko = torch.full((total, Hkv, D), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = torch.full((total, Hkv, D), 9.0, dtype=torch.bfloat16, device="cuda")
    cu = lambda a, t: torch.from_numpy(np.asarray(a)).to(t).cuda()  # noqa: E731
    bw.kv_cache_read(kc, vc, cu(bt, torch.int32), cu(n, torch.int32), cu(offs, torch.int64), scales=sc,
                     kv_starts=None if starts is None else cu(st, torch.int32), k_out=ko, v_out=vo)
    assert bw.stream_status() == 0
    for out, x in ((ko, val[0]), (vo, val[1])):
        want = np.full((total, Hkv, D), 9.0)
        for b in range(len(lens)):
            t = np.arange(st[b], lens[b])
            want[offs[b]:offs[b] + n[b]] = x[bt[b, t // ps], t % ps]
        want = torch.from_numpy(want).bfloat16().float().numpy()
        np.testing.assert_array_equal(out.float().cpu().numpy(), want)


def test_indices_out_of_range_are_skipped_and_reported():
    """Slots, spans and pages outside their range: that token or span is skipped, the
    others are done, and the stream's status says so once."""
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    ps, Hkv, D, pages = 16, 2, 64, 4
    kc, vc, sc = make_cache(pages, ps, Hkv, D, True)
    k = seeded_bf16((4, Hkv, D), 1).cuda()
    slots = torch.tensor([5, pages * ps, 1 << 40, 9]).cuda()
    want, _ = expect_write(kc, sc, 0, k.float().cpu().numpy(), slots.cpu().numpy(), ps)
    bw.kv_cache_write(k, k, kc, vc, slots, scales=sc)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    assert bw.stream_status() == 0
    np.testing.assert_array_equal(raw(kc), want)
    bt = torch.tensor([[0, 99], [1, -5], [2, 3], [0, 1], [0, 1]], dtype=torch.int32).cuda()
    lens = torch.tensor([20, 17, 32, 33, 4], dtype=torch.int32).cuda()      # 33: beyond the table
    offs = torch.tensor([0, 20, 40, 80, 199]).cuda()                        # 199 + 4: beyond the output
    ko = torch.full((200, Hkv, D), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    bw.kv_cache_read(kc, vc, bt, lens, offs, scales=sc, k_out=ko, v_out=vo)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    val = co.cache_values(raw(kc), sc.cpu().numpy()[:, :, 0].transpose(0, 2, 1))
    want = np.full((200, Hkv, D), 9.0)
    want[0:16], want[20:36] = val[0], val[1]
    want[40:72] = np.concatenate([val[2], val[3]])
    np.testing.assert_array_equal(ko.float().cpu().numpy(), torch.from_numpy(want).bfloat16().float().numpy())


def test_empty_calls():
    import blackwell_b200 as bw
    kc, vc, sc = make_cache(2, 8, 1, 64, True)
    before = raw(kc).copy()
    none = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    bw.kv_cache_write(none, none, kc, vc, torch.empty(0, dtype=torch.int64, device="cuda"), scales=sc)
    ko, vo = bw.kv_cache_read(kc, vc, torch.zeros(0, 3, dtype=torch.int32, device="cuda"),
                              torch.zeros(0, dtype=torch.int32, device="cuda"),
                              torch.zeros(0, dtype=torch.int64, device="cuda"), scales=sc, total_rows=0)
    assert ko.shape == (0, 1, 64)
    tab = bw.rope_table(4, 16)
    assert bw.rope(none, None, tab)[0].shape == (0, 1, 64)
    assert bw.stream_status() == 0
    np.testing.assert_array_equal(raw(kc), before)
