"""Decode over the paged 8-bit cache against fp64, at the places where it can go
wrong: lengths around tiles and pages, empty sequences, stale bytes of any value
behind a sequence, rows of very unlike scale, every group size."""
import math

import numpy as np
import pytest
import torch

from oracle import cache_oracle as co
from tests._util import seeded_bf16

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def make(lens, Hkv, G, D, ps, seed, spread=3, extra_pages=2, width_extra=1):
    """A random cache: codes, scale bytes 127 - 7 +- spread; bytes that no sequence owns (the rest of last pages, free
    pages) hold NaN codes and scale bytes 0 or 255; table entries past a sequence are -1 or far out of range."""
    rng = np.random.default_rng(seed)
    need = [(n + ps - 1) // ps for n in lens]
    pages = sum(need) + extra_pages
    perm = rng.permutation(pages)
    bt = rng.choice([-1, 1 << 30, pages], (len(lens), max(max(need), 1) + width_extra)).astype(np.int32)
    codes = np.full((2, pages, ps, Hkv, D), 0x7f, np.uint8)
    sc = rng.choice([0, 255], (pages, Hkv, 2, ps)).astype(np.uint8)
    at = 0
    for b, n in enumerate(lens):
        bt[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        pg, sl = bt[b, t // ps], t % ps
        x = rng.standard_normal((2, n, Hkv, D)) * 100
        codes[:, pg, sl] = co.to_e4m3(np.clip(x, -448, 448))
        sc[pg, :, :, sl] = rng.integers(120 - spread, 121 + spread, (n, Hkv, 2))
    q = seeded_bf16((len(lens), Hkv * G, D), seed + 1)
    return q, codes, sc, bt


def run(q, codes, sc, bt, lens, **kw):
    import blackwell_b200 as bw
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    o, lse = bw.gqa_decode_paged_fp8(q.cuda(), cu(codes[0]).view(F8), cu(codes[1]).view(F8), cu(sc), cu(bt),
                                     torch.tensor(lens, dtype=torch.int32).cuda(), **kw)
    return o, lse


def check(o, lse, q, codes, sc, bt, lens, scale=None):
    """Bounds, with u = 2^-24.  Scores: an fp32 dot of D products and three factors, off by at most dx = (D + 8) u max_t
    scale sum|q k| + 2^-21 |x|max (log2 units and ex2's 2^-22).  LSE: 2 dx + L u for the sum.  O: every weight is rounded
    to fp16 (2^-11 relative; 2^-25 of the largest weight * value scale below fp16's normals) and off by 2 dx, the sums by
    L u: sum p|v| (2^-11 + 4 dx + 2 L u) + 2^-24 max p 2^e 448, then 2^-8 |O| for bf16."""
    ps = codes.shape[2]
    D = q.shape[2]
    scale = scale if scale is not None else 1 / math.sqrt(D)
    o, lse = o.float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    for b, n in enumerate(lens):
        t = np.arange(n)
        pg, sl = bt[b, t // ps], t % ps
        k, v = (co.cache_values(codes[w][pg, sl], sc[pg, :, w, sl]) for w in (0, 1))
        wo, wl, mean_abs, size = co.decode(q[b].double().numpy(), k, v, scale)
        if n == 0:
            assert np.all(o[b] == 0) and np.all(np.isneginf(lse[b]))
            continue
        dx = (D + 8) * 2.0 ** -24 * size + 2.0 ** -21 * np.abs(size)
        assert np.all(np.abs(lse[b] - wl) <= 2 * dx + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * np.abs(wl)), b
        tol = mean_abs * (2.0 ** -11 + 4 * dx + 2 * n * 2.0 ** -24)[:, None] + 2.0 ** -8 * np.abs(wo)
        tol += 2.0 ** -24 * np.abs(v).max() * n
        assert np.all(np.abs(o[b] - wo) <= tol), (b, np.abs(o[b] - wo).max())


@pytest.mark.parametrize("G,Hkv,D,ps,lens", [
    (4, 8, 128, 16, [517]), (1, 1, 64, 8, [1]), (3, 4, 64, 64, [1, 63, 64, 65, 0, 300]),
    (8, 2, 128, 32, [255, 256, 257, 2]), (16, 1, 128, 128, [129, 1000]), (9, 3, 64, 256, [700, 5]),
    (8, 8, 128, 64, [1500, 0, 0, 7]), (5, 5, 128, 8, [77, 8, 9, 16, 15]), (2, 16, 64, 16, [33] * 9),
])
def test_decode_fp8(G, Hkv, D, ps, lens):
    import blackwell_b200 as bw
    q, codes, sc, bt = make(lens, Hkv, G, D, ps, G * 100 + D)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


@pytest.mark.parametrize("lens", [[9000], [20000, 3], [4096, 4097, 64, 0, 8191]])
def test_decode_fp8_split_over_the_length(lens):
    import blackwell_b200 as bw
    q, codes, sc, bt = make(lens, 2, 4, 128, 64, 11)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


def test_decode_fp8_many_sequences_and_all_empty():
    import blackwell_b200 as bw
    lens = list(np.random.default_rng(0).integers(0, 90, 700))
    q, codes, sc, bt = make(lens, 1, 4, 64, 16, 3)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)
    o, lse = run(q[:3], codes, sc, bt[:3], [0, 0, 0])
    assert bw.stream_status() == 0
    assert torch.all(o == 0) and torch.all(torch.isneginf(lse))


def test_decode_fp8_rows_of_unlike_scale():
    """Scales spread over 2^+-30: the largest keys decide, small values next to large
    ones keep their relative weight; peaked and flat rows."""
    import blackwell_b200 as bw
    lens = [200, 640]
    q, codes, sc, bt = make(lens, 2, 8, 128, 16, 21, spread=0)
    rng = np.random.default_rng(5)
    own = sc == 120
    v_part = np.zeros_like(own)
    v_part[:, :, 1] = True
    sc[own & v_part] = rng.integers(127 - 30, 127 + 31, int((own & v_part).sum()))
    sc[own & ~v_part] = rng.integers(127 - 20, 122, int((own & ~v_part).sum()))
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


def test_decode_fp8_small_and_large_queries_and_scales():
    """Q rows of 2^-60 and 2^60 with K scales that make up for them; a given softmax scale."""
    import blackwell_b200 as bw
    lens = [130, 65]
    q, codes, sc, bt = make(lens, 1, 4, 64, 16, 31, spread=0)
    q = q.float()
    q[0] *= 2.0 ** -60
    q[1] *= 2.0 ** 60
    q = q.bfloat16()
    for b, shift in ((0, 60), (1, -60)):
        t = np.arange(lens[b])
        sc[bt[b, t // 16], :, 0, t % 16] = 120 + shift
    o, lse = run(q, codes, sc, bt, lens, scale=0.05)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens, scale=0.05)


def test_decode_fp8_nan_stays_in_its_row():
    """A NaN key makes its head's row NaN, a NaN value its column of that head; nothing else changes."""
    lens = [100, 70]
    q, codes, sc, bt = make(lens, 2, 4, 64, 16, 41)
    o0, l0 = run(q, codes, sc, bt, lens)
    codes[1, bt[0, 0], 3, 1, 5] = 0xff              # V of token 3, head 1, column 5
    o1, l1 = run(q, codes, sc, bt, lens)
    bad = torch.zeros_like(o0, dtype=torch.bool)
    bad[0, 4:, 5] = True
    assert torch.all(torch.isnan(o1[bad])) and torch.equal(o1[~bad], o0[~bad]) and torch.equal(l1, l0)
    codes[0, bt[1, 4], 5, 0, 0] = 0x7f              # K of token 69, head 0
    o2, l2 = run(q, codes, sc, bt, lens)
    assert torch.all(torch.isnan(o2[1, :4])) and torch.all(torch.isnan(l2[1, :4]))
    assert torch.equal(o2[1, 4:], o0[1, 4:]) and torch.equal(o2[0][~bad[0]], o0[0][~bad[0]])


def test_decode_fp8_bad_page_and_length_are_reported():
    """A page outside the cache is read as page 0 and a length beyond the table is cut
    to it; both report BW_ERR_INDEX or run as documented, and the other sequences are right."""
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    lens = [40, 50]
    q, codes, sc, bt = make(lens, 1, 4, 64, 16, 51, width_extra=0)
    good = bt.copy()
    bt[0, 1] = 12345
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == _ffi.BW_ERR_INDEX
    check(o[1:], lse[1:], q[1:], codes, sc, bt[1:], lens[1:])
    zero = good.copy()
    zero[0, 1] = 0
    oz, lz = run(q, codes, sc, zero, lens)
    assert bw.stream_status() == 0
    bad = torch.isnan(oz)                                  # page 0 may hold stale NaN codes
    assert torch.equal(o[~bad], oz[~bad]) and torch.equal(torch.isnan(o), bad)
    long, _ = run(q[1:], codes, sc, good[1:], [10 ** 6])   # table of 4 pages: 64 tokens
    cut, _ = run(q[1:], codes, sc, good[1:], [64])
    assert torch.equal(torch.isnan(long), torch.isnan(cut))
    assert torch.equal(long[~torch.isnan(long)], cut[~torch.isnan(cut)])
    bw.stream_status()


def test_decode_fp8_is_deterministic_and_needs_no_initial_workspace():
    import blackwell_b200 as bw
    lens = [3000, 5, 900]
    q, codes, sc, bt = make(lens, 4, 4, 128, 16, 61)
    n = bw.decode_fp8_workspace_size(3, 16, 4, 128)
    first = None
    for fill in (0x00, 0xff, 0x7f):
        ws = torch.full((n + 256,), fill, dtype=torch.uint8, device="cuda")
        o, lse = run(q, codes, sc, bt, lens, workspace=ws[:n])
        assert torch.all(ws[n:] == fill)
        if first is None:
            first = (o, lse)
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


def test_decode_fp8_in_graphs_and_on_streams():
    """Two graphs with a workspace each, replayed on two streams at once, with lengths
    that changed since the capture."""
    import blackwell_b200 as bw
    lens = [1000, 300]
    q, codes, sc, bt = make(lens, 2, 4, 128, 32, 71)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    kc, vc, s, t = cu(codes[0]).view(F8), cu(codes[1]).view(F8), cu(sc), cu(bt)
    qs = [q.cuda(), (q * 2).cuda()]
    lens_d = torch.tensor([1, 1], dtype=torch.int32).cuda()
    n = bw.decode_fp8_workspace_size(2, 8, 2, 128)
    outs, graphs = [], []
    bw.gqa_decode_paged_fp8(qs[0], kc, vc, s, t, lens_d)
    torch.cuda.synchronize()
    for x in qs:
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        o, l = torch.empty_like(x), torch.empty(2, 8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            bw.gqa_decode_paged_fp8(x, kc, vc, s, t, lens_d, workspace=ws, out=o, lse=l)
        outs.append((o, l, ws))
        graphs.append(g)
    lens_d.copy_(torch.tensor(lens, dtype=torch.int32))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st, g in zip(side, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for x, (o, l, _) in zip(qs, outs):
        check(o, l, x.cpu(), codes, sc, bt, lens)


@pytest.mark.parametrize("ps", [192, 320])
def test_decode_fp8_pages_that_are_no_power_of_two(ps):
    import blackwell_b200 as bw
    lens = [ps, ps + 1, 2 * ps - 1, 1000]
    for D in (64, 128):
        q, codes, sc, bt = make(lens, 2, 4, D, ps, 81)
        o, lse = run(q, codes, sc, bt, lens)
        assert bw.stream_status() == 0
        check(o, lse, q, codes, sc, bt, lens)


@pytest.mark.parametrize("D,B", [(128, 4096), (64, 4096)])
def test_decode_fp8_most_sequences(D, B):
    """The largest batch: its tile counts take the most shared memory."""
    import blackwell_b200 as bw
    lens = list(np.random.default_rng(1).integers(0, 20, B))
    q, codes, sc, bt = make(lens, 1, 2, D, 8, 91)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    some = [0, 1, 77, B - 2, B - 1]
    check(o[some], lse[some], q[some], codes, sc, bt[some], [lens[i] for i in some])


def test_decode_fp8_many_kv_heads():
    """More KV heads than resident blocks: one token group."""
    import blackwell_b200 as bw
    lens = [70, 3]
    q, codes, sc, bt = make(lens, 700, 1, 64, 8, 95)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


@pytest.mark.parametrize("seed", range(12))
def test_decode_fp8_random_shapes(seed):
    import blackwell_b200 as bw
    rng = np.random.default_rng(1000 + seed)
    D, ps = int(rng.choice([64, 128])), int(rng.choice([8, 16, 32, 64, 128, 192]))
    Hkv, G, B = int(rng.integers(1, 10)), int(rng.integers(1, 17)), int(rng.integers(1, 9))
    lens = [int(n) for n in np.exp(rng.uniform(0, math.log(5000), B)).astype(int) - 1]
    q, codes, sc, bt = make(lens, Hkv, G, D, ps, 2000 + seed)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


@pytest.mark.parametrize("D", [64, 128])
def test_decode_fp8_wait_that_runs_out_is_reported(D):
    """The K producers withhold their first tile (test hook): the consumers' bounded
    waits expire, every block unwinds, the call reports BW_ERR_TIMEOUT, and the next
    call on the stream is right."""
    import blackwell_b200 as bw
    from blackwell_b200 import _ffi
    lens = [3000, 0, 700]
    q, codes, sc, bt = make(lens, 4, 4, D, 16, 101)
    old = bw.get_option(_ffi.BW_OPT_TIMEOUT_NS)
    try:
        bw.set_option(_ffi.BW_OPT_TIMEOUT_NS, 20_000_000)   # 20 ms
        bw.set_option(_ffi.BW_OPT_DEBUG_FLAGS, 1)
        run(q, codes, sc, bt, lens)
        assert bw.stream_status() == _ffi.BW_ERR_TIMEOUT
    finally:
        bw.set_option(_ffi.BW_OPT_DEBUG_FLAGS, 0)
        bw.set_option(_ffi.BW_OPT_TIMEOUT_NS, old)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)


@pytest.mark.parametrize("D,extra", [(64, 0), (64, 40), (128, 0), (128, 40)])
def test_decode_fp8_tables_wide_and_narrow_agree(D, extra):
    """The same sequences with a table of few pages (they are not cut then) and with a
    wider one (cut and joined): both within the bounds, empty sequences among them."""
    import blackwell_b200 as bw
    lens = [0, 200, 17, 0, 128, 129, 1, 0]
    q, codes, sc, bt = make(lens, 2, 4, D, 16, 111, width_extra=extra)
    o, lse = run(q, codes, sc, bt, lens)
    assert bw.stream_status() == 0
    check(o, lse, q, codes, sc, bt, lens)
