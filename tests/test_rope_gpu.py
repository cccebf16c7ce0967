"""Rotary tables and rotations against the formulas in fp64 / 80 bits."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as co
from tests._util import seeded_bf16

pytestmark = pytest.mark.gpu


# fp32 output: half a step of the value (2^-24 of at most the magnitude m), at most 2 ulp of sincospif (2 * 2^-23 * m
# at values near 1), the rest's rounding to fp32 (2^-26 quarter turns), and the fp64 phase: three roundings of 2^-53
# and a pow of at most 2 ulp, relative to the number of turns.
def _table_tol(m, turns):
    return m * (2.0 ** -24 + 2.0 ** -22 + 2.0 ** -25) + 2 * np.pi * turns * 2.0 ** -50


@pytest.mark.parametrize("R,length,first,base,kw", [
    (64, 300, 0, 10000.0, {}),
    (2, 1, 0, 10000.0, {}),
    (22, 77, (1 << 20) - 30, 500000.0, {}),
    (128, 100, 131000, 500000.0, dict(scaling="linear", factor=8.0)),
    (128, 64, 1 << 19, 10000.0, dict(scaling="ntk", factor=4.0)),
    (64, 129, 70000, 10000.0, dict(scaling="yarn", factor=40.0, original_length=4096)),
    (6, 40, 100, 500000.0, dict(scaling="yarn", factor=2.0, original_length=2048)),
    (128, 65, 100000, 500000.0, dict(scaling="bands", factor=8.0, original_length=8192)),
    (512, 3, 0, 1000000.0, {}),
])
def test_rope_table(R, length, first, base, kw):
    import blackwell_b200 as bw
    t = bw.rope_table(length, R, base=base, first=first, **kw)
    want = co.table(first, length, R, base, **kw)
    f, m = co.frequencies(R, base, **kw)
    turns = (first + length) * float(f.max()) / (2 * np.pi)
    assert np.abs(t.cpu().numpy().astype(np.float64) - want).max() <= _table_tol(m, turns)


def test_rope_table_continues_and_feeds_the_fused_prologue():
    """Two pieces of a table are the rows of one, and an attention factor scales it."""
    import blackwell_b200 as bw
    whole = bw.rope_table(100, 64)
    assert torch.equal(torch.cat([bw.rope_table(37, 64), bw.rope_table(63, 64, first=37)]), whole)
    torch.testing.assert_close(bw.rope_table(100, 64, attention_factor=2.0), 2 * whole, rtol=0, atol=0)
    x = seeded_bf16((1, 2, 100, 64), 5).cuda()
    # the same rotation up to fp32 rounding (2^-21 of the row's largest, below 8), so at most one bf16 step apart
    a, b = bw.qk_norm_rope(x, whole).float(), bw.rope(x, None, whole)[0].float()
    assert torch.all((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -18)


def _check(y, x, pos, tab, interleaved, inverse, dtype):
    """y against the fp64 rotation of x.  Error of one output u = a c - b s in fp32: two products and a sum, each off
    by at most 2^-24 of itself: <= 2 * 2^-24 (|a c| + |b s|) (1 + 2^-24) < 2^-22 (|a| + |b|) max|c, s|; then the
    rounding to bf16: 2^-8 of the value.  |a| + |b| is at most 2 max|x| of the row."""
    want = co.rotate(x, pos, tab, interleaved, inverse)
    top = np.abs(x).max(-1, keepdims=True) * max(1.0, np.abs(tab).max())
    tol = 2.0 ** -21 * top + (2.0 ** -8 * (np.abs(want) + 2.0 ** -21 * top) if dtype == torch.bfloat16 else 0)
    assert np.all(np.abs(y - want) <= tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("layout,B,Hq,Hkv,S,D,R", [
    ("bhsd", 2, 6, 2, 37, 128, 128), ("bshd", 3, 5, 1, 65, 64, 32), ("thd", 1, 32, 8, 1, 128, 64),
    ("thd", 1, 3, 3, 129, 72, 48), ("bhsd", 1, 1, 0, 300, 256, 16), ("bshd", 1, 9, 0, 7, 24, 16),
])
def test_rope(layout, B, Hq, Hkv, S, D, R, interleaved, inverse, dtype):
    """Layouts, part of the head, positions below 0 and behind the table, odd counts."""
    import blackwell_b200 as bw
    rng = np.random.default_rng(S)
    tab = co.table(0, 50, R).astype(np.float32)
    pos = rng.integers(-3, 55, (B, S)).astype(np.int32)

    def make(H, seed):
        x = torch.randn(B, S, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype)
        flat = x.float().numpy().astype(np.float64).transpose(0, 2, 1, 3)     # [B, H, S, D]
        x = x.cuda()
        return (x[0] if layout == "thd" else x.transpose(1, 2).contiguous() if layout == "bhsd" else x.transpose(1, 2)), flat

    (q, qf), (k, kf) = make(Hq, 1), make(max(Hkv, 1), 2)
    k = k if Hkv else None
    p = torch.from_numpy(pos).cuda()
    qo, ko = bw.rope(q, k, torch.from_numpy(tab).cuda(), positions=p[0] if layout == "thd" else p,
                     interleaved=interleaved, inverse=inverse)
    assert bw.stream_status() == 0
    for y, flat in ((qo, qf), (ko, kf)):
        if y is None:
            assert not Hkv
            continue
        got = y.float().cpu().numpy().astype(np.float64)
        got = got.transpose(1, 0, 2)[None] if layout == "thd" else got
        _check(got, flat, pos[:, None, :], tab, interleaved, inverse, dtype)


def test_rope_strided_slices_in_place_and_offset():
    """Q and K as slices of one projection's output, rotated in place; the V part and
    the rest of the head stay; positions None with an offset."""
    import blackwell_b200 as bw
    T, Hq, Hkv, D, R = 45, 6, 2, 128, 64
    tab = bw.rope_table(64, R)
    qkv = seeded_bf16((T, (Hq + 2 * Hkv) * D), 3).cuda()
    before = qkv.clone()
    q, k = qkv[:, :Hq * D].view(T, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    bw.rope(q, k, tab, pos_offset=19, q_out=q, k_out=k)
    assert torch.equal(qkv[:, (Hq + Hkv) * D:], before[:, (Hq + Hkv) * D:])
    heads = qkv.view(T, -1, D)[:, :Hq + Hkv]
    was = before.view(T, -1, D)[:, :Hq + Hkv]
    assert torch.equal(heads[..., R:], was[..., R:])
    pos = np.arange(T) + 19
    _check(heads.float().cpu().numpy().transpose(1, 0, 2).astype(np.float64),
           was.float().cpu().numpy().transpose(1, 0, 2).astype(np.float64), pos, tab.cpu().numpy(), False, False,
           torch.bfloat16)
    # one further and the last token's position is the table's length: it stays
    past = bw.rope(was, None, tab, pos_offset=20)[0]
    assert torch.equal(past[T - 1], was[T - 1]) and not torch.equal(past[T - 2], was[T - 2])
    # the same out of place
    qo, ko = bw.rope(before[:, :Hq * D].view(T, Hq, D), before[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D), tab,
                     pos_offset=19)
    assert torch.equal(torch.cat([qo, ko], 1), heads)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_inverse_is_the_gradient(interleaved):
    """inverse = 1 on the outputs' gradients: the gradient of sum(w * rope(x)) by the
    formula, and central differences of the forward call itself (linear in x, so a
    difference over h = 1 has only the fp32 rounding of its two sides)."""
    import blackwell_b200 as bw
    B, H, S, D, R = 1, 2, 5, 32, 16
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(B, H, S, D, generator=g).cuda(), torch.randn(B, H, S, D, generator=g).cuda()
    tab = bw.rope_table(9, R, scaling="yarn", factor=4.0, original_length=8)
    pos = torch.tensor([[0, 3, 8, 9, -1]], dtype=torch.int32).cuda()
    dx = bw.rope(w, None, tab, positions=pos, interleaved=interleaved, inverse=True)[0]
    # formula: the transpose of the rotation's matrix, from the oracle applied to the unit vectors
    eye = np.broadcast_to(np.eye(D)[:, None, :], (D, S, D))
    rows = co.rotate(eye, pos.cpu().numpy()[0], tab.cpu().numpy(), interleaved)         # [e, s, :] = M_s e
    want = np.einsum("esd,bhsd->bhse", rows, w.cpu().numpy().astype(np.float64))
    m = max(1.0, float(tab.abs().max()))
    assert np.abs(dx.cpu().numpy() - want).max() <= 2.0 ** -21 * m * float(w.abs().max())
    for e in (0, 3, R // 2, R - 1, R, D - 1):
        d = torch.zeros_like(x)
        d[..., e] = 1.0
        up = bw.rope(x + d, None, tab, positions=pos, interleaved=interleaved)[0].double()
        dn = bw.rope(x - d, None, tab, positions=pos, interleaved=interleaved)[0].double()
        diff = ((up - dn) / 2 * w.double()).sum(-1)
        # each side: fp32 rounding of x +- d and of the rotation, <= 2^-21 (|x| + 1) m a value, over D values of w
        tol = 2.0 ** -20 * (float(x.abs().max()) + 1) * m * float(w.abs().max()) * 3
        assert (diff - dx[..., e].double()).abs().max() <= tol


def test_rope_on_another_stream_and_in_a_graph():
    import blackwell_b200 as bw
    tab = bw.rope_table(128, 64)
    q, k = seeded_bf16((33, 4, 64), 1).cuda(), seeded_bf16((33, 2, 64), 2).cuda()
    pos = torch.arange(33, dtype=torch.int32).cuda()
    want = bw.rope(q, k, tab, positions=pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bw.rope(q, k, tab, positions=pos)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bw.rope(q, k, tab, positions=pos, q_out=qo, k_out=ko)
    pos += 50
    graph.replay()
    torch.cuda.synchronize()
    want = bw.rope(q, k, tab, positions=pos)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
