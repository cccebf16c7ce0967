"""The serving path as it is used: rotary table -> K rotated and quantised into
pages -> decode; and a prompt in two chunks, the first read back for the second's
attention."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as orc
from oracle import cache_oracle as co
from tests._util import LSE_TOL, O_TOL, seeded_bf16

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
Hq, Hkv, D, R, PS = 8, 2, 128, 64, 16


def _cache(pages, fp8):
    if fp8:
        z = torch.full((2, pages, PS, Hkv, D), 0x7f, dtype=torch.uint8, device="cuda")
        return z[0].view(F8), z[1].view(F8), torch.zeros(pages, Hkv, 2, PS, dtype=torch.uint8, device="cuda")
    z = torch.zeros(2, pages, PS, Hkv, D, dtype=torch.bfloat16, device="cuda")
    return z[0], z[1], None


@pytest.mark.parametrize("fp8", [True, False])
def test_chunks_then_decode(fp8):
    """Two sequences: 45 and 70 prompt tokens written in two chunks, attention of the second chunk over the read-back
    prefix, then three decode steps.  Everything is compared with attention over the cache's own values, so the
    quantisation is exact in the comparison and the tolerances are the attention kernels'."""
    import blackwell_b200 as bw
    B, steps = 2, 3
    prompt, cut = [45, 70], [20, 33]
    total = [n + steps for n in prompt]
    width = max((n + PS - 1) // PS for n in total)
    pages = B * width + 1
    bt = torch.from_numpy(np.random.default_rng(1).permutation(pages)[:B * width].reshape(B, width).astype(np.int32)).cuda()
    kc, vc, sc = _cache(pages, fp8)
    tab = bw.rope_table(128, R, scaling="linear", factor=2.0)
    xs = [seeded_bf16((n, (Hq + 2 * Hkv) * D), 10 + b).cuda() for b, n in enumerate(total)]
    q = [x[:, :Hq * D].view(-1, Hq, D) for x in xs]
    k = [x[:, Hq * D:(Hq + Hkv) * D].view(-1, Hkv, D) for x in xs]
    v = [x[:, (Hq + Hkv) * D:].view(-1, Hkv, D) for x in xs]
    scale = 1 / math.sqrt(D)

    def write(b, lo, hi):
        pos = torch.arange(lo, hi, device="cuda")
        slots = bt[b][pos // PS].long() * PS + pos % PS
        bw.kv_cache_write(k[b][lo:hi], v[b][lo:hi], kc, vc, slots, scales=sc, cos_sin_cache=tab, positions=pos.int())

    def held(b, n):
        """Values of the cache, by the oracle: rotation in fp32, rounding to the cache's type."""
        kr = co.rotate(k[b][:n].float().cpu().numpy().transpose(1, 0, 2), np.arange(n), tab.cpu().numpy(), False,
                       dtype=np.float32).transpose(1, 0, 2)
        out = []
        for x in (kr, v[b][:n].float().cpu().numpy()):
            out.append(co.cache_values(*co.quantise_rows(x)) if fp8 else torch.from_numpy(np.ascontiguousarray(x)).bfloat16().double().numpy())
        return out

    for b in range(B):
        write(b, 0, cut[b])
        write(b, cut[b], prompt[b])
        # the second chunk attends to everything before it
        n = prompt[b]
        lens = torch.tensor([n], dtype=torch.int32).cuda()
        ko, vo = bw.kv_cache_read(kc, vc, bt[b:b + 1], lens, torch.zeros(1, dtype=torch.int64).cuda(), scales=sc,
                                  total_rows=n)
        pos = torch.arange(cut[b], n, dtype=torch.int32).cuda()
        qr, _ = bw.rope(q[b][cut[b]:n], None, tab, positions=pos)
        as_bhsd = lambda t: t[None].transpose(1, 2)  # noqa: E731
        o, lse = bw.gqa_causal_offset_fwd(as_bhsd(qr), as_bhsd(ko), as_bhsd(vo), cut[b], scale)
        assert bw.stream_status() == 0
        hk, hv = held(b, n)
        np.testing.assert_array_equal(ko.double().cpu().numpy(), hk)
        np.testing.assert_array_equal(vo.double().cpu().numpy(), hv)
        rows = [(0, h, i) for h in range(Hq) for i in (0, n - cut[b] - 1)]
        ro, rl = orc.fp64_rows(as_bhsd(qr).cpu(), torch.from_numpy(hk)[None].transpose(1, 2),
                               torch.from_numpy(hv)[None].transpose(1, 2), scale, True, rows, cut[b])
        got = np.stack([o[0, h, i].float().cpu().numpy() for _, h, i in rows])
        assert np.abs(got - ro).max() <= O_TOL
        assert max(abs(float(lse[0, h, i]) - rl[j]) for j, (_, h, i) in enumerate(rows)) <= LSE_TOL
    ws = torch.empty(bw.decode_fp8_workspace_size(B, Hq, Hkv, D), dtype=torch.uint8, device="cuda")
    for step in range(steps):
        at = [n + step for n in prompt]
        pos = torch.tensor(at, dtype=torch.int32).cuda()
        x = torch.stack([xs[b][at[b]] for b in range(B)])
        qn, kn, vn = x[:, :Hq * D].view(B, Hq, D), x[:, Hq * D:(Hq + Hkv) * D].view(B, Hkv, D), x[:, (Hq + Hkv) * D:].view(B, Hkv, D)
        slots = bt[torch.arange(B).cuda(), pos.long() // PS].long() * PS + pos % PS
        bw.kv_cache_write(kn, vn, kc, vc, slots, scales=sc, cos_sin_cache=tab, positions=pos)
        qr, _ = bw.rope(qn, None, tab, positions=pos)
        qr = qr.contiguous()
        if fp8:
            o, lse = bw.gqa_decode_paged_fp8(qr, kc, vc, sc, bt, pos + 1, workspace=ws)
        else:
            o, lse = bw.gqa_decode_paged(qr, kc, vc, bt, pos + 1)
        assert bw.stream_status() == 0
        for b in range(B):
            hk, hv = held(b, at[b] + 1)
            wo, wl, _, _ = co.decode(qr[b].double().cpu().numpy(), hk, hv, scale)
            assert np.abs(o[b].float().cpu().numpy() - wo).max() <= O_TOL
            assert np.abs(lse[b].cpu().numpy() - wl).max() <= LSE_TOL


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB a tensor: tokens in its first and last pages, written,
    read back and attended to."""
    import blackwell_b200 as bw
    h, d, ps = 8, 128, 64
    pages = (5 << 30) // (ps * h * d)
    kc = torch.empty(pages, ps, h, d, dtype=torch.uint8, device="cuda").view(F8)
    vc = torch.empty(pages, ps, h, d, dtype=torch.uint8, device="cuda").view(F8)
    sc = torch.empty(pages, h, 2, ps, dtype=torch.uint8, device="cuda")
    bt = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32).cuda()
    n = 2 * ps + 9
    k, v = seeded_bf16((n, h, d), 1).cuda(), seeded_bf16((n, h, d), 2).cuda()
    pos = torch.arange(n, device="cuda")
    bw.kv_cache_write(k, v, kc, vc, bt[0][pos // ps].long() * ps + pos % ps, scales=sc)
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    ko, vo = bw.kv_cache_read(kc, vc, bt, lens, torch.zeros(1, dtype=torch.int64).cuda(), scales=sc, total_rows=n)
    q = seeded_bf16((1, 2 * h, d), 3).cuda()
    o, lse = bw.gqa_decode_paged_fp8(q, kc, vc, sc, bt, lens)
    assert bw.stream_status() == 0
    held = [co.cache_values(*co.quantise_rows(x.float().cpu().numpy())) for x in (k, v)]
    np.testing.assert_array_equal(ko.double().cpu().numpy(), held[0])
    np.testing.assert_array_equal(vo.double().cpu().numpy(), held[1])
    wo, wl, _, _ = co.decode(q[0].double().cpu().numpy(), held[0], held[1], 1 / math.sqrt(d))
    assert np.abs(o[0].float().cpu().numpy() - wo).max() <= O_TOL
    assert np.abs(lse[0].cpu().numpy() - wl).max() <= LSE_TOL


def test_first_calls_of_a_process_can_be_captured():
    """Every entry point captured into a graph before it ever ran outside one."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch, blackwell_b200 as bw
z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")
q, k = z(2, 4, 64) + 1, z(2, 2, 64) + 1
kc, vc, sc = z(3, 8, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), z(3, 8, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), z(3, 2, 2, 8, dtype=torch.uint8)
bt, lens, offs = torch.tensor([[1], [2]], dtype=torch.int32).cuda(), torch.tensor([1, 1], dtype=torch.int32).cuda(), torch.tensor([0, 1]).cuda()
tab, pos, slots = z(8, 64, dtype=torch.float32), z(2, dtype=torch.int32), torch.tensor([8, 16]).cuda()
o, lse, ws = z(2, 4, 64), z(2, 4, dtype=torch.float32), z(bw.decode_fp8_workspace_size(2, 4, 2, 64), dtype=torch.uint8)
ko, vo, qo = z(2, 2, 64), z(2, 2, 64), z(2, 4, 64)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    bw.rope_table(8, 64, out=tab)
    bw.rope(q, None, tab, positions=pos, q_out=qo)
    bw.kv_cache_write(k, k, kc, vc, slots, scales=sc, cos_sin_cache=tab, positions=pos)
    bw.kv_cache_read(kc, vc, bt, lens, offs, scales=sc, k_out=ko, v_out=vo)
    bw.gqa_decode_paged_fp8(qo, kc, vc, sc, bt, lens, workspace=ws, out=o, lse=lse)
g.replay()
torch.cuda.synchronize()
assert torch.all(ko == 1) and torch.all(vo == 1) and torch.all(o == 1) and torch.all(lse == 8), (ko, o, lse)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]


def test_calls_from_two_host_threads():
    """Two threads, each on its own stream with its own workspace and outputs, over one cache."""
    import threading

    import blackwell_b200 as bw
    h, d = 2, 128
    lens_l = [700, 90]
    bt = torch.arange(2 * 44, dtype=torch.int32).view(2, 44).cuda()
    kc, vc, sc = _cache(88, True)
    for b, n in enumerate(lens_l):
        k, v = seeded_bf16((n, h, d), 20 + b).cuda(), seeded_bf16((n, h, d), 30 + b).cuda()
        pos = torch.arange(n, device="cuda")
        bw.kv_cache_write(k, v, kc, vc, bt[b][pos // PS].long() * PS + pos % PS, scales=sc)
    lens = torch.tensor(lens_l, dtype=torch.int32).cuda()
    qs = [seeded_bf16((2, 8, d), 40 + i).cuda() for i in range(2)]
    want = [bw.gqa_decode_paged_fp8(q, kc, vc, sc, bt, lens) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(200):
                o, lse = bw.gqa_decode_paged_fp8(qs[i], kc, vc, sc, bt, lens)
                if _ % 50 == 0:
                    st.synchronize()
                    if not (torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])):
                        bad.append(i)
            st.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
