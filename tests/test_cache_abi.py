"""Refusals of the rotary and cache entry points, without a GPU: bad arguments
come back as status codes before anything touches the device, and the torch
front end names what is wrong."""
import ctypes

import pytest
import torch

import blackwell_b200 as bw
from blackwell_b200 import _ffi

P = 0x100000          # 256-byte aligned, never read
NONE, LINEAR, NTK, YARN, BANDS = range(5)


def _scaling(**kw):
    s = _ffi.BwRopeScaling(NONE, 10000.0, 1.0, 0.0)
    for k, v in kw.items():
        setattr(s, k, v)
    return ctypes.addressof(s), s


@pytest.mark.parametrize("kw,want", [
    (dict(table=None), "NULL"), (dict(length=0), "SHAPE"), (dict(R=7), "SHAPE"), (dict(R=0), "SHAPE"),
    (dict(R=514), "SHAPE"), (dict(first=-1), "SHAPE"), (dict(first=(1 << 31) - 4), "SHAPE"), (dict(table=P + 2), "ALIGN"),
    (dict(scaling=dict(base=1.0)), "SHAPE"), (dict(scaling=dict(base=float("nan"))), "SHAPE"),
    (dict(scaling=dict(kind=5)), "SHAPE"), (dict(scaling=dict(kind=LINEAR, factor=0.0)), "SHAPE"),
    (dict(scaling=dict(kind=YARN, factor=4.0)), "SHAPE"), (dict(scaling=dict(kind=BANDS, factor=4.0)), "SHAPE"),
    (dict(R=2, scaling=dict(kind=NTK, factor=4.0)), "SHAPE"), (dict(scaling=dict(attention_factor=-1.0)), "SHAPE"),
    (dict(scaling=dict(kind=BANDS, factor=4.0, original_length=100.0, low_freq_factor=5.0)), "SHAPE"),
])
def test_rope_table_refuses(kw, want):
    sp, keep = _scaling(**kw.pop("scaling", {}))
    a = dict(table=P, length=10, R=64, first=0) | kw
    rc = _ffi.lib().bw_rope_table(a["table"], a["length"], a["R"], a["first"], sp, None)
    assert rc == getattr(_ffi, "BW_ERR_" + want)


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), "NULL"), (dict(q_out=None), "NULL"), (dict(table=None), "NULL"), (dict(k_out=None), "NULL"),
    (dict(k=None), "NULL"), (dict(k=None, k_out=None), "SHAPE"), (dict(dtype=2), "SHAPE"), (dict(dtype=7), "SHAPE"),
    (dict(B=0), "SHAPE"), (dict(S=0), "SHAPE"), (dict(Hq=0), "SHAPE"), (dict(Hkv=0), "SHAPE"), (dict(D=60), "SHAPE"),
    (dict(D=520), "SHAPE"), (dict(R=24), "SHAPE"), (dict(R=0), "SHAPE"), (dict(R=80), "SHAPE"), (dict(length=-1), "SHAPE"),
    (dict(B=1 << 20, S=1 << 12), "SHAPE"), (dict(q=P + 8), "ALIGN"), (dict(k_out=P + 2), "ALIGN"),
    (dict(table=P + 4), "ALIGN"), (dict(positions=P + 2), "ALIGN"), (dict(qs=_i64(4096, 1024, 60)), "ALIGN"),
    (dict(qs=_i64(4096, 0, 64)), "ALIGN"), (dict(ks=_i64(4096, -1024, 64)), "ALIGN"),
])
def test_rope_refuses(kw, want):
    a = dict(q=P, q_out=P, k=P, k_out=P, dtype=0, B=2, Hq=8, Hkv=2, S=16, D=64, qs=None, ks=None, table=P, length=10,
             R=64, positions=P) | kw
    rc = _ffi.lib().bw_rope(a["q"], a["q_out"], a["k"], a["k_out"], a["dtype"], a["B"], a["Hq"], a["Hkv"], a["S"],
                            a["D"], a["qs"], None, a["ks"], None, a["table"], a["length"], a["R"], a["positions"], 0, 0,
                            0, None)
    assert rc == getattr(_ffi, "BW_ERR_" + want)


WRITE = dict(k=P, v=P, ks=None, vs=None, T=4, Hkv=2, D=64, kc=P, vc=P, sc=P, dt=2, ps=16, pages=8, slots=P, table=P,
             length=10, R=64, pos=P)


@pytest.mark.parametrize("kw,want", [
    (dict(k=None), "NULL"), (dict(vc=None), "NULL"), (dict(slots=None), "NULL"), (dict(sc=None), "NULL"),
    (dict(pos=None), "NULL"), (dict(T=-1), "SHAPE"), (dict(Hkv=0), "SHAPE"), (dict(D=96), "SHAPE"), (dict(dt=1), "SHAPE"),
    (dict(ps=12), "SHAPE"), (dict(ps=4), "SHAPE"), (dict(ps=96), "SHAPE"), (dict(pages=0), "SHAPE"),
    (dict(pages=1 << 28), "SHAPE"), (dict(R=8), "SHAPE"), (dict(R=128), "SHAPE"), (dict(length=-1), "SHAPE"),
    (dict(T=1 << 30, Hkv=2), "SHAPE"), (dict(k=P + 8), "ALIGN"), (dict(vc=P + 8), "ALIGN"), (dict(slots=P + 4), "ALIGN"),
    (dict(ks=_i64(100, 64)), "ALIGN"), (dict(vs=_i64(128, 0)), "ALIGN"), (dict(T=0, k=None), "OK"),
])
def test_kv_cache_write_refuses(kw, want):
    a = WRITE | kw
    rc = _ffi.lib().bw_kv_cache_write(a["k"], a["v"], a["ks"], a["vs"], a["T"], a["Hkv"], a["D"], a["kc"], a["vc"],
                                      a["sc"], a["dt"], a["ps"], a["pages"], a["slots"], a["table"], a["length"], a["R"],
                                      a["pos"], 0, None)
    assert rc == (0 if want == "OK" else getattr(_ffi, "BW_ERR_" + want))


READ = dict(kc=P, vc=P, sc=P, dt=2, ps=16, pages=8, bt=P, width=4, lens=P, starts=None, offs=P, B=2, Hkv=2, D=64, ko=P,
            vo=P, rows=100)


@pytest.mark.parametrize("kw,want", [
    (dict(kc=None), "NULL"), (dict(sc=None), "NULL"), (dict(bt=None), "NULL"), (dict(offs=None), "NULL"),
    (dict(vo=None), "NULL"), (dict(dt=1), "SHAPE"), (dict(B=-1), "SHAPE"), (dict(B=4097), "SHAPE"), (dict(D=32), "SHAPE"),
    (dict(width=0), "SHAPE"), (dict(width=1 << 27), "SHAPE"), (dict(ps=24), "SHAPE"), (dict(rows=-1), "SHAPE"),
    (dict(ko=P + 8), "ALIGN"), (dict(offs=P + 4), "ALIGN"), (dict(starts=P + 2), "ALIGN"), (dict(B=0, kc=None), "OK"),
    (dict(rows=0, ko=None), "OK"),
])
def test_kv_cache_read_refuses(kw, want):
    a = READ | kw
    rc = _ffi.lib().bw_kv_cache_read(a["kc"], a["vc"], a["sc"], a["dt"], a["ps"], a["pages"], a["bt"], a["width"],
                                     a["lens"], a["starts"], a["offs"], a["B"], a["Hkv"], a["D"], a["ko"], a["vo"],
                                     a["rows"], None)
    assert rc == (0 if want == "OK" else getattr(_ffi, "BW_ERR_" + want))


DECODE = dict(q=P, kc=P, vc=P, sc=P, bt=P, lens=P, o=P, lse=None, B=2, Hq=8, Hkv=2, D=64, ps=16, pages=8, width=4,
              scale=0.125, ws=P, n=1 << 30)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), "NULL"), (dict(sc=None), "NULL"), (dict(bt=None), "NULL"), (dict(o=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(B=0), "SHAPE"), (dict(B=4097), "SHAPE"), (dict(Hq=7), "SHAPE"), (dict(Hq=34), "SHAPE"), (dict(D=96), "SHAPE"),
    (dict(ps=20), "SHAPE"), (dict(pages=0), "SHAPE"), (dict(width=0), "SHAPE"), (dict(width=1 << 27), "SHAPE"),
    (dict(scale=0.0), "SHAPE"), (dict(scale=float("inf")), "SHAPE"), (dict(Hkv=2048, Hq=2048), "SHAPE"),
    (dict(B=4096, width=1 << 22), "SHAPE"), (dict(q=P + 8), "ALIGN"), (dict(sc=P + 4), "ALIGN"), (dict(ws=P + 8), "ALIGN"),
    (dict(lens=P + 2), "ALIGN"), (dict(n=100), "WORKSPACE"),
])
def test_decode_fp8_refuses(kw, want):
    a = DECODE | kw
    rc = _ffi.lib().bw_gqa_decode_paged_fp8(a["q"], a["kc"], a["vc"], a["sc"], a["bt"], a["lens"], a["o"], a["lse"],
                                            a["B"], a["Hq"], a["Hkv"], a["D"], a["ps"], a["pages"], a["width"],
                                            a["scale"], a["ws"], a["n"], None)
    assert rc == getattr(_ffi, "BW_ERR_" + want)


def test_decode_fp8_workspace_covers_every_part():
    size = _ffi.lib().bw_gqa_decode_paged_fp8_workspace_size
    for B, Hkv, G, D in [(1, 8, 4, 128), (64, 8, 8, 128), (4096, 1, 16, 64), (3, 5, 3, 64)]:
        parts = (1024 // Hkv + B) * Hkv
        assert size(B, Hkv * G, Hkv, D) >= 4 * (B + 1) + parts * G * (D + 1) * 4
    assert size(0, 8, 2, 64) == 0 and size(1, 7, 2, 64) == 0
    assert bw.decode_fp8_workspace_size(2, 8, 2, 64) == size(2, 8, 2, 64)


def test_index_error_has_a_text():
    assert _ffi.strerror(_ffi.BW_ERR_INDEX) != "unknown error"


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_front_end_refuses_what_it_cannot_run():
    """Wrong types and shapes, and tensors that are not on the GPU, raise before any call."""
    f8 = torch.float8_e4m3fn
    kc, sc = _cpu(4, 16, 2, 64, dtype=f8), _cpu(4, 2, 2, 16, dtype=torch.uint8)
    k, slots = _cpu(3, 2, 64), _cpu(3, dtype=torch.int64)
    tab, pos = _cpu(10, 64, dtype=torch.float32), _cpu(3, dtype=torch.int32)
    for call in (
        lambda: bw.kv_cache_write(k, k, kc, kc, slots, sc),                               # all on the CPU
        lambda: bw.kv_cache_write(k, k, kc, kc, slots),                                    # no scales
        lambda: bw.kv_cache_write(k, k, kc.to(torch.bfloat16), kc.to(torch.bfloat16), slots, sc),   # scales with bf16
        lambda: bw.kv_cache_write(k, k, kc, kc, slots, sc.view(4, 2, 16, 2)),
        lambda: bw.kv_cache_write(k[:, :1], k[:, :1], kc, kc, slots, sc),
        lambda: bw.kv_cache_write(k, k, kc, kc, slots[:2], sc),
        lambda: bw.kv_cache_write(k, k, kc, kc, slots, sc, cos_sin_cache=tab),
        lambda: bw.kv_cache_write(k, k, kc, kc, slots, sc, positions=pos),
        lambda: bw.kv_cache_write(k.transpose(1, 2).contiguous().transpose(1, 2), k, kc, kc, slots, sc),
        lambda: bw.kv_cache_read(kc, kc, _cpu(2, 4, dtype=torch.int32), _cpu(2, dtype=torch.int32),
                                 _cpu(2, dtype=torch.int64), sc, total_rows=5),
        lambda: bw.kv_cache_read(kc, kc, _cpu(2, 4, dtype=torch.int32), _cpu(2, dtype=torch.int32),
                                 _cpu(2, dtype=torch.int64), sc),
        lambda: bw.gqa_decode_paged_fp8(_cpu(2, 8, 64), kc, kc, sc, _cpu(2, 4, dtype=torch.int32),
                                        _cpu(2, dtype=torch.int32)),
        lambda: bw.gqa_decode_paged_fp8(_cpu(2, 8, 128), kc, kc, sc, _cpu(2, 4, dtype=torch.int32),
                                        _cpu(2, dtype=torch.int32)),
        lambda: bw.rope(_cpu(2, 4, 8, 64), None, tab),
        lambda: bw.rope(_cpu(4, 64), None, tab),
        lambda: bw.rope(_cpu(3, 4, 64), _cpu(2, 4, 64), tab),
        lambda: bw.rope(_cpu(3, 4, 64), None, tab, k_out=_cpu(3, 4, 64)),
        lambda: bw.rope(_cpu(3, 4, 64), None, tab[:, ::2]),
        lambda: bw.rope(_cpu(3, 4, 64), None, tab, q_out=_cpu(3, 4, 32)),
        lambda: bw.rope_table(8, 64, scaling="dynamic"),
        lambda: bw.rope_table(8, 64, out=_cpu(8, 64, dtype=torch.float32)),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: bw.kv_cache_write(k.float(), k.float(), kc, kc, slots, sc),
        lambda: bw.kv_cache_write(k, k, kc, kc, slots.int(), sc),
        lambda: bw.gqa_decode_paged_fp8(_cpu(2, 8, 64), kc.to(torch.bfloat16), kc.to(torch.bfloat16), None,
                                        _cpu(2, 4, dtype=torch.int32), _cpu(2, dtype=torch.int32)),
        lambda: bw.rope(_cpu(3, 4, 64, dtype=torch.float16), None, tab),
    ):
        with pytest.raises(TypeError):
            call()
