"""Rotary positions and the paged key-value cache on torch tensors.

What a server needs around ``gqa_decode_paged``: rotary tables and rotations
with a position for every token, writes of new tokens into a paged cache (bf16
or 8-bit), spans read back for a chunk's attention, and the decode over the
8-bit cache.  Everything runs in the native library on the current CUDA stream;
there is no fallback path.

The 8-bit cache is ``k_cache`` / ``v_cache`` float8_e4m3fn
[num_pages, page_size, Hkv, D] with ``scales`` uint8 [num_pages, Hkv, 2, page_size]
(0: K, 1: V): the value of a row is code * 2**(scale - 127).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _ffi

_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
_E4M3 = torch.float8_e4m3fn


_A3, _A2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
# The current stream's handle without a Stream object around it (3 us of a call's 17 otherwise).
_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch.cuda.current_device


def _on_gpu(*tensors):
    """The index of the current CUDA device, on which every tensor given lies."""
    first = None
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d < 0:
                raise ValueError(f"expected CUDA tensors, got a {t.dtype} {tuple(t.shape)} tensor on {t.device}")
            if d != first:
                if first is not None:
                    raise ValueError(f"the tensors are on different devices (cuda:{first} and cuda:{d})")
                first = d
    dev = _device()
    if first is not None and first != dev:
        raise ValueError(f"the tensors are on cuda:{first}, the current device is cuda:{dev}")
    return dev


def _want(name, t, dtype, shape):
    """A contiguous tensor of this dtype and shape."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} tensor, got {tuple(t.shape)}")


def _table(t):
    if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous():
        raise ValueError("cos_sin_cache must be a contiguous fp32 [length, rotary_dim] tensor")


def rope_table(length, rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=0, attention_factor=0.0,
               beta_fast=0.0, beta_slow=0.0, low_freq_factor=0.0, high_freq_factor=0.0, first=0, out=None):
    """cos | sin table fp32 [length, rotary_dim] of the positions first .. first + length - 1.

    scaling: "none", "linear" (positions / factor), "ntk" (a larger base), "yarn"
    (low frequencies interpolated, cos and sin times 0.1 ln(factor) + 1) or
    "bands" (interpolated by wavelength against original_length); the schedules'
    formulas and the meaning of 0 are at bw_rope_scaling in include/bw_attn.h."""
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
    length, rotary_dim = int(length), int(rotary_dim)
    dev = _on_gpu(out)
    if out is None:
        out = torch.empty((length, rotary_dim), dtype=torch.float32, device=torch.device("cuda", dev))
    else:
        _want("out", out, torch.float32, (length, rotary_dim))
    s = _ffi.BwRopeScaling(_SCALINGS[scaling], base, factor, original_length, attention_factor, beta_fast, beta_slow,
                           low_freq_factor, high_freq_factor)
    rc = _ffi.lib().bw_rope_table(out.data_ptr(), length, rotary_dim, int(first), ctypes.addressof(s),
                                  _raw_stream(dev))
    _ffi.check(rc, "bw_rope_table")
    return out


def _bhs(name, t):
    """Strides of a [B, H, S, D] tensor or of [tokens, H, D] (B = tokens, S = 1); None: contiguous."""
    if t.is_contiguous():
        return None
    st = t.stride()
    if st[-1] != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    return _A3(st[0], st[1], st[2] if len(st) == 4 else 0)


def rope(q, k, cos_sin_cache, positions=None, pos_offset=0, interleaved=False, inverse=False, q_out=None, k_out=None):
    """Rotates the first cos_sin_cache.shape[1] elements of every head of q and k
    (one launch; k may be None) -> (q_out, k_out).

    q, k: bf16 or fp32 [B, H, S, D] views (BHSD, or BSHD through .transpose(1, 2))
    with int32 positions [B, S], or [tokens, H, D] with positions [tokens]; None:
    0, 1, ... along S.  A token whose position + pos_offset is outside the table
    is copied.  interleaved: pairs (2i, 2i + 1) instead of (i, i + R / 2).
    inverse: the transposed rotation, which maps gradients of the outputs to
    gradients of the inputs.  q_out may be q (in place)."""
    nd, dtype, shape = q.dim(), q.dtype, q.shape
    if nd == 4:
        B, Hq, S, D = shape
    elif nd == 3:
        (B, Hq, D), S = shape, 1
    else:
        raise ValueError("q must be [B, H, S, D] or [tokens, H, D]")
    if dtype != torch.bfloat16 and dtype != torch.float32:
        raise TypeError(f"q must be bfloat16 or float32, got {dtype}")
    _table(cos_sin_cache)
    if q_out is None:
        q_out = torch.empty_like(q)
    elif q_out.shape != shape or q_out.dtype != dtype:
        raise ValueError(f"q_out must be a {dtype} {tuple(shape)} tensor")
    if k is None:
        if k_out is not None:
            raise ValueError("k_out without k")
        Hkv, kp, kop, ks, kos = 0, None, None, None, None
    else:
        k_shape = k.shape
        if k.dim() != nd or k.dtype != dtype or k_shape[0] != B or k_shape[2:] != shape[2:]:
            raise ValueError(f"k must be q's {dtype} tensor but for the number of heads, got {k.dtype} {tuple(k_shape)}")
        Hkv = k_shape[1]
        if k_out is None:
            k_out = torch.empty_like(k)
        elif k_out.shape != k_shape or k_out.dtype != dtype:
            raise ValueError(f"k_out must be a {dtype} {tuple(k_shape)} tensor")
        kp, kop, ks, kos = k.data_ptr(), k_out.data_ptr(), _bhs("k", k), _bhs("k_out", k_out)
    dev = _on_gpu(q, k, cos_sin_cache, positions, q_out, k_out)
    pos = None
    if positions is not None:
        _want("positions", positions, torch.int32, (B, S) if nd == 4 else (B,))
        pos = positions.data_ptr()
    elif nd == 3:   # 0, 1, ... along the tokens: one sequence
        B, S = 1, B
        turn = lambda t, st: None if t is None else _A3(0, t.stride(1), t.stride(0))  # noqa: E731
    if q.numel() == 0:
        return q_out, k_out
    qs, qos = _bhs("q", q), _bhs("q_out", q_out)
    if pos is None and nd == 3:
        qs, qos, ks, kos = turn(q, qs), turn(q_out, qos), turn(k, ks), turn(k_out, kos)
    rc = _ffi.lib().bw_rope(
        q.data_ptr(), q_out.data_ptr(), kp, kop, _ffi.BW_BF16 if dtype == torch.bfloat16 else _ffi.BW_F32, B, Hq, Hkv,
        S, D, qs, qos, ks, kos, cos_sin_cache.data_ptr(), cos_sin_cache.shape[0], cos_sin_cache.shape[1], pos,
        int(pos_offset), int(bool(interleaved)), int(bool(inverse)), _raw_stream(dev))
    _ffi.check(rc, "bw_rope")
    return q_out, k_out


def _cache(k_cache, v_cache, scales):
    """(dtype code, num_pages, page_size, Hkv, D) of a paged cache."""
    if k_cache.dim() != 4 or k_cache.dtype not in (torch.bfloat16, _E4M3):
        raise ValueError("k_cache must be a bfloat16 or float8_e4m3fn [num_pages, page_size, Hkv, D] tensor")
    num_pages, page_size, Hkv, D = k_cache.shape
    if not k_cache.is_contiguous():
        raise ValueError("k_cache must be contiguous")
    _want("v_cache", v_cache, k_cache.dtype, k_cache.shape)
    if k_cache.dtype == torch.bfloat16:
        if scales is not None:
            raise ValueError("a bfloat16 cache has no scales")
        return _ffi.BW_BF16, num_pages, page_size, Hkv, D
    if scales is None:
        raise ValueError("a float8_e4m3fn cache needs scales")
    _want("scales", scales, torch.uint8, (num_pages, Hkv, 2, page_size))
    return _ffi.BW_E4M3, num_pages, page_size, Hkv, D


def kv_cache_write(k, v, k_cache, v_cache, slots, scales=None, cos_sin_cache=None, positions=None, interleaved=False):
    """Writes new tokens into their slots of a paged cache -> (k_cache, v_cache).

    k, v: bf16 [tokens, Hkv, D] views with a contiguous last dimension (slices of
    one projection's output, say); slots int64 [tokens]: page * page_size + place,
    negative to skip the token; the slots of a call differ.  k_cache, v_cache:
    bf16, or float8_e4m3fn with uint8 scales.  With cos_sin_cache (fp32
    [length, rotary_dim]) and positions (int32 [tokens]) K is rotated on the way."""
    code, num_pages, page_size, Hkv, D = _cache(k_cache, v_cache, scales)
    if k.dim() != 3 or k.shape[1:] != (Hkv, D) or v.shape != k.shape:
        raise ValueError(f"k and v must be [tokens, {Hkv}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError("k and v must be bfloat16")
    T = k.shape[0]
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("k and v must have a contiguous last dimension")
    _want("slots", slots, torch.int64, (T,))
    table = pos = None
    length = R = 0
    if cos_sin_cache is not None:
        _table(cos_sin_cache)
        if positions is None:
            raise ValueError("cos_sin_cache needs positions")
        _want("positions", positions, torch.int32, (T,))
        table, pos = cos_sin_cache.data_ptr(), positions.data_ptr()
        length, R = cos_sin_cache.shape
    elif positions is not None:
        raise ValueError("positions need cos_sin_cache")
    dev = _on_gpu(k, v, k_cache, v_cache, slots, scales, cos_sin_cache, positions)
    rc = _ffi.lib().bw_kv_cache_write(
        k.data_ptr(), v.data_ptr(), _A2(ks[0], ks[1]), _A2(vs[0], vs[1]), T, Hkv, D, k_cache.data_ptr(),
        v_cache.data_ptr(), scales.data_ptr() if scales is not None else None, code, page_size, num_pages,
        slots.data_ptr(), table, length, R, pos, int(bool(interleaved)), _raw_stream(dev))
    _ffi.check(rc, "bw_kv_cache_write")
    return k_cache, v_cache


def kv_cache_read(k_cache, v_cache, block_table, kv_lens, out_offsets, scales=None, kv_starts=None, total_rows=None,
                  k_out=None, v_out=None):
    """Reads spans of sequences back as bf16 rows -> (k_out, v_out) [total_rows, Hkv, D].

    block_table int32 [B, max_pages]; tokens [kv_starts[b], kv_starts[b] +
    kv_lens[b]) of sequence b (int32; kv_starts None: from 0) go to the rows
    out_offsets[b] + 0, 1, ... (int64).  Other rows of given outputs are left as
    they are; without outputs give total_rows."""
    code, num_pages, page_size, Hkv, D = _cache(k_cache, v_cache, scales)
    B = kv_lens.numel()
    if block_table.dim() != 2:
        raise ValueError("block_table must be [B, max_pages]")
    _want("block_table", block_table, torch.int32, (B, block_table.shape[1]))
    _want("kv_lens", kv_lens, torch.int32, (B,))
    _want("out_offsets", out_offsets, torch.int64, (B,))
    if kv_starts is not None:
        _want("kv_starts", kv_starts, torch.int32, (B,))
    if total_rows is None:
        if k_out is None:
            raise ValueError("give k_out and v_out, or total_rows")
        total_rows = k_out.shape[0]
    dev = _on_gpu(k_cache, v_cache, block_table, kv_lens, out_offsets, scales, kv_starts, k_out, v_out)
    shape = (int(total_rows), Hkv, D)
    if k_out is None:
        k_out = torch.empty(shape, dtype=torch.bfloat16, device=k_cache.device)
    if v_out is None:
        v_out = torch.empty(shape, dtype=torch.bfloat16, device=k_cache.device)
    _want("k_out", k_out, torch.bfloat16, shape)
    _want("v_out", v_out, torch.bfloat16, shape)
    rc = _ffi.lib().bw_kv_cache_read(
        k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr() if scales is not None else None, code, page_size,
        num_pages, block_table.data_ptr(), block_table.shape[1], kv_lens.data_ptr(),
        kv_starts.data_ptr() if kv_starts is not None else None, out_offsets.data_ptr(), B, Hkv, D, k_out.data_ptr(),
        v_out.data_ptr(), shape[0], _raw_stream(dev))
    _ffi.check(rc, "bw_kv_cache_read")
    return k_out, v_out


def decode_fp8_workspace_size(B, Hq, Hkv, D):
    """Bytes of workspace that ``gqa_decode_paged_fp8`` needs."""
    return int(_ffi.lib().bw_gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D))


def gqa_decode_paged_fp8(q, k_cache, v_cache, scales, block_table, kv_lens, scale=None, workspace=None, out=None,
                         lse=None):
    """``gqa_decode_paged`` over the 8-bit cache -> (O bf16 [B, Hq, D], LSE fp32 [B, Hq]).

    q bf16 [B, Hq, D]; k_cache, v_cache float8_e4m3fn [num_pages, page_size, Hkv, D]
    with uint8 scales [num_pages, Hkv, 2, page_size]; block_table int32
    [B, max_pages]; kv_lens int32 [B].  workspace: a uint8 tensor of
    ``decode_fp8_workspace_size`` bytes, one for each call that may run at the
    same time as another; allocated when None."""
    code, num_pages, page_size, Hkv, D = _cache(k_cache, v_cache, scales)
    if code != _ffi.BW_E4M3:
        raise TypeError("k_cache and v_cache must be float8_e4m3fn (gqa_decode_paged reads a bfloat16 cache)")
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [B, Hq, {D}]")
    B, Hq, _ = q.shape
    _want("q", q, torch.bfloat16, (B, Hq, D))
    if block_table.dim() != 2:
        raise ValueError("block_table must be [B, max_pages]")
    max_pages = block_table.shape[1]
    _want("block_table", block_table, torch.int32, (B, max_pages))
    _want("kv_lens", kv_lens, torch.int32, (B,))
    dev = _on_gpu(q, k_cache, v_cache, scales, block_table, kv_lens, workspace, out, lse)
    if out is None:
        out = torch.empty_like(q)
    else:
        _want("out", out, torch.bfloat16, (B, Hq, D))
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device)
    else:
        _want("lse", lse, torch.float32, (B, Hq))
    if workspace is None:
        workspace = torch.empty(decode_fp8_workspace_size(B, Hq, Hkv, D), dtype=torch.uint8, device=q.device)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    rc = _ffi.lib().bw_gqa_decode_paged_fp8(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), block_table.data_ptr(),
        kv_lens.data_ptr(), out.data_ptr(), lse.data_ptr(), B, Hq, Hkv, D, page_size, num_pages, max_pages,
        float(scale if scale is not None else 1.0 / math.sqrt(D)), workspace.data_ptr(), workspace.nbytes,
        _raw_stream(dev))
    _ffi.check(rc, "bw_gqa_decode_paged_fp8")
    return out, lse
