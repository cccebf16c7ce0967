"""Rotary positions and the paged key-value cache on torch tensors.

What a server needs around ``gqa_decode_paged``: rotary tables and rotations
with a position for every token, writes of new tokens into a paged cache (bf16
or 8-bit), spans read back for a chunk's attention, and the decode over the
8-bit cache.  Everything runs in the native library on the current CUDA stream;
there is no fallback path.  The checks of the arguments are native too
(front/front.cpp): in Python they took longer than the kernels of a decode step.

The 8-bit cache is ``k_cache`` / ``v_cache`` float8_e4m3fn
[num_pages, page_size, Hkv, D] with ``scales`` uint8 [num_pages, Hkv, 2, page_size]
(0: K, 1: V): the value of a row is code * 2**(scale - 127).
"""
from __future__ import annotations

import importlib
import math

import torch

from . import _ffi

_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
_WANTS_GRADIENT = -1   # of the front end's rope: nothing was done, an argument requires gradients
_front = None


def _load():
    """The checked native calls (raises if they were not built)."""
    global _front
    if _front is None:
        if not _ffi.FRONT_PATH.exists():
            raise RuntimeError(f"native front end missing: {_ffi.FRONT_PATH} "
                               "(build it with `python -m blackwell_b200.build`)")
        _ffi.lib()
        front = importlib.import_module("blackwell_b200._front")
        if front.built_with_torch != torch.__version__:
            raise RuntimeError(f"{_ffi.FRONT_PATH} was built with torch {front.built_with_torch}, this is "
                               f"{torch.__version__} (build it again with `python -m blackwell_b200.build`)")
        _front = front
    return _front


def rope_table(length, rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=0, attention_factor=0.0,
               beta_fast=0.0, beta_slow=0.0, low_freq_factor=0.0, high_freq_factor=0.0, first=0, out=None):
    """cos | sin table fp32 [length, rotary_dim] of the positions first .. first + length - 1.

    scaling: "none", "linear" (positions / factor), "ntk" (a larger base), "yarn"
    (low frequencies interpolated, cos and sin times 0.1 ln(factor) + 1) or
    "bands" (interpolated by wavelength against original_length); the schedules'
    formulas and the meaning of 0 are at bw_rope_scaling in include/bw_attn.h."""
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
    if out is None:
        out = torch.empty((length, rotary_dim), dtype=torch.float32,
                          device=torch.device("cuda", torch.cuda.current_device()))
    elif out.shape != (length, rotary_dim):
        raise ValueError(f"out must be [{length}, {rotary_dim}], got {tuple(out.shape)}")
    rc = (_front or _load()).rope_table(out, first, _SCALINGS[scaling], base, factor, original_length, attention_factor,
                                        beta_fast, beta_slow, low_freq_factor, high_freq_factor)
    if rc:
        _ffi.check(rc, "bw_rope_table")
    return out


def _rows_of_16_bytes(t):
    """A gradient as the call takes tensors: autograd hands over expanded and otherwise strided ones."""
    if t is None or (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
            n == 1 or (s > 0 and s * t.element_size() % 16 == 0) for n, s in zip(t.shape[:-1], t.stride()))):
        return t
    return t.contiguous()


class _Rope(torch.autograd.Function):
    """The rotation with its gradient, the inverse rotation of the outputs' gradients."""

    @staticmethod
    def forward(ctx, q, k, cos_sin_cache, positions, pos_offset, interleaved, inverse):
        ctx.save_for_backward(cos_sin_cache, positions)
        ctx.how = pos_offset, interleaved, inverse
        ctx.set_materialize_grads(False)
        return rope(q, k, cos_sin_cache, positions, pos_offset, interleaved, inverse)   # gradients are off here

    @staticmethod
    def backward(ctx, dq, dk):
        (table, positions), (pos_offset, interleaved, inverse) = ctx.saved_tensors, ctx.how
        dq, dk = _rows_of_16_bytes(dq), _rows_of_16_bytes(dk)
        turn = lambda a, b: rope(a, b, table, positions, pos_offset, interleaved, not inverse)  # noqa: E731
        if dq is not None:
            dq, dk = turn(dq, dk)
        elif dk is not None:
            dk, _ = turn(dk, None)
        return dq, dk, None, None, None, None, None


def rope(q, k, cos_sin_cache, positions=None, pos_offset=0, interleaved=False, inverse=False, q_out=None, k_out=None):
    """Rotates the first cos_sin_cache.shape[1] elements of every head of q and k
    (one launch; k may be None) -> (q_out, k_out).

    q, k: bf16 or fp32 [B, H, S, D] views (BHSD, or BSHD through .transpose(1, 2))
    with int32 positions [B, S], or [tokens, H, D] with positions [tokens]; None:
    0, 1, ... along S.  A token whose position + pos_offset is outside the table
    is copied.  interleaved: pairs (2i, 2i + 1) instead of (i, i + R / 2).
    inverse: the transposed rotation, which maps gradients of the outputs to
    gradients of the inputs.  q_out may be q (in place).

    Differentiable in q and k; given outputs, and a table that requires gradients,
    are refused then."""
    given = q_out is not None or k_out is not None
    if q_out is None:
        q_out = torch.empty_like(q)
    if k_out is None and k is not None:
        k_out = torch.empty_like(k)
    rc = (_front or _load()).rope(q, q_out, k, k_out, cos_sin_cache, positions, pos_offset, interleaved, inverse)
    if rc:
        if rc == _WANTS_GRADIENT:
            if cos_sin_cache.requires_grad:
                raise ValueError("no gradient is computed for cos_sin_cache")
            if given:
                raise ValueError("gradients do not pass through given outputs: leave q_out and k_out out, or call under no_grad")
            return _Rope.apply(q, k, cos_sin_cache, positions, pos_offset, interleaved, inverse)
        _ffi.check(rc, "bw_rope")
    return q_out, k_out


def kv_cache_write(k, v, k_cache, v_cache, slots, scales=None, cos_sin_cache=None, positions=None, interleaved=False):
    """Writes new tokens into their slots of a paged cache -> (k_cache, v_cache).

    k, v: bf16 [tokens, Hkv, D] views with a contiguous last dimension (slices of
    one projection's output, say); slots int64 [tokens]: page * page_size + place,
    negative to skip the token; the slots of a call differ.  k_cache, v_cache:
    bf16, or float8_e4m3fn with uint8 scales.  With cos_sin_cache (fp32
    [length, rotary_dim]) and positions (int32 [tokens]) K is rotated on the way."""
    rc = (_front or _load()).kv_cache_write(k, v, k_cache, v_cache, slots, scales, cos_sin_cache, positions, interleaved)
    if rc:
        _ffi.check(rc, "bw_kv_cache_write")
    return k_cache, v_cache


def kv_cache_read(k_cache, v_cache, block_table, kv_lens, out_offsets, scales=None, kv_starts=None, total_rows=None,
                  k_out=None, v_out=None):
    """Reads spans of sequences back as bf16 rows -> (k_out, v_out) [total_rows, Hkv, D].

    block_table int32 [B, max_pages]; tokens [kv_starts[b], kv_starts[b] +
    kv_lens[b]) of sequence b (int32; kv_starts None: from 0) go to the rows
    out_offsets[b] + 0, 1, ... (int64).  Other rows of given outputs are left as
    they are; without outputs give total_rows."""
    if k_out is None or v_out is None:
        if total_rows is None and k_out is None and v_out is None:
            raise ValueError("give k_out and v_out, or total_rows")
        given = k_out if k_out is not None else v_out
        rows = given.shape[0] if given is not None else int(total_rows)
        shape = (rows, *k_cache.shape[2:])
        k_out = torch.empty(shape, dtype=torch.bfloat16, device=k_cache.device) if k_out is None else k_out
        v_out = torch.empty(shape, dtype=torch.bfloat16, device=k_cache.device) if v_out is None else v_out
    if total_rows is not None and k_out.shape[0] != total_rows:
        raise ValueError(f"k_out has {k_out.shape[0]} rows, total_rows is {total_rows}")
    rc = (_front or _load()).kv_cache_read(k_cache, v_cache, block_table, kv_lens, out_offsets, scales, kv_starts, k_out,
                                           v_out)
    if rc:
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
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
    if workspace is None:
        B, Hq, D = q.shape
        workspace = torch.empty(decode_fp8_workspace_size(B, Hq, k_cache.shape[2], D), dtype=torch.uint8,
                                device=q.device)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    rc = (_front or _load()).gqa_decode_paged_fp8(q, k_cache, v_cache, scales, block_table, kv_lens, scale, workspace,
                                                  out, lse)
    if rc:
        _ffi.check(rc, "bw_gqa_decode_paged_fp8")
    return out, lse
