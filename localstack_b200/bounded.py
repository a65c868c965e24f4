"""Attention over a bounded cache: sliding window with sinks, and decode with accumulated weights.

A service that runs past its cache's budget keeps a few first tokens (sinks) and a recent window
(attn_decode_window, attn_prefill_window), or the keys that the queries so far have attended to most:
attn_decode_weights adds each key's softmax weights to a row of accumulated weights, and evict.py
drops the keys whose sums are smallest. Everything works on the paged cache of attn.py (f16) or q8.py
(q8_0 planes); the reference has no counterpart (its cache is full when its cells are used up,
src/kv_cache.cpp:59-83).
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import check, lib
from .attn import _DT, HEAD_DIM, DecodeWorkspace, _p, _stream, layout_of
from .q8 import Q8Cache

_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_OUT_DTYPES = (torch.float32, torch.bfloat16)


class WeightsWorkspace:
    """Caller-owned scratch for attn_decode_weights (lstk_cuda_attn_decode_weights_workspace_size):
    the decode's, and the scores of one step over sequences of up to max_seq_len keys."""

    def __init__(self, n_seqs, n_head, n_head_kv, max_seq_len, device="cuda"):
        nbytes = lib().lstk_cuda_attn_decode_weights_workspace_size(n_seqs, n_head, n_head_kv, HEAD_DIM, max_seq_len)
        self.buf = torch.empty(nbytes, dtype=torch.uint8, device=device)


def _decode_args(q, block_tables, seq_lens, out, out_dtype, want_lse, lse_out):
    """Checks the shapes a decode call relies on; returns (B, Hq, out, lse_out), allocated when None."""
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.dtype not in (torch.float16, torch.float32):
        raise ValueError("q must be f16 or f32 [B][Hq][128]")
    B, Hq, _ = q.shape
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block_tables and seq_lens must be int32")
    if block_tables.dim() != 2 or block_tables.shape[0] != B or seq_lens.numel() != B:
        raise ValueError("block_tables must be [B][max_blocks] and seq_lens [B]")
    if not (q.is_contiguous() and block_tables.is_contiguous() and seq_lens.is_contiguous()):
        raise ValueError("q, block_tables and seq_lens must be contiguous")
    if out is None:
        if out_dtype not in _OUT_DTYPES:
            raise ValueError("out_dtype must be float32 or bfloat16")
        out = torch.empty((B, Hq, HEAD_DIM), dtype=out_dtype, device=q.device)
    elif out.dtype not in _OUT_DTYPES or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be a contiguous f32 or bf16 tensor of q's shape")
    if lse_out is None:
        if want_lse:
            lse_out = torch.empty((B, Hq), dtype=torch.float32, device=q.device)
    elif lse_out.dtype != torch.float32 or lse_out.shape != (B, Hq) or not lse_out.is_contiguous():
        raise ValueError("lse_out must be a contiguous f32 [B][Hq] tensor")
    return B, Hq, out, lse_out


def _planes(kq, vq):
    if kq.qs.shape != vq.qs.shape:
        raise ValueError("the K and V caches must have the same shape")
    return kq.layout, (_p(kq.qs), _p(kq.d), _p(vq.qs), _p(vq.d)), kq.qs.device


def _caches(k_cache, v_cache):
    if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or not v_cache.is_contiguous():
        raise ValueError("the K and V caches must have the same shape")
    return layout_of(k_cache), (_p(k_cache), _p(v_cache)), k_cache.device


def _decode_window(fn, layout, cache, device, q, block_tables, seq_lens, window, n_sink, scale, max_seq_len, out,
                   out_dtype, lse_out, want_lse, workspace, n_ctas, stream):
    B, Hq, out, lse_out = _decode_args(q, block_tables, seq_lens, out, out_dtype, want_lse, lse_out)
    if workspace is None or workspace.n_seqs < B:
        workspace = DecodeWorkspace(B, Hq, layout.n_head_kv, q.device)
    check(fn(ctypes.byref(layout), *cache, _p(q), _DT[q.dtype], B, Hq, _p(block_tables), block_tables.shape[1],
             _p(seq_lens), int(max_seq_len), int(window), int(n_sink), _SCALE if scale is None else float(scale),
             _p(out), _DT[out.dtype], _p(lse_out), _p(workspace.buf), workspace.buf.numel(), int(n_ctas),
             _stream(stream, device)))
    return (out, lse_out) if want_lse else out


def attn_decode_window(k_cache, v_cache, q, block_tables, seq_lens, window, n_sink=0, scale=None, max_seq_len=0,
                       out=None, out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0,
                       stream=None):
    """attn_decode restricted to a sliding window and sinks: sequence b's query, at position
    seq_lens[b] - 1, sees its last `window` keys (its own among them) and its first `n_sink`.

    Only the visible keys' pages are read. out (or out_dtype) is f32 or bf16; lse covers the visible
    keys. Other arguments as attn_decode."""
    layout, cache, device = _caches(k_cache, v_cache)
    return _decode_window(lib().lstk_cuda_attn_decode_window, layout, cache, device, q, block_tables, seq_lens,
                          window, n_sink, scale, max_seq_len, out, out_dtype, lse_out, want_lse, workspace, n_ctas,
                          stream)


def attn_decode_window_q8(kq: Q8Cache, vq: Q8Cache, q, block_tables, seq_lens, window, n_sink=0, scale=None,
                          max_seq_len=0, out=None, out_dtype=torch.float32, lse_out=None, want_lse=False,
                          workspace=None, n_ctas=0, stream=None):
    """attn_decode_window over q8_0 planes: attn_decode_q8's semantics, the query's block scale taken as
    amax * (1 / 127) in f32 (its last bit may differ from the quotient's)."""
    layout, cache, device = _planes(kq, vq)
    return _decode_window(lib().lstk_cuda_attn_decode_window_q8, layout, cache, device, q, block_tables, seq_lens,
                          window, n_sink, scale, max_seq_len, out, out_dtype, lse_out, want_lse, workspace, n_ctas,
                          stream)


def _decode_weights(fn, layout, cache, device, q, block_tables, seq_lens, acc, scale, max_seq_len, out, out_dtype,
                    lse_out, want_lse, workspace, n_ctas, stream):
    B, Hq, out, lse_out = _decode_args(q, block_tables, seq_lens, out, out_dtype, want_lse, lse_out)
    if acc.dtype != torch.float32 or acc.dim() != 2 or acc.shape[0] != B or acc.stride(1) != 1:
        raise ValueError("acc must be f32 [B][cells] with contiguous rows")
    if B > 1 and acc.stride(0) < acc.shape[1]:
        raise ValueError("the rows of acc must not overlap")
    cells = block_tables.shape[1] * 32
    max_seq_len = int(max_seq_len) if 0 < max_seq_len <= cells else cells
    if acc.shape[1] < max_seq_len:
        raise ValueError("a row of acc must hold max_seq_len keys (0: every key of a block table)")
    if workspace is None:
        workspace = WeightsWorkspace(B, Hq, layout.n_head_kv, max_seq_len, q.device)
    check(fn(ctypes.byref(layout), *cache, _p(q), _DT[q.dtype], B, Hq, _p(block_tables), block_tables.shape[1],
             _p(seq_lens), max_seq_len, _SCALE if scale is None else float(scale), _p(acc),
             acc.stride(0) if B > 1 else acc.shape[1], _p(out), _DT[out.dtype], _p(lse_out), _p(workspace.buf),
             workspace.buf.numel(), int(n_ctas), _stream(stream, device)))
    return (out, lse_out) if want_lse else out


def attn_decode_weights(k_cache, v_cache, q, block_tables, seq_lens, acc, scale=None, max_seq_len=0, out=None,
                        out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0, stream=None):
    """attn_decode that also adds every visible key's softmax weights, summed over the query heads, to
    acc[b][i] (f32 [B][>= max_seq_len], updated in place; entries at or past a sequence's length keep
    their values). out (or out_dtype) is f32 or bf16. `workspace` is a WeightsWorkspace for at least
    these sizes; a sequence longer than max_seq_len (0: the block table's cells) reports an index
    status and attends to its first max_seq_len keys. Other arguments as attn_decode."""
    layout, cache, device = _caches(k_cache, v_cache)
    return _decode_weights(lib().lstk_cuda_attn_decode_weights, layout, cache, device, q, block_tables, seq_lens, acc,
                           scale, max_seq_len, out, out_dtype, lse_out, want_lse, workspace, n_ctas, stream)


def attn_decode_weights_q8(kq: Q8Cache, vq: Q8Cache, q, block_tables, seq_lens, acc, scale=None, max_seq_len=0,
                           out=None, out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0,
                           stream=None):
    """attn_decode_weights over q8_0 planes, with attn_decode_window_q8's semantics."""
    layout, cache, device = _planes(kq, vq)
    return _decode_weights(lib().lstk_cuda_attn_decode_weights_q8, layout, cache, device, q, block_tables, seq_lens,
                           acc, scale, max_seq_len, out, out_dtype, lse_out, want_lse, workspace, n_ctas, stream)


def _prefill_args(layout, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, out, out_dtype, workspace):
    """Checks the shapes a prefill call relies on; returns (total, Hq, B, out, workspace), allocated when None."""
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.dtype not in (torch.float16, torch.float32) or not q.is_contiguous():
        raise ValueError("q must be a contiguous f16 or f32 tensor [total_tokens][Hq][128]")
    total, Hq, _ = q.shape
    B = q_pos0.numel()
    for name, t in (("q_seq_start", q_seq_start), ("q_pos0", q_pos0), ("kv_lens", kv_lens),
                    ("block_tables", block_tables)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")
    if q_seq_start.numel() != B + 1 or kv_lens.numel() != B or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("q_seq_start [B+1], q_pos0 / kv_lens [B] and block_tables [B][max_blocks] must agree")
    if out is None:
        if out_dtype not in _OUT_DTYPES:
            raise ValueError("out_dtype must be float32 or bfloat16")
        out = torch.empty((total, Hq, HEAD_DIM), dtype=out_dtype, device=q.device)
    elif out.dtype not in _OUT_DTYPES or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be a contiguous f32 or bf16 tensor of q's shape")
    if q.dtype == torch.float32:  # the f16 copy of q lives in the workspace; f16 queries need none
        need = lib().lstk_cuda_attn_prefill_workspace_size(B, Hq, layout.n_head_kv, HEAD_DIM, int(max_q_len),
                                                           block_tables.shape[1], total, _DT[q.dtype])
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=q.device)
    return total, Hq, B, out, workspace


def attn_prefill_window(k_cache, v_cache, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window, n_sink=0,
                        scale=None, out=None, out_dtype=torch.float32, workspace=None, stream=None):
    """attn_prefill restricted to a sliding window and sinks: the query at position p sees its last
    `window` keys up to p (its own among them) and the first `n_sink`, all below kv_lens.

    Tiles that no query sees are neither read nor computed. out (or out_dtype) is f32 or bf16; a query
    that sees no key gets zeros. Other arguments as attn_prefill."""
    layout, cache, device = _caches(k_cache, v_cache)
    total, Hq, B, out, workspace = _prefill_args(layout, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, out,
                                                 out_dtype, workspace)
    check(lib().lstk_cuda_attn_prefill_window(
        ctypes.byref(layout), *cache, _p(q), _DT[q.dtype], B, Hq, _p(q_seq_start), int(max_q_len), total, _p(q_pos0),
        _p(kv_lens), _p(block_tables), block_tables.shape[1], int(window), int(n_sink),
        _SCALE if scale is None else float(scale), _p(out), _DT[out.dtype], _p(workspace),
        workspace.numel() if workspace is not None else 0, _stream(stream, device)))
    return out


def attn_prefill_window_q8(kq: Q8Cache, vq: Q8Cache, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window,
                           n_sink=0, scale=None, out=None, out_dtype=torch.float32, workspace=None, scratch=None,
                           stream=None):
    """attn_prefill_window over q8_0 planes: the pages that some query sees are dequantised into
    `scratch` (uint8 of lstk_cuda_q8_prefill_scratch_size bytes, allocated when None) and the
    tensor-core prefill runs on it, as attn_prefill_q8 does."""
    layout, cache, device = _planes(kq, vq)
    total, Hq, B, out, workspace = _prefill_args(layout, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, out,
                                                 out_dtype, workspace)
    need = lib().lstk_cuda_q8_prefill_scratch_size(B, block_tables.shape[1], layout.n_head_kv)
    if scratch is None or scratch.numel() < need:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    check(lib().lstk_cuda_attn_prefill_window_q8(
        ctypes.byref(layout), *cache, _p(q), _DT[q.dtype], B, Hq, _p(q_seq_start), int(max_q_len), total, _p(q_pos0),
        _p(kv_lens), _p(block_tables), block_tables.shape[1], int(window), int(n_sink),
        _SCALE if scale is None else float(scale), _p(out), _DT[out.dtype], _p(workspace),
        workspace.numel() if workspace is not None else 0, _p(scratch), scratch.numel(), _stream(stream, device)))
    return out
