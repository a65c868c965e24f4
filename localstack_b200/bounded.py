"""Attention over a bounded cache: sliding window with sinks, and decode with accumulated weights.

A service that runs past its cache's budget keeps a few first tokens (sinks) and a recent window
(attn_decode_window, attn_prefill_window), or the keys that the queries so far have attended to most:
attn_decode_weights adds each key's softmax weights to a row of accumulated weights, and evict.py
drops the keys whose sums are smallest. Everything works on the paged cache of attn.py (f16) or q8.py
(q8_0 planes); the reference has no counterpart (its cache is full when its cells are used up,
src/kv_cache.cpp:59-83).
"""
from __future__ import annotations

import torch

from ._lib import check, host, lib
from .attn import _DT, HEAD_DIM
from .q8 import Q8Cache


class WeightsWorkspace:
    """Caller-owned scratch for attn_decode_weights (lstk_cuda_attn_decode_weights_workspace_size):
    the decode's, and the scores of one step over sequences of up to max_seq_len keys."""

    def __init__(self, n_seqs, n_head, n_head_kv, max_seq_len, device="cuda"):
        nbytes = lib().lstk_cuda_attn_decode_weights_workspace_size(n_seqs, n_head, n_head_kv, HEAD_DIM, max_seq_len)
        self.buf = torch.empty(nbytes, dtype=torch.uint8, device=device)


def _buf(workspace):
    return None if workspace is None else workspace.buf


def attn_decode_window(k_cache, v_cache, q, block_tables, seq_lens, window, n_sink=0, scale=None, max_seq_len=0,
                       out=None, out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0,
                       stream=None):
    """attn_decode restricted to a sliding window and sinks: sequence b's query, at position
    seq_lens[b] - 1, sees its last `window` keys (its own among them) and its first `n_sink`.

    Only the visible keys' pages are read. out (or out_dtype) is f32 or bf16; lse covers the visible
    keys. `workspace` is a DecodeWorkspace. Other arguments as attn_decode."""
    rc, out, lse_out = host().window(k_cache, None, v_cache, None, q, block_tables, seq_lens, window, n_sink, scale,
                                     max_seq_len, out, out_dtype, lse_out, want_lse, _buf(workspace), n_ctas, stream)
    if rc:
        check(rc)
    return (out, lse_out) if want_lse else out


def attn_decode_window_q8(kq: Q8Cache, vq: Q8Cache, q, block_tables, seq_lens, window, n_sink=0, scale=None,
                          max_seq_len=0, out=None, out_dtype=torch.float32, lse_out=None, want_lse=False,
                          workspace=None, n_ctas=0, stream=None):
    """attn_decode_window over q8_0 planes: attn_decode_q8's semantics, the query's block scale taken as
    amax * (1 / 127) in f32 (its last bit may differ from the quotient's)."""
    rc, out, lse_out = host().window(kq.qs, kq.d, vq.qs, vq.d, q, block_tables, seq_lens, window, n_sink, scale,
                                     max_seq_len, out, out_dtype, lse_out, want_lse, _buf(workspace), n_ctas, stream)
    if rc:
        check(rc)
    return (out, lse_out) if want_lse else out


def attn_decode_weights(k_cache, v_cache, q, block_tables, seq_lens, acc, scale=None, max_seq_len=0, out=None,
                        out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0, stream=None):
    """attn_decode that also adds every visible key's softmax weights, summed over the query heads, to
    acc[b][i] (f32 [B][>= max_seq_len], updated in place; entries at or past a sequence's length keep
    their values). out (or out_dtype) is f32 or bf16. `workspace` is a WeightsWorkspace for at least
    these sizes; a sequence longer than max_seq_len (0: the block table's cells) reports an index
    status and attends to its first max_seq_len keys. Other arguments as attn_decode."""
    rc, out, lse_out = host().weights(k_cache, None, v_cache, None, q, block_tables, seq_lens, acc, scale, max_seq_len,
                                      out, out_dtype, lse_out, want_lse, _buf(workspace), n_ctas, stream)
    if rc:
        check(rc)
    return (out, lse_out) if want_lse else out


def attn_decode_weights_q8(kq: Q8Cache, vq: Q8Cache, q, block_tables, seq_lens, acc, scale=None, max_seq_len=0,
                           out=None, out_dtype=torch.float32, lse_out=None, want_lse=False, workspace=None, n_ctas=0,
                           stream=None):
    """attn_decode_weights over q8_0 planes, with attn_decode_window_q8's semantics."""
    rc, out, lse_out = host().weights(kq.qs, kq.d, vq.qs, vq.d, q, block_tables, seq_lens, acc, scale, max_seq_len, out,
                                      out_dtype, lse_out, want_lse, _buf(workspace), n_ctas, stream)
    if rc:
        check(rc)
    return (out, lse_out) if want_lse else out


def prefill_window_workspace_bytes(q, n_head_kv, max_q_len, block_tables, window, n_sink=0):
    """Bytes of workspace with which attn_prefill_window splits a call of these shapes along the keys where
    that pays (on the current device)."""
    total, Hq, _ = q.shape
    return lib().lstk_cuda_attn_prefill_window_workspace_size(
        block_tables.shape[0], Hq, n_head_kv, HEAD_DIM, int(max_q_len), block_tables.shape[1], total, _DT[q.dtype],
        int(window), int(n_sink))


def attn_prefill_window(k_cache, v_cache, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window, n_sink=0,
                        scale=None, out=None, out_dtype=torch.float32, workspace=None, stream=None):
    """attn_prefill restricted to a sliding window and sinks: the query at position p sees its last
    `window` keys up to p (its own among them) and the first `n_sink`, all below kv_lens.

    Tiles that no query sees are neither read nor computed. out (or out_dtype) is f32 or bf16; a query
    that sees no key gets zeros. workspace: uint8, None to allocate one that lets few queries behind long
    contexts be split over the SMs (prefill_window_workspace_bytes); a smaller one, of at least
    lstk_cuda_attn_prefill_workspace_size bytes, runs unsplit. Other arguments as attn_prefill."""
    rc, out = host().prefill(k_cache, None, v_cache, None, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len,
                             window, n_sink, scale, out, out_dtype, workspace, None, stream)
    if rc:
        check(rc)
    return out


def attn_prefill_window_q8(kq: Q8Cache, vq: Q8Cache, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window,
                           n_sink=0, scale=None, out=None, out_dtype=torch.float32, workspace=None, scratch=None,
                           stream=None):
    """attn_prefill_window over q8_0 planes: the pages that some query sees are dequantised into
    `scratch` (uint8 of lstk_cuda_q8_prefill_scratch_size bytes, allocated when None) and the
    tensor-core prefill runs on it, as attn_prefill_q8 does."""
    rc, out = host().prefill(kq.qs, kq.d, vq.qs, vq.d, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window,
                             n_sink, scale, out, out_dtype, workspace, scratch, stream)
    if rc:
        check(rc)
    return out
