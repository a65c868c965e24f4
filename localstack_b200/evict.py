"""Eviction from the paged cache by accumulated attention weight (lstk_kv_weights,
include/lstk_cuda_attn.h).

A serving loop adds up what each cached key receives (bounded.attn_decode_weights on KvWeights.acc),
and when rows have grown past their budget drops the keys with the smallest sums:

    moves = weights.select(pages.seq_lens, budget, n_sink, n_recent)   # which keys stay
    for k, v in layers: kv_move(k, v, pages.block_tables, moves)        # their K and V rows
    weights.finish(pages, moves)                                        # lengths, blocks, acc, positions

Only the queries given to attn_decode_weights add up. A prompt's prefill (attn_prefill, attn_prefill_window)
leaves its keys at zero, and select ranks keys of equal weight by index alone, so a prompt that is to be cut
needs weights first: give its last R queries to attn_decode_weights as R rows with the slot's block table
repeated, seq_lens = their positions + 1 and an acc row of zeros each, and add the rows' sum to the slot's acc:

    attn_decode_weights(k, v, q[-R:], table.expand(R, -1).contiguous(), positions + 1, rows)
    weights.acc[slot, :rows.shape[1]] += rows.sum(0)

A sequence is removed, or its newest tokens are taken back, by weights.release(pages, slot, keep):
DevicePages.release alone leaves the row's weights and positions to the tokens that come after.

The reference has no counterpart: its cache is full when its cells are used up
(src/kv_cache.cpp:59-83).
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass

import torch

from ._lib import KvWeightsState, check, host, lib
from .attn import _p, _stream
from .q8 import Q8Cache

BLOCK = 32


@dataclass
class KvMoves:
    """The moves of one eviction: row b's key at index src[b][j] goes to index dst[b][j], j < n[b]; entries
    behind them are -1. int32 device tensors [rows], [rows][max_moves], [rows][max_moves]."""

    n: torch.Tensor
    src: torch.Tensor
    dst: torch.Tensor
    budget: int


class KvWeights:
    """Accumulated weights and token positions of the cached keys of n_rows slots (one row per slot of a
    DevicePages of max_blocks blocks a slot), zero for new sequences.

    acc f32 [n_rows][cells]: pass it to attn_decode_weights. pos int32 [n_rows][cells], held and shift
    int32 [n_rows]: the key at index i is the token at position pos[i] (i < held) or i + shift."""

    def __init__(self, n_rows, max_blocks, device="cuda"):
        cells = max_blocks * BLOCK
        self._set(torch.zeros((n_rows, cells), dtype=torch.float32, device=device),
                  torch.zeros((n_rows, cells), dtype=torch.int32, device=device),
                  torch.zeros(n_rows, dtype=torch.int32, device=device),
                  torch.zeros(n_rows, dtype=torch.int32, device=device))

    @classmethod
    def from_tensors(cls, acc, pos, held, shift):
        """A state over existing tensors (no copy)."""
        if acc.dtype != torch.float32 or acc.dim() != 2:
            raise ValueError("acc must be f32 [rows][cells]")
        if any(t.dtype != torch.int32 for t in (pos, held, shift)):
            raise ValueError("pos, held and shift must be int32")
        if pos.shape != acc.shape or held.shape != acc.shape[:1] or shift.shape != acc.shape[:1]:
            raise ValueError("pos must be [rows][cells], held and shift [rows]")
        if any(not t.is_contiguous() or t.device != acc.device for t in (acc, pos, held, shift)):
            raise ValueError("acc, pos, held and shift must be contiguous, on one device")
        w = cls.__new__(cls)
        w._set(acc, pos, held, shift)
        return w

    def _set(self, acc, pos, held, shift):
        self.acc, self.pos, self.held, self.shift = acc, pos, held, shift
        self.n_rows, self.row_cells = acc.shape
        self.device = acc.device
        self.state = KvWeightsState(acc.data_ptr(), pos.data_ptr(), held.data_ptr(), shift.data_ptr(), self.n_rows,
                                    self.row_cells)

    def select(self, seq_lens, budget, n_sink=0, n_recent=0, moves=None, stream=None):
        """The moves that hold every row to `budget` keys: tokens at positions < n_sink and the last
        n_recent stay, then the largest acc (lower index first among equal ones). Rows at or below the
        budget have none. `moves` (an earlier result for the same sizes) is written again if given."""
        budget = int(budget)
        given = (None, None, None) if moves is None else (moves.n, moves.src, moves.dst)
        rc, n, src, dst = host().select(self.acc, self.pos, self.held, self.shift, seq_lens, budget, n_sink, n_recent,
                                        *given, stream)
        if rc:
            check(rc)
        if moves is None:
            return KvMoves(n, src, dst, budget)
        moves.budget = budget
        return moves

    def finish(self, pages, moves, stream=None):
        """Ends an eviction: acc and pos follow the moves, the rows of `pages` (a DevicePages) are
        truncated to the budget and their blocks freed. Call it once, after every layer's kv_move."""
        if moves.n.shape != (self.n_rows,) or moves.src.shape[0] != self.n_rows or moves.dst.shape != moves.src.shape:
            raise ValueError("moves and weights must have the same rows")
        if any(t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.device
               for t in (moves.n, moves.src, moves.dst)):
            raise ValueError("moves must be contiguous int32 tensors on the weights' device")
        if pages.device != self.device:
            raise ValueError("pages and weights must be on one device")
        check(lib().lstk_cuda_kv_evict_finish(ctypes.byref(pages.state), ctypes.byref(self.state), moves.budget,
                                              _p(moves.n), _p(moves.src), _p(moves.dst), moves.src.shape[1],
                                              _stream(stream, self.device)))

    def positions(self, positions, slots):
        """Token positions (for kv_append's RoPE) of new tokens that DevicePages.alloc placed at
        `positions`, one slot index per token."""
        return positions + self.shift[slots.long()]

    def reset(self, slot):
        """Clears the row of a removed sequence, on the current stream."""
        self.acc[slot].zero_()
        self.held[slot].zero_()
        self.shift[slot].zero_()

    def release(self, pages, slot, keep=0, stream=None):
        """pages.release(slot, keep) together with the row: keep <= 0 removes the sequence and clears the row;
        else the first `keep` keys stay and the weights behind them are cleared (a token appended there later
        would start with another token's weight).

        The keys below held[slot] are in no order of tokens, so a cut among them would drop arbitrary ones:
        ValueError, nothing changed (remove the sequence instead). For keep > 0 held[slot] is read back, which
        waits for the stream: such a call cannot be captured into a graph."""
        slot, keep = int(slot), int(keep)
        if not 0 <= slot < self.n_rows:
            raise ValueError("slot out of range")
        if pages.device != self.device:
            raise ValueError("pages and weights must be on one device")
        with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
            if keep > 0 and keep < int(self.held[slot]):
                raise ValueError("keep is below held: the row's keys are not in token order there")
            pages.release(slot, keep, stream)
            if keep > 0:
                self.acc[slot, keep:].zero_()
            else:
                self.reset(slot)


def kv_move(k_cache, v_cache, block_tables, moves: KvMoves, stream=None):
    """Carries out an eviction's moves on one layer's K and V caches (f16 [n_cells][n_head_kv][128])."""
    (rc,) = host().move(k_cache, None, v_cache, None, block_tables, moves.n, moves.src, moves.dst, stream)
    if rc:
        check(rc)


def kv_move_q8(kq: Q8Cache, vq: Q8Cache, block_tables, moves: KvMoves, stream=None):
    """kv_move on q8_0 planes."""
    (rc,) = host().move(kq.qs, kq.d, vq.qs, vq.d, block_tables, moves.n, moves.src, moves.dst, stream)
    if rc:
        check(rc)
