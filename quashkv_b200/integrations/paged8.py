"""A paged KV cache in 8 bits, and block tables that live on the device.

``QuashKVPaged8Cache`` stands beside ``QuashKVPagedCache`` (vllm_backend.py): the same pool of pages, block tables and
calls, with one byte a coordinate (e4m3 or int8) and one scale for each page and KV head, for keys and for values, in
place of rotated 2- to 4-bit codes.  It takes 2.5 times the memory and is the format for what 3 bits cost too much.

``PageTables`` keeps tables, lengths and the stack of free pages in device memory: a step of a serving loop (extend,
append, attention) then has no host loop and no copy, and can be captured into a CUDA graph.  Its tables serve both caches.

The functions are the same operators over tensors that the caller owns:

    plan = extend_pages(block_table, seq_lens, new_lens, free_pages, pool, block_size, max_tokens)
    append_paged8(keys, values, k_codes, v_codes, k_scales, v_scales, plan.slots)
    out = attention_paged8(queries, k_codes, v_codes, k_scales, v_scales, block_table, plan.seq_lens, max_kv_len,
                           causal=True, query_starts=plan.query_starts, max_q_len=max_q_len, start_lens=seq_lens)

The reference stops before real pages (quashkv/integrations/vllm_backend.py:82-195).  Only CUDA tensors are accepted;
there is no CPU implementation, and nothing here has a derivative.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence

import torch

from .. import _lib, ops
from .vllm_backend import PagePool

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class PagePlan(NamedTuple):
    """What ``extend_pages`` decides, as new tensors: the pool's lengths and counts after the call are in it."""
    slots: torch.Tensor          # (max_tokens) int64: block * block_size + offset of each new token, -1 where it has none
    query_starts: torch.Tensor   # (n_seq + 1) int32: first new token of each sequence
    seq_lens: torch.Tensor       # (n_seq) int32: tokens held after the call
    pool: torch.Tensor           # (2) int32: free pages, tokens that found no place so far


class StepPlan(NamedTuple):
    """What ``PageTables.extend`` decides; lengths and counts have been updated in place."""
    slots: torch.Tensor          # as in PagePlan
    query_starts: torch.Tensor
    start_lens: torch.Tensor     # (n_seq) int32: tokens held before the call


def extend_pages(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                 pool: torch.Tensor, block_size: int, max_tokens: int) -> PagePlan:
    """Pages and slots for ``new_lens`` (n_seq) more tokens of every sequence.

    ``block_table`` (n_seq, max_blocks) gets the new pages behind the ceil(seq_lens / block_size) that a sequence has;
    ``free_pages`` is a stack of which the first ``pool[0]`` are free, taken from the top in the order of the sequences.
    All int32.  ``max_tokens`` (known on the host) is at least the sum of ``new_lens``: the new tokens of all sequences one
    after the other, as a model computes them.  Tokens for which the stack or the row of the table is too short get slot
    -1, are not counted in ``seq_lens``, and are added to ``pool[1]``; they are the last ones of their sequence, and causal
    attention of the others needs ``start_lens`` then (see ``attention_paged8``).  Lengths and counts are returned and not changed, so
    that a plan can be dropped; ``PageTables.extend`` changes them in place."""
    ops._need_cuda(block_table, "extend_pages")
    return PagePlan(*ops.extend_pages(block_table, seq_lens, new_lens, free_pages, pool, block_size, max_tokens))


def append_paged8(keys: torch.Tensor, values: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                  k_scales: torch.Tensor, v_scales: torch.Tensor, slots: Optional[torch.Tensor] = None,
                  block_table: Optional[torch.Tensor] = None, start_lens: Optional[torch.Tensor] = None) -> None:
    """Quantise keys and values into their pages.

    ``keys``, ``values``: (tokens, kv_heads, head_size) with ``slots`` (tokens) int64, a negative one for a token that is
    not stored; or (n_seq, kv_heads, tokens, head_size) with ``block_table`` and ``start_lens``, the position of each
    sequence's first token.  Any strides.  ``*_codes`` (num_blocks, kv_heads, block_size, head_size), a view in any memory
    order whose tokens are contiguous, float8_e4m3fn or int8; ``*_scales`` (num_blocks, kv_heads) fp32.

    Consecutive tokens with consecutive slots in one page form a run.  Its scale is the least power of two with which
    its largest magnitude is no more than the largest code (448 or 127); the page takes it where the run begins the page, else the larger
    of it and the page's own, and the codes in front of the run are rounded to the new scale.  An infinity or a NaN makes the scale of
    its page and head NaN.  The tokens of one page have to form ONE run of a call: a page that gets two (a slot listed
    twice among them) is left with either's scale.  Slots outside the pool and positions outside the table are dropped
    and counted (``dropped_tokens``)."""
    ops._need_cuda(keys, "append_paged8")
    ops.append_paged8(keys, values, k_codes, v_codes, k_scales, v_scales, slots, block_table, start_lens)


def dropped_tokens() -> int:
    """(Token, head) pairs that appends on the current device could not store.  Waits for the device."""
    return int(_lib.lib().qkv_dropped_paged8_tokens())


def attention_paged8(queries: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor,
                     v_scales: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, max_kv_len: int,
                     scale: Optional[float] = None, causal: bool = False, query_starts: Optional[torch.Tensor] = None,
                     max_q_len: Optional[int] = None, start_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over pages of 8-bit codes; the result has the queries' shape and their type: fp32, bf16 or
    fp16.  Queries of any other type, fp64 among them, are taken as fp32 and give fp32.

    ``queries``: (n_seq, q_heads, q_len, head_size), or with ``query_starts`` (n_seq + 1) int32 a ragged batch (tokens,
    q_heads, head_size) whose tokens query_starts[i] .. query_starts[i + 1] - 1 are sequence i's, at most ``max_q_len``
    of them (default: as many as there are).  Query head h reads KV head h // (q_heads // kv_heads).  ``seq_lens`` (n_seq)
    int32 with ``max_kv_len`` an upper bound of them known on the host.  With ``causal`` a query sees the positions up to its
    own: the queries of a sequence are its last positions, or, with ``start_lens`` (n_seq) int32 (the lengths before the
    step), query t is at start_lens + t.  The two are the same where every new token has found a place; where some have not,
    only the second is right, and a query whose own token has none sees the tokens that the sequence holds.  Rows that see
    nothing, and rows of no sequence, are zeros.

    Scales are 0 or more, or NaN, which reaches what sees the page; a value scale below 2^-126 counts as 0 (appends make none below
    2^-120).  Codes must not hold NaN within a sequence's length, and may be anything behind it.  A block number outside the pool
    hides its tokens."""
    ops._need_cuda(queries, "attention_paged8")
    if scale is None:
        scale = 1.0 / math.sqrt(queries.shape[-1])
    if query_starts is None:
        max_q_len = 0
    elif max_q_len is None:
        max_q_len = queries.shape[0]
    return ops.attention_paged8(queries, k_codes, v_codes, k_scales, v_scales, block_table, seq_lens, int(max_kv_len),
                                query_starts, int(max_q_len), float(scale), bool(causal), start_lens)


class PageTables:
    """Block tables, lengths and free pages of up to ``max_seqs`` sequences (rows) in device memory.

    ``block_table`` (max_seqs, max_blocks), ``seq_lens`` (max_seqs), ``free_pages`` (num_blocks) and ``pool`` (2: free
    pages, tokens refused) are int32 tensors that the calls update in place, on the current stream: no host copy, so that
    a step can be captured into a CUDA graph and replayed with other ``new_lens``."""

    def __init__(self, num_blocks: int, max_seqs: int, max_blocks: int, block_size: int = 16, device="cuda"):
        if min(num_blocks, max_seqs, max_blocks, block_size) < 1:
            raise ValueError("num_blocks, max_seqs, max_blocks and block_size must be positive")
        if max_seqs > _lib.PAGES_MAX_SEQS:
            raise ValueError(f"at most {_lib.PAGES_MAX_SEQS} sequences")
        self.num_blocks, self.block_size = num_blocks, block_size
        self.device = torch.device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.block_table = torch.zeros((max_seqs, max_blocks), **i32)
        self.seq_lens = torch.zeros((max_seqs,), **i32)
        self.free_pages = torch.arange(num_blocks - 1, -1, -1, **i32)        # block 0 goes out first
        self.pool = torch.tensor([num_blocks, 0], **i32)

    def extend(self, new_lens: torch.Tensor, max_tokens: int) -> StepPlan:
        """Pages for ``new_lens`` (max_seqs) int32 more tokens, 0 for rows that get none (see ``extend_pages``).  Give the plan's
        ``start_lens`` to causal attention, so that it is right for a row that did not get all of its tokens, too (``QuashKVPagedCache`` takes
        none: there the queries of such a row are not at their positions)."""
        ops._need_cuda(new_lens, "PageTables.extend")
        return StepPlan(*ops.extend_pages_(self.block_table, self.seq_lens, new_lens, self.free_pages, self.pool,
                                           self.block_size, int(max_tokens)))

    def shrink(self, keep_lens: torch.Tensor) -> None:
        """Keep the first ``keep_lens`` (max_seqs) int32 tokens of every row (never more than it has) and return the
        pages behind them: 0 ends a request, fewer tokens take back rejected drafts."""
        ops._need_cuda(keep_lens, "PageTables.shrink")
        ops.shrink_pages_(self.block_table, self.seq_lens, keep_lens, self.free_pages, self.pool, self.block_size)

    def release(self, rows: torch.Tensor) -> None:
        """End the requests of ``rows`` (max_seqs, bool): their pages go back."""
        self.shrink(torch.where(rows, torch.zeros_like(self.seq_lens), self.seq_lens))

    def free_blocks(self) -> int:
        """Pages on the stack.  Waits for the device."""
        return int(self.pool[0])

    def refused_tokens(self) -> int:
        """Tokens that found no place since the tables were made.  Waits for the device."""
        return int(self.pool[1])


class QuashKVPaged8Cache(PagePool):
    """A pool of 8-bit KV pages shared by many sequences of one attention layer.

    ``codes`` is "e4m3" or "int8"; ``layout`` "hnd" keeps a page's tokens of one head together, "nhd" a token's heads.
    ``k_codes`` / ``v_codes`` are (num_blocks, num_kv_heads, block_size, head_size) in both, ``k_scales`` / ``v_scales``
    (num_blocks, num_kv_heads); coordinate = code * scale.  ``block_size`` is a multiple of 16, ``head_size`` 32, 64, 96
    or 128.  Attention returns the queries' type (see ``attention_paged8``)."""

    def __init__(self, num_blocks: int, num_kv_heads: int, head_size: int, block_size: int = 16, codes: str = "e4m3",
                 layout: str = "hnd", device="cuda"):
        super().__init__(num_blocks, num_kv_heads, head_size, block_size, device)
        if codes not in CODES or layout not in ("hnd", "nhd"):
            raise ValueError(f"codes {codes!r} and layout {layout!r}: expected one of {sorted(CODES)} and 'hnd' or 'nhd'")
        if block_size % 16 != 0 or head_size not in (32, 64, 96, 128):
            raise ValueError(f"block_size {block_size} must be a multiple of 16 and head_size {head_size} one of 32, 64, 96, 128")
        self.codes = codes
        heads_first = layout == "hnd"
        shape = (num_blocks, num_kv_heads, block_size, head_size) if heads_first else (num_blocks, block_size, num_kv_heads, head_size)
        for name in ("k_codes", "v_codes"):
            plane = torch.zeros(shape, dtype=torch.uint8, device=self.device).view(CODES[codes])
            setattr(self, name, plane if heads_first else plane.transpose(1, 2))
        for name in ("k_scales", "v_scales"):
            setattr(self, name, torch.zeros((num_blocks, num_kv_heads), dtype=torch.float32, device=self.device))

    @property
    def planes(self) -> tuple:
        return self.k_codes, self.v_codes, self.k_scales, self.v_scales

    def append(self, seq_ids: Sequence, keys: torch.Tensor, values: torch.Tensor) -> None:
        """keys, values (n_seq, num_kv_heads, new_tokens, head_size): the next ``new_tokens`` positions of every listed
        sequence (new sequences start at position 0; the entries of an id that is listed more than once follow one
        another, each in a call of its own, because they can share a page).  A call that raises, for want of pages or
        otherwise, leaves lengths and pages as they were."""
        ops._need_cuda(keys, "QuashKVPaged8Cache.append")
        n, H, T, D = keys.shape
        if n != len(seq_ids) or H != self.num_kv_heads or D != self.head_size or values.shape != keys.shape:
            raise ValueError(f"Expected keys and values of shape ({len(seq_ids)}, {self.num_kv_heads}, T, {self.head_size})")
        if n == 0 or T == 0:
            return
        turns, seen = [], {}
        for i, s in enumerate(seq_ids):
            turn = seen[s] = seen.get(s, -1) + 1
            if turn == len(turns):
                turns.append([])
            turns[turn].append(i)
        with self._storing(seq_ids, T) as starts:
            table, _, _ = self.block_table(seq_ids)
            starts = torch.tensor(starts, dtype=torch.int32, device=self.device)
            if len(turns) == 1:
                return self.append_with_tables(keys, values, table, starts)
            for turn in turns:
                at = torch.tensor(turn, device=self.device)
                self.append_with_tables(keys[at], values[at], table[at], starts[at])

    def append_with_tables(self, keys: torch.Tensor, values: torch.Tensor, block_table: torch.Tensor,
                           start_lens: torch.Tensor) -> None:
        """The same store for a caller that owns the page allocation: ``block_table`` (n_seq, max_blocks) int32 and
        ``start_lens`` (n_seq) int32 on the device.  A token whose position lies outside its row of the table is not
        stored, and counted (``dropped_tokens``).  The pool's own bookkeeping is not involved."""
        append_paged8(keys, values, *self.planes, block_table=block_table, start_lens=start_lens)

    def append_slots(self, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor) -> None:
        """keys, values (tokens, num_kv_heads, head_size) to ``slots`` (tokens) int64, as ``PageTables.extend`` gives them."""
        append_paged8(keys, values, *self.planes, slots)

    def attention_with_tables(self, queries: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, max_kv_len: int,
                              scale: Optional[float] = None, causal: bool = False,
                              query_starts: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                              start_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of every sequence over its own pages (see ``attention_paged8``)."""
        return attention_paged8(queries, *self.planes, block_table, seq_lens, max_kv_len, scale=scale, causal=causal,
                                query_starts=query_starts, max_q_len=max_q_len, start_lens=start_lens)

    def attention(self, seq_ids: Sequence, queries: torch.Tensor, scale: Optional[float] = None,
                  causal: bool = False) -> torch.Tensor:
        """queries (n_seq, q_heads, q_len, head_size) of every listed sequence over its own pages; with ``causal`` the
        q_len query rows are the last q_len positions of each sequence."""
        table, lens, longest = self.block_table(seq_ids)
        if longest == 0:
            raise ValueError("No KV pages stored yet")
        return self.attention_with_tables(queries, table, lens, longest, scale=scale, causal=causal)

    def decompress(self, seq_id) -> tuple:
        """The stored keys and values of one sequence, fp32, each (num_kv_heads, tokens, head_size)."""
        n, bs = self.seq_len(seq_id), self.block_size
        pages = torch.tensor(self._blocks.get(seq_id, []), dtype=torch.int64, device=self.device)

        def rows(codes, scales):
            x = codes.view(torch.uint8)[pages].view(CODES[self.codes]).float() * scales[pages][..., None, None]
            return x.transpose(0, 1).reshape(self.num_kv_heads, -1, self.head_size)[:, :n]
        return rows(self.k_codes, self.k_scales), rows(self.v_codes, self.v_scales)
