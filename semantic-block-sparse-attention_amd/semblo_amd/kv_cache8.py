"""A dense layer's key/value cache in 8 bits, the attention over it, and eviction from it.

The sparse layer's decode state (arena.py) holds bf16 K/V behind a prompt's clusters, for one request.  This
cache is for the layers that read every key: a batch of sequences, half the bytes per key, every size and
length on the device (calls can be captured in a HIP graph and replayed).  The reference leaves such layers to its
serving engine.

    cache = QuantizedKVCache(num_seqs=8, num_kv_heads=4, head_dim=256, capacity=131072, device="cuda")
    cache.append(k, v)                     # new tokens of every sequence, quantised block by block
    out = cache.attend(q)                  # the newest tokens' attention, each over what precedes it
    cache.attend(q, accumulate=True)       # besides, the attention that each block receives is added up
    cache.evict(keep=1024, sink=1, recent=16)     # the least attended blocks go

A block is 64 tokens of one (sequence, KV head), in OCP e4m3 (``fmt="e4m3"``) or signed integers (``"int8"``), with
one fp32 scale for its keys and one for its values: the largest magnitude over 448, or 127.  The rows of a sequence's
last block are kept in bf16 as well, and the block is quantised again whole whenever rows join it, so
that what a cache holds does not depend on how its tokens were split into calls.

Calls on one cache belong on one stream, or on streams that wait for one another.  Its tensors are fixed when it is made:
what they hold may be copied over, the attributes not be replaced.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

BLOCK = 64                       # SBSA_CACHE8_BLOCK
MAX_BLOCKS = 16384               # SBSA_CACHE8_MAX_BLOCKS
FORMATS = {"e4m3": 0, "int8": 1}
CODE_TYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class _Cache8(ctypes.Structure):
    """``sbsa_cache8`` of include/sbsa.h."""
    _fields_ = [(name, ctypes.c_void_p) for name in
                ("codes_k", "codes_v", "scales", "tail", "table", "weights", "lengths", "open_block", "counters",
                 "overflow")] + \
               [(name, ctypes.c_int32) for name in ("num_seqs", "num_kv_heads", "num_blocks", "head_dim", "format")]


def _check(t: torch.Tensor, what: str, shape, dtype) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor {list(shape)}, got {t.dtype} {list(t.shape)}")


class CacheTables:
    """Which blocks a cache's sequences hold: ``table`` [S, Hkv, N] int32, the place of each block (a permutation of
    0 .. N-1: the places behind a sequence's last block are free), ``weights`` [S, Hkv, N] fp32, the attention
    each block has received, ``lengths`` [S, Hkv] int32, the tokens held (the same for a sequence's heads), and
    ``open_block`` [S, Hkv] int32, the block whose rows are also kept in bf16 (-1: none)."""

    __slots__ = ("table", "weights", "lengths", "open_block")

    def __init__(self, table, weights, lengths, open_block) -> None:
        if table.dim() != 3:
            raise ValueError("table must be [sequences, KV heads, blocks]")
        s, h, n = table.shape
        _check(table, "table", (s, h, n), torch.int32)
        _check(weights, "weights", (s, h, n), torch.float32)
        _check(lengths, "lengths", (s, h), torch.int32)
        _check(open_block, "open_block", (s, h), torch.int32)
        if not 1 <= n <= MAX_BLOCKS:
            raise ValueError(f"a sequence holds 1 to {MAX_BLOCKS} blocks of {BLOCK} tokens, got {n}")
        if s < 1 or h < 1:
            raise ValueError("a cache holds at least one sequence and one KV head")
        self.table, self.weights, self.lengths, self.open_block = table, weights, lengths, open_block

    @classmethod
    def new(cls, num_seqs: int, num_kv_heads: int, num_blocks: int, device) -> "CacheTables":
        """The tables of empty sequences."""
        s, h = int(num_seqs), int(num_kv_heads)
        table = torch.arange(num_blocks, dtype=torch.int32, device=device).expand(s, h, -1).contiguous()
        return cls(table, torch.zeros(s, h, num_blocks, device=device),
                   torch.zeros(s, h, dtype=torch.int32, device=device),
                   torch.full((s, h), -1, dtype=torch.int32, device=device))

    def empty_like(self) -> "CacheTables":
        """Tables of the same shape, their contents still to be written (``evict``'s ``into``)."""
        return CacheTables(*(torch.empty_like(getattr(self, name)) for name in self.__slots__))

    def evict(self, keep: int, *, sink: int = 0, recent: int = 1, into: "CacheTables | None" = None) -> "CacheTables":
        """Cuts every (sequence, head) to at most ``keep`` blocks: the first ``sink`` blocks, the last ``recent``
        (one at least, the open block) and the heaviest of the others stay, in their order; of equal weights
        the earlier, and a weight that is not above 0 (a NaN too) counts as 0.  Sequences of ``keep`` blocks or fewer are left.
        Only the tables change: the blocks that go leave their places free.  ``into``: other tables to
        write instead (to see what would go, or to go on with both); returns the tables written."""
        keep, sink, recent = int(keep), int(sink), int(recent)
        if sink < 0 or recent < 1 or sink + recent > keep:
            raise ValueError(f"evict keeps sink ({sink}, at least 0) + recent ({recent}, at least 1) blocks within "
                             f"keep ({keep})")
        out = self if into is None else into
        if out is not self:
            if out.table.shape != self.table.shape:
                raise ValueError(f"into holds tables {list(out.table.shape)}, these are {list(self.table.shape)}")
        s, h, n = self.table.shape
        mine = (self.table, self.weights, self.lengths, self.open_block)
        others = mine if out is self else (out.table, out.weights, out.lengths, out.open_block)
        at, to = [t.data_ptr() for t in mine], [t.data_ptr() for t in others]
        for a, b, name in zip(at, to, self.__slots__):      # (contiguous, of 4-byte elements)
            if a != b and abs(a - b) < (s * h * n if name in ("table", "weights") else s * h) * 4:
                raise ValueError(f"into's {name} overlaps the tables' own")
        if out is self:
            _lib.require_one_device(*mine)
        else:
            _lib.require_one_device(*mine, *others)
        _lib.call_on(self.table.device, "sbsa_cache8_evict", *at, *to, s, h, n, keep, sink, recent)
        return out


class QuantizedKVCache:
    """An 8-bit key/value cache of ``num_seqs`` sequences of up to ``capacity`` tokens (rounded up to whole
    blocks; at most 1,048,576), for ``num_kv_heads`` heads of dimension 128 or 256."""

    def __init__(self, *, num_seqs: int, num_kv_heads: int, head_dim: int, capacity: int, fmt: str = "e4m3",
                 device) -> None:
        n = -(-int(capacity) // BLOCK)
        if not 1 <= n <= MAX_BLOCKS:
            raise ValueError(f"capacity must be 1 to {MAX_BLOCKS * BLOCK} tokens, got {capacity}")
        tables = CacheTables.new(num_seqs, num_kv_heads, n, device)
        s, h, d = int(num_seqs), int(num_kv_heads), int(head_dim)
        self._set(torch.empty(s, h, n, BLOCK, d, dtype=torch.uint8, device=device),
                  torch.empty(s, h, n, d, BLOCK, dtype=torch.uint8, device=device),
                  torch.empty(2, s, h, n, dtype=torch.float32, device=device),
                  torch.empty(2, s, h, BLOCK, d, dtype=torch.bfloat16, device=device), tables, fmt)

    @classmethod
    def over(cls, codes_k, codes_v, scales, tail, tables: CacheTables, *, fmt: str = "e4m3") -> "QuantizedKVCache":
        """A cache over tensors that are there already: ``codes_k`` [S, Hkv, N, 64, D] and ``codes_v`` [S, Hkv, N, D, 64]
        uint8, ``scales`` [2, S, Hkv, N] fp32 (keys, values), ``tail`` [2, S, Hkv, 64, D] bfloat16."""
        self = cls.__new__(cls)
        self._set(codes_k, codes_v, scales, tail, tables, fmt)
        return self

    def _set(self, codes_k, codes_v, scales, tail, tables, fmt) -> None:
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        s, h, n = tables.table.shape
        d = codes_k.shape[-1]
        if d not in (128, 256):
            raise ValueError(f"the 8-bit cache takes head dimensions 128 and 256, got {d}")
        _check(codes_k, "codes_k", (s, h, n, BLOCK, d), torch.uint8)
        _check(codes_v, "codes_v", (s, h, n, d, BLOCK), torch.uint8)
        _check(scales, "scales", (2, s, h, n), torch.float32)
        _check(tail, "tail", (2, s, h, BLOCK, d), torch.bfloat16)
        _lib.require_one_device(codes_k, codes_v, scales, tail, tables.table, tables.weights, tables.lengths,
                                tables.open_block)
        self.codes_k, self.codes_v, self.scales, self.tail, self.tables = codes_k, codes_v, scales, tail, tables
        self.fmt, self.device = fmt, codes_k.device
        self.num_seqs, self.num_kv_heads, self.num_blocks, self.head_dim = s, h, n, d
        # what the kernels' struct points to stays alive, whatever becomes of the attributes
        self._alive = (codes_k, codes_v, scales, tail, *(getattr(tables, name) for name in tables.__slots__))
        # the append's tickets, zero between calls, and its flag for rows that found no room
        self._counters = torch.zeros(s * h + 1, dtype=torch.int32, device=self.device)
        self._struct = _Cache8(
            *(_lib.ptr(t) for t in (codes_k, codes_v, scales, tail, tables.table, tables.weights, tables.lengths,
                                    tables.open_block, self._counters, self._counters[s * h:])),
            s, h, n, d, FORMATS[fmt])
        self._ref = ctypes.byref(self._struct)
        self._scale = d ** -0.5
        self._needs: dict = {}          # workspace bytes by a call's sizes

    @property
    def capacity(self) -> int:
        """Tokens that a sequence has room for."""
        return self.num_blocks * BLOCK

    @property
    def lengths(self) -> torch.Tensor:
        """Tokens held by each sequence and head, int32 [S, Hkv], on the device."""
        return self.tables.lengths

    @property
    def weights(self) -> torch.Tensor:
        """Attention received by each block, fp32 [S, Hkv, N]."""
        return self.tables.weights

    def overflowed(self) -> bool:
        """Whether an append since the last ``reset`` of all sequences dropped rows that found no room (waits for the GPU)."""
        return bool(self._counters[-1].item())

    def reset(self, seq: int | None = None) -> None:
        """Empties the sequence ``seq`` (None: all)."""
        at = slice(None) if seq is None else int(seq)
        self.tables.lengths[at].zero_()
        self.tables.open_block[at].fill_(-1)
        self.tables.weights[at].zero_()
        if seq is None:
            self._counters.zero_()

    def _rows(self, x: torch.Tensor, what: str, heads: int | None) -> torch.Tensor:
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{what} must be [tokens, {heads or 'heads'}, {self.head_dim}], got {list(x.shape)}")
        if x.dtype is not torch.bfloat16:
            raise ValueError(f"{what} must be bfloat16, got {x.dtype}")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("the 8-bit cache has no backward pass: call it under torch.no_grad()")
        # the kernels move pieces of 16 bytes; rows that lie otherwise are copied
        st, sh, one = x.stride()
        if one != 1 or st % 8 or sh % 8 or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        return x

    def _spread(self, tokens: int, offsets, max_rows):
        """(offsets' pointer, hint) of a call's rows."""
        if offsets is None:
            if tokens % self.num_seqs:
                raise ValueError(f"{tokens} rows do not go evenly over {self.num_seqs} sequences: pass offsets")
            return None, 0
        _check(offsets, "offsets", (self.num_seqs + 1,), torch.int32)
        return offsets.data_ptr(), int(max_rows or 0)

    def append(self, k: torch.Tensor, v: torch.Tensor, *, offsets: torch.Tensor | None = None,
               start: torch.Tensor | None = None, max_rows: int | None = None) -> None:
        """New tokens behind those that each sequence holds.  ``k`` (after the rotary embedding) and ``v`` are
        [T, Hkv, D] bfloat16 of any token and head strides: T / S rows of each sequence in turn, or with ``offsets``
        (int32 [S + 1] on the device) rows offsets[s] .. offsets[s + 1] of sequence s.  ``start`` (int32 [S] on
        the device): the rows go to position start[s] instead of the sequence's end, which must not lie before it, and the
        sequence ends behind them, so that a rejected guess is written over (with no rows: cut off); rows
        before ``start`` in its block are quantised again from their bf16 rows if it is the block last
        written, else from their codes.  Rows past the capacity are dropped (``overflowed``); where the host can
        tell, the call raises instead.  ``max_rows``: a hint, the most rows of a sequence."""
        k, v = self._rows(k, "k", self.num_kv_heads), self._rows(v, "v", self.num_kv_heads)
        tokens = k.shape[0]
        if v.shape[0] != tokens:
            raise ValueError(f"{tokens} keys and {v.shape[0]} values")
        at, hint = self._spread(tokens, offsets, max_rows)
        if at is None and tokens // self.num_seqs > self.capacity:
            raise ValueError(f"{tokens // self.num_seqs} rows of a sequence pass its room of {self.capacity}")
        if start is not None:
            _check(start, "start", (self.num_seqs,), torch.int32)
        _lib.require_one_device(self._alive[0], k, v, offsets, start)
        kst, ksh, _ = k.stride()
        vst, vsh, _ = v.stride()
        _lib.call_on(self.device, "sbsa_cache8_append", self._ref, k.data_ptr(), kst, ksh, v.data_ptr(), vst, vsh, tokens,
                     at, None if start is None else start.data_ptr(), hint)

    def attend(self, q: torch.Tensor, *, offsets: torch.Tensor | None = None, max_rows: int | None = None,
               sm_scale: float | None = None, accumulate: bool = False, return_lse: bool = False,
               out: torch.Tensor | None = None):
        """Attention of the newest tokens (their K/V are in the cache already): ``q`` [T, Hq, D] bfloat16, rows to sequences as
        in ``append``; row i of a sequence's n sees its first length - n + i + 1 tokens, and gives 0 (and an LSE of
        -inf) where there are none.  Hq / Hkv up to 16.  Rows of no sequence keep what ``out`` held, and have no LSE.
        ``accumulate`` adds to ``weights`` the probabilities each block received, over the rows and the query heads
        of its KV head.  ``max_rows``: a hint, the most rows of a sequence.  Rows times query heads stay below
        2^24.  Returns out [T, Hq, D], or (out, lse [T, Hq] fp32, natural)."""
        q = self._rows(q, "q", None)
        tokens, hq, d = q.shape
        if hq < 1 or hq % self.num_kv_heads or hq // self.num_kv_heads > 16:
            raise ValueError(f"{hq} query heads on {self.num_kv_heads} KV heads: 1 to 16 of them to each")
        at, hint = self._spread(tokens, offsets, max_rows)
        accumulate = bool(accumulate)
        if out is None:
            out = _lib.rows_like(q)
        elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(0) % 8 or \
                out.stride(1) % 8 or out.data_ptr() % 16 or not all(out.stride()):
            raise ValueError(f"out must be bfloat16 {list(q.shape)} with rows on 16 bytes, no two on the same")
        elif _lib.overlap(out, q):
            raise ValueError("out overlaps q")
        _lib.require_one_device(self._alive[0], q, out, offsets)
        # (empty_strided: as in rows_like)
        lse = torch.empty_strided((tokens, hq), (hq, 1), dtype=torch.float32, device=self.device) if return_lse else None
        # the workspace goes by sizes that the host knows; made anew by each call, so that captured graphs and streams have
        # their own
        key = (hq, tokens, hint, at is None, accumulate)
        need = self._needs.get(key)
        if need is None:
            if len(self._needs) > 4096:
                self._needs.clear()
            need = self._needs[key] = _lib.query("sbsa_cache8_attend_workspace_bytes", self._ref, hq, tokens, hint,
                                                 at is not None, accumulate)
        work = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=self.device) if need else None
        qst, qsh, _ = q.stride()
        ost, osh, _ = out.stride()
        _lib.call_on(self.device, "sbsa_cache8_attend", self._ref, q.data_ptr(), qst, qsh, hq, tokens, at, hint,
                     self._scale if sm_scale is None else sm_scale, out.data_ptr(), ost, osh,
                     None if lse is None else lse.data_ptr(), accumulate, None if work is None else work.data_ptr(), need)
        return (out, lse) if return_lse else out

    def evict(self, keep: int, *, sink: int = 0, recent: int = 1) -> None:
        """``CacheTables.evict`` on the cache's own tables."""
        self.tables.evict(keep, sink=sink, recent=recent)

    def read(self, seq: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """What the first ``length`` tokens of a sequence stand for, fp32 [length, Hkv, D] keys and values (for
        checks and moves: not a hot path)."""
        n = -(-int(length) // BLOCK)
        place = self.tables.table[seq, :, :n].long()
        heads = torch.arange(self.num_kv_heads, device=self.device)[:, None]
        kind = CODE_TYPES[self.fmt]
        k = self.codes_k[seq][heads, place].view(kind).float() * self.scales[0, seq][heads, place][..., None, None]
        v = self.codes_v[seq][heads, place].view(kind).float() * self.scales[1, seq][heads, place][..., None, None]
        k, v = k.flatten(1, 2), v.transpose(-1, -2).flatten(1, 2)
        return k[:, :length].transpose(0, 1), v[:, :length].transpose(0, 1)
