"""A paged key-value cache: pools of pages for every layer, and the pages that each sequence holds.

Tokens of a sequence live in pages of ``page_size`` places; a page belongs to one sequence and holds the
same tokens in every layer, so one table serves all of them.  The pools are 16-bit, or int8 / e4m3 codes
with one fp32 scale per token and head, quantized as they are written (ops.kv_write, or ops.rope_kv_write,
which turns the keys to their positions on the way), read back (ops.kv_read) or read in place by the attention
of a batch of prompts (ops.paged_prompt_attention), of the next token (ops.paged_attention) and of trees of
drafted tokens (ops.paged_tree_attention).  No counterpart in the reference, whose text encoders run without
a cache.
"""
from typing import NamedTuple

import torch

from . import ops

__all__ = ["PagedKVCache", "Prompts", "Drafts"]

_KINDS = {None: None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


class Prompts(NamedTuple):
    """Where the newest tokens of a batch of sequences are: PagedKVCache.prompts."""
    block_table: torch.Tensor    # [batch, columns] int32
    lengths: torch.Tensor        # [batch] int32, the new tokens included
    longest: int
    starts: torch.Tensor         # [batch + 1] int32: the sequences' rows, end to end
    positions: torch.Tensor      # [tokens] int32


class Drafts(NamedTuple):
    """Where a tree of drafted tokens of each of a batch of sequences is: PagedKVCache.drafts."""
    block_table: torch.Tensor
    lengths: torch.Tensor        # [batch] int32, the drafts included
    longest: int
    parents: torch.Tensor        # [batch, n] int32
    positions: torch.Tensor      # [batch * n] int32


class PagedKVCache:
    def __init__(self, layers, pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, codes=None, device="cuda"):
        """pages of page_size tokens (a multiple of 16) for `layers` layers; dtype: of keys and values;
        codes: None (kept in dtype), "int8" or "fp8"."""
        if codes not in _KINDS:
            raise ValueError(f"unknown codes {codes!r}")
        if page_size <= 0 or page_size % 16 or head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"pages of {page_size} tokens of {head_dim} dims: multiples of 16, at most 256 dims")
        self.page_size, self.dtype, self.device = page_size, dtype, torch.device(device)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=_KINDS[codes] or dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = None
        if codes is not None:
            self.k_scale, self.v_scale = (torch.ones(shape[:4], dtype=torch.float32, device=device) for _ in range(2))
        self._free = list(range(pages - 1, -1, -1))
        self._held, self._length, self._next = {}, {}, 0

    # -- sequences (host side)
    @property
    def free_pages(self):
        return len(self._free)

    def open(self):
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._held[seq], self._length[seq] = [], 0
        return seq

    def close(self, seq):
        """Gives the sequence's pages back."""
        self._free += reversed(self._held.pop(seq))
        del self._length[seq]

    def length(self, seq):
        return self._length[seq]

    def extend(self, seqs, tokens):
        """Room for `tokens` more tokens of each of the sequences (a number, or one for each): their slots,
        [tokens of all] int64, in order.  RuntimeError, with nothing changed, when the pages do not suffice."""
        page, starts = self.page_size, [self._length[s] for s in seqs]
        more = list(tokens) if isinstance(tokens, (list, tuple)) else [tokens] * len(seqs)
        if len(more) != len(seqs) or (isinstance(tokens, (list, tuple)) and min(more, default=0) < 0):
            raise ValueError(f"{tokens} tokens for {len(seqs)} sequences")
        need = [-(-(a + m) // page) - len(self._held[s]) for s, a, m in zip(seqs, starts, more)]
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is extended twice")
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        for s, n, m in zip(seqs, need, more):
            self._held[s] += [self._free.pop() for _ in range(n)]
            self._length[s] += m
        return self._slots((s, range(a, a + m)) for s, a, m in zip(seqs, starts, more))

    def slots(self, seq):
        """The slots of all tokens of a sequence, [length] int64."""
        return self._slots([(seq, range(self._length[seq]))])

    def _slots(self, places):
        page = self.page_size
        return torch.tensor([self._held[s][t // page] * page + t % page for s, at in places for t in at], dtype=torch.int64).to(self.device)

    def table(self, seqs):
        """(block_table [batch, columns] int32, lengths [batch] int32, longest length) of the sequences."""
        cols = max((len(self._held[s]) for s in seqs), default=0)
        rows = [self._held[s] + [-1] * (cols - len(self._held[s])) for s in seqs]
        lengths = [self._length[s] for s in seqs]
        return (torch.tensor(rows, dtype=torch.int32).reshape(len(seqs), cols).to(self.device),
                torch.tensor(lengths, dtype=torch.int32).to(self.device), max(lengths, default=0))

    def prompts(self, seqs, new):
        """Prompts: the last new[i] tokens of each of the sequences, for the layers' prompts and for attend_prompts."""
        lengths = [self._length[s] for s in seqs]
        if len(new) != len(seqs) or any(not 0 <= n <= a for n, a in zip(new, lengths)):
            raise ValueError(f"{new} new tokens of sequences of {lengths}")
        starts, positions = [0], []
        for n, a in zip(new, lengths):
            starts.append(starts[-1] + n)
            positions.extend(range(a - n, a))
        return Prompts(*self.table(seqs), *(torch.tensor(x, dtype=torch.int32).to(self.device) for x in (starts, positions)))

    def drafts(self, seqs, parents):
        """Drafts: the last n tokens of each of the sequences as trees.  parents: [len(seqs)][n], the draft that
        each goes on from, an earlier one, or -1, the text in front."""
        rows, positions = [list(p) for p in parents], []
        if len(rows) != len(seqs) or len({len(p) for p in rows}) > 1:
            raise ValueError(f"{len(seqs)} sequences take as many rows of parents, all of one length")
        for s, row in zip(seqs, rows):
            text, depth = self._length[s] - len(row), []
            if text < 0:
                raise ValueError(f"{len(row)} drafts in a sequence of {self._length[s]} tokens")
            for i, p in enumerate(row):
                if not -1 <= p < i:
                    raise ValueError(f"draft {i} cannot go on from {p}")
                depth.append(0 if p < 0 else depth[p] + 1)
            positions += [text + d for d in depth]
        n = len(rows[0]) if rows else 0
        return Drafts(*self.table(seqs), torch.tensor(rows, dtype=torch.int32).reshape(len(seqs), n).to(self.device),
                      torch.tensor(positions, dtype=torch.int32).to(self.device))

    def accept(self, seq, n, kept):
        """Of the last n tokens of a sequence, its drafts, those of `kept` stay, in every layer, right behind the text;
        the others go, and the pages that they alone took.  kept: numbers of drafts, ascending (one way down the tree)."""
        kept, page = list(kept), self.page_size
        text = self._length[seq] - n
        if n < 0 or text < 0 or any(not a < b for a, b in zip([-1] + kept, kept + [n])):
            raise ValueError(f"drafts {kept} of {n} in a sequence of {self._length[seq]} tokens")
        moved = [(i, k) for i, k in enumerate(kept) if i != k]
        if moved:
            to, of = (self._slots([(seq, (text + m[i] for m in moved))]) for i in (0, 1))
            for pool in (self.k, self.v, self.k_scale, self.v_scale):
                if pool is not None:
                    x = pool.view(torch.uint8) if pool.dtype is torch.float8_e4m3fn else pool
                    x[:, to // page, :, to % page] = x[:, of // page, :, of % page]
        self._length[seq] = text + len(kept)
        held = -(-self._length[seq] // page)
        self._free += reversed(self._held[seq][held:])
        del self._held[seq][held:]

    # -- a layer's keys and values
    def _pools(self, layer):
        scales = (None, None) if self.k_scale is None else (self.k_scale[layer], self.v_scale[layer])
        return (self.k[layer], self.v[layer]) + scales

    def write(self, layer, k, v, slots):
        """New tokens' keys and values, [tokens, kv heads, head dim], to their slots."""
        ops.kv_write(k, v, slots, *self._pools(layer))

    def append(self, layer, q, k, v, positions, inv_freq, slots, **options):
        """New tokens' keys, turned to their positions, and values to their slots, and the queries, turned likewise;
        options of ops.rope_kv_write."""
        return ops.rope_kv_write(q, k, v, positions, inv_freq, slots, *self._pools(layer), **options)

    def read(self, layer, slots, out_dtype=None):
        """(keys, values) of the slots, [tokens, kv heads, head dim] of out_dtype (default: the cache's dtype)."""
        return ops.kv_read(slots, *self._pools(layer), out_dtype=out_dtype or self.dtype)

    def attend(self, layer, q, block_table, lengths, max_len=None, **options):
        """Attention of one new token per sequence, q [batch, heads, head dim]; options of ops.paged_attention."""
        k, v, ks, vs = self._pools(layer)
        return ops.paged_attention(q, k, v, block_table, lengths, ks, vs, max_len=max_len, **options)

    def attend_prompts(self, layer, q, prompts, **options):
        """Attention of the newest tokens of a batch of sequences, q [tokens, heads, head dim]; options of
        ops.paged_prompt_attention."""
        k, v, ks, vs = self._pools(layer)
        return ops.paged_prompt_attention(q, k, v, prompts.block_table, prompts.starts, prompts.lengths, ks, vs,
                                          max_len=prompts.longest, **options)

    def attend_drafts(self, layer, q, drafts, **options):
        """Attention of a tree of drafts of each sequence, q [batch, n, heads, head dim]; options of ops.paged_tree_attention."""
        k, v, ks, vs = self._pools(layer)
        return ops.paged_tree_attention(q, k, v, drafts.block_table, drafts.lengths, drafts.parents, ks, vs,
                                        max_len=drafts.longest, **options)
