"""A paged key-value cache: pools of pages for every layer, and the pages that each sequence holds.

Tokens of a sequence live in pages of ``page_size`` places; a page belongs to one sequence and holds the
same tokens in every layer, so one table serves all of them.  The pools are 16-bit, or int8 / e4m3 codes
with one fp32 scale per token and head, quantized as they are written (ops.kv_write), read back by the
prompt's attention (ops.kv_read) and read in place by the next token's (ops.paged_attention).  No
counterpart in the reference, whose text encoders run without a cache.
"""
import torch

from . import ops

__all__ = ["PagedKVCache"]

_KINDS = {None: None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


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
        """Room for `tokens` more tokens of each of the sequences: their slots, [len(seqs) * tokens] int64,
        in order.  RuntimeError, with nothing changed, when the pages do not suffice."""
        page, starts = self.page_size, [self._length[s] for s in seqs]
        need = [-(-(a + tokens) // page) - len(self._held[s]) for s, a in zip(seqs, starts)]
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is extended twice")
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        for s, n in zip(seqs, need):
            self._held[s] += [self._free.pop() for _ in range(n)]
            self._length[s] += tokens
        return self._slots((s, range(a, a + tokens)) for s, a in zip(seqs, starts))

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

    # -- a layer's keys and values
    def _pools(self, layer):
        scales = (None, None) if self.k_scale is None else (self.k_scale[layer], self.v_scale[layer])
        return (self.k[layer], self.v[layer]) + scales

    def write(self, layer, k, v, slots):
        """New tokens' keys and values, [tokens, kv heads, head dim], to their slots."""
        ops.kv_write(k, v, slots, *self._pools(layer))

    def read(self, layer, slots, out_dtype=None):
        """(keys, values) of the slots, [tokens, kv heads, head dim] of out_dtype (default: the cache's dtype)."""
        return ops.kv_read(slots, *self._pools(layer), out_dtype=out_dtype or self.dtype)

    def attend(self, layer, q, block_table, lengths, max_len=None, **options):
        """Attention of one new token per sequence, q [batch, heads, head dim]; options of ops.paged_attention."""
        k, v, ks, vs = self._pools(layer)
        return ops.paged_attention(q, k, v, block_table, lengths, ks, vs, max_len=max_len, **options)
