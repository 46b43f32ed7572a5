"""A pre-norm text decoder layer on quantized linears and a paged key-value cache.

The layer that the int8 / fp8 / int4 linears, the fused norm (norm.RMSNorm), the gated MLP epilogue and
the cache (kv_cache.PagedKVCache) make together.  The forms of a step are here: the tokens of a prompt, and one
new token of each of a batch of sequences, whose attention reads the cache in place.  A layer with a Rotary
turns queries and keys as it writes the cache, takes the prompts of a batch of sequences and trees of
drafted tokens in one call each, all on the cache in place, and may have a window; one without turns them by
torch operations at base 10000 and reads a prompt's sequence back from the cache.

    rows, h = norm1(x + h);  q, k, v = q_proj(rows), k_proj(rows), v_proj(rows)
    cache <- rope(k), v;     x = o_proj(attention(rope(q), cache))
    rows, h = norm2(x + h);  x = down(silu(gate(rows)) * up(rows))
"""
import torch
from torch import nn

from .norm import RMSNorm, linear
from .quant_linear import QuantLinear

__all__ = ["DecoderLayer", "Rotary", "rope", "prompt_attention"]


def rope(x, positions, base=10000.0):
    """Rotary positions: pairs (i, i + dim / 2) of x [tokens, heads, dim] turned by positions base^(-2 i / dim)."""
    half = x.shape[-1] // 2
    freq = base ** (-torch.arange(half, device=x.device, dtype=torch.float32) / half)
    angle = positions.to(torch.float32)[:, None, None] * freq
    a, b = x.float().chunk(2, -1)
    c, s = angle.cos(), angle.sin()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def prompt_attention(q, k, v, first, rows=256):
    """Causal attention of the tokens first, first + 1, ... (q [new, heads, dim]) on a sequence's keys and
    values [tokens, kv heads, dim], in fp32, `rows` tokens at a time."""
    new, heads, dim = q.shape
    group = heads // k.shape[1]
    kt = k.float().permute(1, 2, 0).contiguous()                       # [kv heads, dim, tokens]
    vt = v.float().transpose(0, 1).contiguous()
    at = torch.arange(k.shape[0], device=q.device)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    for a in range(0, new, rows):
        part = q[a:a + rows].float().reshape(-1, k.shape[1], group, dim).permute(1, 2, 0, 3)
        n = part.shape[2]
        scores = torch.matmul(part.reshape(k.shape[1], -1, dim), kt).reshape(k.shape[1], group, n, -1) * dim ** -0.5
        seen = at <= (first + a + torch.arange(n, device=q.device))[:, None]
        p = torch.softmax(scores.masked_fill(~seen, float("-inf")), -1)
        o = torch.matmul(p.reshape(k.shape[1], group * n, -1), vt).reshape(k.shape[1], group, n, dim)
        out[a:a + rows] = o.permute(2, 0, 1, 3).reshape(n, heads, dim).to(q.dtype)
    return out


class Rotary:
    """Rotary positions of a layer's heads: angles per position, base^(-2 i / dim) of pair i, or inv_freq, fp64 [pairs].

    dim: of the head's dims, the first ones that are turned (a multiple of 16); interleaved: pairs are neighbours;
    axes: for tokens with several positions (time, height and width, say) which of them turns each pair."""

    def __init__(self, dim, base=10000.0, inv_freq=None, interleaved=False, axes=None):
        if dim <= 0 or dim % 16:
            raise ValueError(f"{dim} dims turned: a multiple of 16")
        if inv_freq is None:
            inv_freq = float(base) ** (-torch.arange(dim // 2, dtype=torch.float64) * 2 / dim)
        self._freq = torch.as_tensor(inv_freq, dtype=torch.float64).cpu()
        self._axes = None if axes is None else torch.as_tensor(axes, dtype=torch.int32).cpu()
        if self._freq.shape != (dim // 2,) or (self._axes is not None and self._axes.shape != (dim // 2,)):
            raise ValueError(f"inv_freq and axes have {dim // 2} pairs")
        self.dim, self.interleaved, self._at = dim, interleaved, {}

    def on(self, device):
        """(inv_freq, axes) on the device."""
        if device not in self._at:
            self._at[device] = self._freq.to(device), None if self._axes is None else self._axes.to(device)
        return self._at[device]


class DecoderLayer(nn.Module):
    """One layer; its linears are QuantLinear modules (install_quant_linears) or plain ones before that.

    heads, kv_heads, head_dim: of the attention; mlp: hidden features of the gated MLP (up_proj holds the
    gate's rows, then the up rows); rotary: a Rotary, which layers may share; window, sinks: a token sees the last
    `window` (0: all) and the first `sinks` of those in front of it, with a rotary.

    With a rotary, the attention of prompts and drafts holds a probability as one 16-bit number (ops.paged_prompt_attention),
    a step's as two, and a layer without one has its prompt's in fp32: outputs of the same text by different forms differ
    by such roundings."""

    def __init__(self, hidden, heads, kv_heads, head_dim, mlp, eps=1e-6, dtype=torch.bfloat16, device=None, rotary=None, window=0, sinks=0):
        super().__init__()
        if rotary is None and (window or sinks):
            raise ValueError("a window is of a layer with a rotary")
        if window < 0 or sinks < 0 or (sinks and not window) or (rotary is not None and rotary.dim > head_dim):
            raise ValueError("window and sinks are 0 or more, sinks with a window; a rotary turns at most the head's dims")
        self.rotary, self.window, self.sinks = rotary, window, sinks
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm1, self.norm2 = (RMSNorm(hidden, eps, dtype, device) for _ in range(2))

        def lin(i, o):
            return nn.Linear(i, o, bias=False, dtype=dtype, device=device)
        self.q_proj, self.k_proj, self.v_proj = lin(hidden, heads * head_dim), lin(hidden, kv_heads * head_dim), lin(hidden, kv_heads * head_dim)
        self.o_proj, self.up_proj, self.down_proj = lin(heads * head_dim, hidden), lin(hidden, 2 * mlp), lin(mlp, hidden)

    def _projections(self, x, h, positions):
        q, k, v, h = self._unturned(x, h)
        return rope(q, positions), rope(k, positions), v, h

    def _unturned(self, x, h):
        qkv = (self.q_proj, self.k_proj, self.v_proj)
        rows, h = self.norm1(x, h, qkv)
        return *(linear(p, rows).reshape(-1, n, self.head_dim) for p, n in zip(qkv, (self.heads, self.kv_heads, self.kv_heads))), h

    def _rest(self, attended, h):
        x = self.o_proj(attended.reshape(attended.shape[0], -1))
        rows, h = self.norm2(x, h, (self.up_proj,))
        if isinstance(self.up_proj, QuantLinear):
            hidden = linear(self.up_proj, rows, "silu_gate")
        else:
            gate, up = self.up_proj(rows).chunk(2, -1)
            hidden = nn.functional.silu(gate.float()) * up.float()
        return self.down_proj(hidden.to(x.dtype)), h

    def prompt(self, x, h, cache, layer, seq, slots):
        """The newest tokens of a sequence, x [tokens, hidden], whose slots cache.extend gave.  h: the
        residual stream (None in front of the first layer).  (x, h) for the next layer.  With a rotary each layer has the
        cache make its prompts([seq], ...), copies to the device among it: prompts() takes one made once, and may be captured."""
        return self(x, h, cache, layer, slots, seq=seq)

    def prompts(self, x, h, cache, layer, slots, prompts, positions=None):
        """The newest tokens of a batch of sequences, end to end in x [tokens, hidden]; prompts: cache.prompts(seqs, new)
        with them counted; positions: others than theirs, [tokens] or [n, tokens].  Of a layer with a rotary."""
        return self(x, h, cache, layer, slots, prompts=prompts, positions=positions)

    def step(self, x, h, cache, layer, slots, table, positions=None):
        """One new token of each sequence, x [batch, hidden]; table: cache.table(seqs) with it counted; positions: others
        than its place, with a rotary."""
        return self(x, h, cache, layer, slots, table=table, positions=positions)

    def drafts(self, x, h, cache, layer, slots, drafts, positions=None):
        """A tree of drafted tokens of each sequence, x [batch * n, hidden]; drafts: cache.drafts(seqs, parents) with them
        counted.  Of a layer with a rotary.  cache.accept then keeps those that were right."""
        return self(x, h, cache, layer, slots, drafts=drafts, positions=positions)

    def forward(self, x, h, cache, layer, slots, seq=None, table=None, prompts=None, drafts=None, positions=None):
        """prompt (seq), prompts, step (table) or drafts, as a module call: a sharded layer gathers its weights in its hooks."""
        if sum(a is not None for a in (seq, table, prompts, drafts)) != 1:
            raise ValueError("a decoder layer takes a prompt's sequence, a step's table, a batch's prompts or its drafts")
        if self.rotary is not None:
            return self._paged(x, h, cache, layer, slots, seq, table, prompts, drafts, positions)
        if prompts is not None or drafts is not None or positions is not None:
            raise ValueError("batches of prompts, drafts and positions are for a layer with a rotary")
        return self._step(x, h, cache, layer, slots, table) if seq is None else self._prompt(x, h, cache, layer, seq, slots)

    def _paged(self, x, h, cache, layer, slots, seq, table, prompts, drafts, positions):
        if seq is not None:
            prompts = cache.prompts([seq], [x.shape[0]])
        if positions is None:
            positions = table[1] - 1 if table is not None else (drafts if prompts is None else prompts).positions
        q, k, v, h = self._unturned(x, h)
        inv_freq, axes = self.rotary.on(x.device)
        axes = axes if positions.dim() == 2 else None    # (one position: of all axes)
        q = cache.append(layer, q, k, v, positions, inv_freq, slots, axes=axes, interleaved=self.rotary.interleaved)
        seen = dict(window=self.window, sinks=self.sinks)
        if prompts is not None:
            out = cache.attend_prompts(layer, q, prompts, **seen)
        elif table is not None:
            out = cache.attend(layer, q, *table, **seen)
        else:
            out = cache.attend_drafts(layer, q.reshape(*drafts.parents.shape, *q.shape[1:]), drafts, **seen)
        return self._rest(out.reshape(x.shape[0], self.heads, self.head_dim), h)

    def _prompt(self, x, h, cache, layer, seq, slots):
        first = cache.length(seq) - x.shape[0]
        q, k, v, h = self._projections(x, h, torch.arange(first, first + x.shape[0], device=x.device))
        cache.write(layer, k, v, slots)
        # (fp32: the values that the codes stand for, as the step's attention takes them)
        return self._rest(prompt_attention(q, *cache.read(layer, cache.slots(seq), torch.float32), first), h)

    def _step(self, x, h, cache, layer, slots, table):
        block_table, lengths, longest = table
        q, k, v, h = self._projections(x, h, lengths - 1)
        cache.write(layer, k, v, slots)
        return self._rest(cache.attend(layer, q, block_table, lengths, longest), h)
