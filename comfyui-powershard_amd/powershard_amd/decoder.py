"""A pre-norm text decoder layer on quantized linears and a paged key-value cache.

The layer that the int8 / fp8 / int4 linears, the fused norm (norm.RMSNorm), the gated MLP epilogue and
the cache (kv_cache.PagedKVCache) make together.  Both forms of a step are here: the tokens of a prompt,
whose attention reads the sequence back from the cache, and one new token of each of a batch of
sequences, whose attention reads the cache in place.

    rows, h = norm1(x + h);  q, k, v = q_proj(rows), k_proj(rows), v_proj(rows)
    cache <- rope(k), v;     x = o_proj(attention(rope(q), cache))
    rows, h = norm2(x + h);  x = down(silu(gate(rows)) * up(rows))
"""
import torch
from torch import nn

from .norm import RMSNorm, linear
from .quant_linear import QuantLinear

__all__ = ["DecoderLayer", "rope", "prompt_attention"]


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


class DecoderLayer(nn.Module):
    """One layer; its linears are QuantLinear modules (install_quant_linears) or plain ones before that.

    heads, kv_heads, head_dim: of the attention; mlp: hidden features of the gated MLP (up_proj holds the
    gate's rows, then the up rows)."""

    def __init__(self, hidden, heads, kv_heads, head_dim, mlp, eps=1e-6, dtype=torch.bfloat16, device=None):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm1, self.norm2 = (RMSNorm(hidden, eps, dtype, device) for _ in range(2))

        def lin(i, o):
            return nn.Linear(i, o, bias=False, dtype=dtype, device=device)
        self.q_proj, self.k_proj, self.v_proj = lin(hidden, heads * head_dim), lin(hidden, kv_heads * head_dim), lin(hidden, kv_heads * head_dim)
        self.o_proj, self.up_proj, self.down_proj = lin(heads * head_dim, hidden), lin(hidden, 2 * mlp), lin(mlp, hidden)

    def _projections(self, x, h, positions):
        qkv = (self.q_proj, self.k_proj, self.v_proj)
        rows, h = self.norm1(x, h, qkv)
        q, k, v = (linear(p, rows).reshape(-1, n, self.head_dim) for p, n in zip(qkv, (self.heads, self.kv_heads, self.kv_heads)))
        return rope(q, positions), rope(k, positions), v, h

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
        residual stream (None in front of the first layer).  (x, h) for the next layer."""
        return self(x, h, cache, layer, slots, seq=seq)

    def step(self, x, h, cache, layer, slots, table):
        """One new token of each sequence, x [batch, hidden]; table: cache.table(seqs) with it counted."""
        return self(x, h, cache, layer, slots, table=table)

    def forward(self, x, h, cache, layer, slots, seq=None, table=None):
        """prompt (seq) or step (table), as a module call: a sharded layer gathers its weights in its hooks."""
        if (seq is None) == (table is None):
            raise ValueError("a decoder layer takes a prompt's sequence or a step's table")
        return self._step(x, h, cache, layer, slots, table) if seq is None else self._prompt(x, h, cache, layer, seq, slots)

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
