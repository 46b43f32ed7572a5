"""PagedKVCache's batches of prompts, trees of drafts and accepted drafts, and the decoder layer's Rotary (host side)."""
import pytest
import torch

from powershard_amd.decoder import DecoderLayer, Rotary
from powershard_amd.kv_cache import PagedKVCache


def cache(codes=None, pages=8):
    return PagedKVCache(2, pages, 16, 2, 32, codes=codes, device="cpu")


def test_prompts():
    c = cache()
    a, b = c.open(), c.open()
    first = c.extend([a, b], (5, 20))
    assert first.shape == (25,) and torch.equal(first, torch.cat([c.slots(a), c.slots(b)]))
    c.extend([a, b], [0, 3])
    p = c.prompts([b, a], [3, 5])
    assert p.lengths.tolist() == [23, 5] and p.longest == 23 and p.starts.tolist() == [0, 3, 8]
    assert p.positions.tolist() == [20, 21, 22, 0, 1, 2, 3, 4] and torch.equal(p.block_table, c.table([b, a])[0])
    assert c.prompts([], []).starts.tolist() == [0]
    for seqs, new in (([a], [6]), ([a], [-1]), ([a, b], [1])):
        with pytest.raises(ValueError):
            c.prompts(seqs, new)
    for tokens in ([1], [1, -1]):
        with pytest.raises(ValueError):
            c.extend([a, b], tokens)
    assert c.length(a) == 5 and c.length(b) == 23


def test_drafts():
    c = cache()
    a, b = c.open(), c.open()
    c.extend([a, b], [9, 4])
    d = c.drafts([a, b], [[-1, 0, 0, 2], [-1, -1, 1, 1]])
    assert d.parents.tolist() == [[-1, 0, 0, 2], [-1, -1, 1, 1]] and d.lengths.tolist() == [9, 4]
    assert d.positions.tolist() == [5, 6, 6, 7, 0, 0, 1, 1]
    assert c.drafts([a], [[]]).parents.shape == (1, 0) and c.drafts([], []).parents.shape == (0, 0)
    for seqs, rows in (([a], [[0]]), ([a], [[-1, 1]]), ([a], [[-2]]), ([a, b], [[-1]]), ([a, b], [[-1], [-1, 0]]), ([b], [[-1] * 5])):
        with pytest.raises(ValueError):
            c.drafts(seqs, rows)


@pytest.mark.parametrize("codes", [None, "int8", "fp8"])
@pytest.mark.parametrize("text,n,kept", [(5, 4, []), (5, 4, [0, 1, 2, 3]), (14, 6, [1, 4]), (0, 40, [0, 17, 39]), (16, 16, [15]), (15, 18, [0, 2]),
                                         (7, 0, [])])
def test_accept(codes, text, n, kept):
    c = cache(codes)
    other, a = c.open(), c.open()
    c.extend([other], 3)
    slots = c.extend([a], text + n)
    g = torch.Generator().manual_seed(text)
    for pool in (c.k, c.v):
        bits = pool if codes == "int8" else pool.view(torch.uint8) if codes else pool.view(torch.int16)
        bits.copy_(torch.randint(0, 100, bits.shape, generator=g))
    for pool in (c.k_scale, c.v_scale):
        if pool is not None:
            pool.uniform_(generator=g)

    def rows(pool, at):
        return pool.float()[:, at // 16, :, at % 16]
    before = [rows(p, slots) for p in (c.k, c.v, c.k_scale, c.v_scale) if p is not None]
    aside = [rows(p, c.slots(other)) for p in (c.k, c.v)]
    c.accept(a, n, kept)
    stay = list(range(text)) + [text + i for i in kept]
    assert c.length(a) == len(stay) and torch.equal(c.slots(a), slots[:len(stay)])
    assert c.free_pages == 8 - 1 - -(-len(stay) // 16)
    for was, p in zip(before, (c.k, c.v, c.k_scale, c.v_scale)):
        assert torch.equal(rows(p, c.slots(a)), was[stay])
    for was, p in zip(aside, (c.k, c.v)):
        assert torch.equal(rows(p, c.slots(other)), was)
    c.extend([a], 16)


def test_accept_refusals():
    c = cache()
    a = c.open()
    c.extend([a], 5)
    for n, kept in ((6, [0]), (3, [3]), (3, [1, 0]), (3, [1, 1]), (3, [-1]), (-1, [])):
        with pytest.raises(ValueError):
            c.accept(a, n, kept)
    assert c.length(a) == 5


def test_rotary_and_layer_refusals():
    r = Rotary(64, base=500.0, axes=[0, 1, 2, 2] * 8)
    freq, axes = r.on(torch.device("cpu"))
    assert freq.dtype == torch.float64 and torch.allclose(freq, 500.0 ** (-torch.arange(32).double() / 32)) and axes.dtype == torch.int32
    assert Rotary(16, inv_freq=[1.0] * 8).on(torch.device("cpu"))[0].tolist() == [1.0] * 8
    for kw in (dict(dim=24), dict(dim=0), dict(dim=32, inv_freq=[1.0] * 8), dict(dim=32, axes=[0])):
        with pytest.raises(ValueError):
            Rotary(**kw)
    for kw in (dict(window=5), dict(sinks=1), dict(rotary=r, sinks=1), dict(rotary=r, window=-1), dict(rotary=Rotary(128))):
        with pytest.raises(ValueError):
            DecoderLayer(64, 2, 1, 64, 64, **kw)
    layer, c = DecoderLayer(64, 2, 1, 64, 64), cache()
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    for kw in (dict(prompts=c.prompts([], [])), dict(drafts=c.drafts([], [])), dict(seq=0, positions=x), dict(), dict(seq=0, table=c.table([]))):
        with pytest.raises(ValueError):
            layer(x, None, c, 0, None, **kw)
