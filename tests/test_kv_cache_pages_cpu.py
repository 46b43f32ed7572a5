"""PagedKVCache's pages (host side, no kernel): slots, tables, exhaustion, reuse, refusals; prompt_attention
and rope against their formulas on the CPU."""
import pytest
import torch

from powershard_amd.kv_cache import PagedKVCache


def cache(pages=6, codes=None, **kw):
    return PagedKVCache(2, pages, 16, 2, 64, codes=codes, device="cpu", **kw)


def test_slots_fill_pages_in_order():
    c = cache()
    a, b = c.open(), c.open()
    first = c.extend([a, b], 10)
    assert first.dtype == torch.int64 and len(set(first.tolist())) == 20
    more = c.extend([a], 20)
    assert torch.equal(c.slots(a), torch.cat([first[:10], more])) and c.length(a) == 30 and c.length(b) == 10
    pages = c.slots(a) // 16
    assert torch.equal(c.slots(a) % 16, torch.arange(30) % 16) and (pages[:16] == pages[0]).all() and (pages[16:] == pages[16]).all()
    table, lengths, longest = c.table([b, a])
    assert table.dtype == lengths.dtype == torch.int32 and lengths.tolist() == [10, 30] and longest == 30
    assert table.tolist() == [[int(first[10]) // 16, -1], [int(pages[0]), int(pages[16])]]
    assert c.table([])[0].shape == (0, 0)
    empty = c.open()
    assert c.table([empty])[0].shape == (1, 0) and c.slots(empty).shape == (0,)


def test_exhaustion_changes_nothing_and_closing_frees():
    c = cache(pages=3)
    a, b = c.open(), c.open()
    c.extend([a], 33)
    assert c.free_pages == 0
    with pytest.raises(RuntimeError):
        c.extend([a, b], 1)
    assert c.length(a) == 33 and c.length(b) == 0
    c.extend([a], 15)
    c.close(a)
    assert c.free_pages == 3
    assert sorted((c.extend([b], 48) // 16).unique().tolist()) == [0, 1, 2]
    with pytest.raises(KeyError):
        c.extend([a], 1)
    with pytest.raises(ValueError):
        c.extend([b, b], 0)


def test_pools_and_refusals():
    assert cache().k.shape == (2, 6, 2, 16, 64) and cache().k_scale is None and cache(dtype=torch.float16).v.dtype == torch.float16
    c = cache(codes="fp8")
    assert c.k.dtype == torch.float8_e4m3fn and c.v_scale.shape == (2, 6, 2, 16)
    for kw in (dict(codes="int4"), dict(page_size=24), dict(page_size=0), dict(head_dim=72), dict(head_dim=512)):
        args = dict(layers=1, pages=2, page_size=16, kv_heads=1, head_dim=64, device="cpu") | kw
        with pytest.raises(ValueError):
            PagedKVCache(**args)
    with pytest.raises(RuntimeError):   # the kernels need a GPU
        c.write(0, torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64))


@pytest.mark.parametrize("new,total,rows", [(1, 1, 4), (7, 7, 3), (5, 12, 256)])
def test_prompt_attention(new, total, rows):
    from powershard_amd.decoder import prompt_attention
    g = torch.Generator().manual_seed(new)
    q, k, v = (torch.randn(n, h, 32, generator=g) for n, h in ((new, 6), (total, 2), (total, 2)))
    got = prompt_attention(q, k, v, total - new, rows)
    for t in range(new):
        seen = total - new + t + 1
        for h in range(6):
            p = torch.softmax(k[:seen, h // 3].double() @ q[t, h].double() / 32 ** 0.5, 0)
            assert torch.allclose(got[t, h].double(), p @ v[:seen, h // 3].double(), atol=1e-5)


def test_rope_turns_pairs():
    from powershard_amd.decoder import rope
    x = torch.randn(3, 2, 8, generator=torch.Generator().manual_seed(1), dtype=torch.float32)
    y = rope(x, torch.tensor([0, 5, 9]))
    assert torch.equal(y[0], x[0])
    z = torch.complex(x[1, :, :4], x[1, :, 4:]) * torch.exp(1j * 5 * 10000.0 ** (-torch.arange(4) / 4))
    assert torch.allclose(y[1], torch.cat([z.real, z.imag], -1), atol=1e-6)
