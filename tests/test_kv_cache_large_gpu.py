"""PagedKVCache.accept on pools of more than 2^31 elements: the kept drafts' rows move in every layer, and nothing else does."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", ["int8", "fp8", None])
def test_accept_past_2_31_elements(gpu, codes):
    from powershard_amd.kv_cache import PagedKVCache
    layers, pages, page, heads, dim = 33, 512, 64, 16, 128
    cache = PagedKVCache(layers, pages, page, heads, dim, codes=codes, device=gpu)
    assert cache.k.numel() > 2 ** 31
    pools = [p for p in (cache.k, cache.v, cache.k_scale, cache.v_scale) if p is not None]
    for i, p in enumerate(pools):
        bits = p.view(torch.uint8 if p.dtype.itemsize == 1 else torch.int16 if p.dtype.itemsize == 2 else torch.int32)
        bits.copy_(torch.arange(dim if p.dim() == 5 else page, device=gpu) + i)
        bits += torch.randint(0, 97, (layers, pages, heads) + (page, 1)[:p.dim() - 3], dtype=bits.dtype, device=gpu)
    first, seq = cache.open(), cache.open()
    cache.extend([first], (pages - 4) * page)
    cache.extend([seq], 3 * page + 6)                        # the last four pages; drafts 0 .. 8 lie on two of them
    of = [cache._held[seq][t // page] * page + t % page for t in range(3 * page + 6)]
    n, kept = 9, [1, 4, 8]
    text = 3 * page + 6 - n
    before = [p.clone() for p in pools]
    cache.accept(seq, n, kept)
    assert cache.length(seq) == text + 3
    for p, old in zip(pools, before):
        bits = [x.view(torch.uint8) if x.dtype is torch.float8_e4m3fn else x for x in (p, old)]
        for i, k in enumerate(kept):
            a, b = of[text + i], of[text + k]
            bits[1][:, a // page, :, a % page] = old.view(bits[1].dtype)[:, b // page, :, b % page]    # (ascending: no row is read after it)
        assert torch.equal(*bits)
