"""The paged cache's write and read-back against their formulas.

A write's arithmetic is fp32 with a fixed order (maximum, one division, one product and one rounding per
element), so codes and scales equal the same operations in torch; against 64 bits a code is the nearest
one up to 2^-22 of itself (the quotient's and the product's roundings).  A read is one product and one
rounding: exact."""
import pytest
import torch

from conftest import seeded

pytestmark = pytest.mark.gpu

CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0), "none": (None, None)}


def make_pools(pages, H, page, D, codes, dtype, gpu, fill=None):
    kind = CODES[codes][0] or dtype
    shape = (pages, H, page, D)
    k, v = (torch.zeros(shape, dtype=kind, device=gpu) for _ in range(2))
    if fill is not None:
        for t in (k, v):
            t.view(torch.uint8).fill_(fill)
    ks, vs = ((torch.full(shape[:3], float("nan"), device=gpu) for _ in range(2)) if codes != "none" else (None, None))
    return k, v, ks, vs


def by_slot(pool):
    """[slots, heads, ...] of a pool [pages, heads, page, ...]."""
    t = pool.transpose(1, 2)
    return t.reshape((-1,) + t.shape[2:])


def reference(x, codes):
    """(codes, scale) of rows x in fp32, as the library states them."""
    kind, lim = CODES[codes]
    f = x.float().cpu()
    amax = f.abs().amax(-1, keepdim=True)
    zero = amax < 2.0 ** -120
    mul = torch.where(zero, 0.0, torch.full_like(amax, lim) / amax)   # (lim / amax would be a reciprocal times lim)
    u = f * mul
    q = u.round().clamp(-127, 127).to(torch.int8) if codes == "int8" else u.clamp(-448, 448).to(kind)
    return q, torch.where(zero, 1.0, amax / lim).squeeze(-1)


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


@pytest.mark.parametrize("codes", ["int8", "fp8", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 16), (7, 3, 48, 16), (64, 8, 128, 16), (100, 5, 80, 48), (33, 2, 256, 64),
                                        (200, 40, 64, 32), (9, 1, 240, 112)])
def test_write_and_read(gpu, codes, dtype, T, H, D, page):
    from powershard_amd import ops
    g = seeded(T + D)
    pages = -(-T // page) + 3
    k, v, ks, vs = make_pools(pages, H, page, D, codes, dtype, gpu, fill=0x7F)
    before = [t.clone() for t in (k, v)]
    kv = (torch.randn(T, 2, H, D, generator=g) * torch.exp2(torch.randint(-6, 7, (T, 2, H, 1), generator=g).float())).to(dtype).to(gpu)
    slots = torch.randperm(pages * page, generator=g)[:T].to(gpu)
    ops.kv_write(kv[:, 0], kv[:, 1], slots, k, v, ks, vs)
    others = torch.ones(pages * page, dtype=torch.bool)
    others[slots.cpu()] = False
    seen = ops.kv_read(slots, k, v, ks, vs, out_dtype=dtype)
    f32 = ops.kv_read(slots, k, v, ks, vs, out_dtype=torch.float32)
    for i, (pool, scales, old) in enumerate(((k, ks, before[0]), (v, vs, before[1]))):
        got = by_slot(pool.view(torch.uint8) if codes == "fp8" else pool)
        assert same(got[others.to(gpu)], by_slot(old.view(torch.uint8) if codes == "fp8" else old)[others.to(gpu)])
        x = kv[:, i]
        if codes == "none":
            assert same(got[slots], x) and same(seen[i], x) and torch.equal(f32[i], x.float())
            continue
        q, s = reference(x, codes)
        assert same(got[slots], q)
        assert torch.equal(by_slot(scales)[slots].cpu(), s)
        assert by_slot(scales)[others.to(gpu)].isnan().all()
        # against 64 bits
        amax = x.double().cpu().abs().amax(-1, keepdim=True)
        u = x.double().cpu() / amax * CODES[codes][1]
        step = torch.ones_like(u) if codes == "int8" else torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3)
        assert ((q.float().double() - u).abs() <= 0.5 * step + 2.0 ** -22 * u.abs()).all()
        value = q.float() * s.unsqueeze(-1)
        assert torch.equal(f32[i].cpu(), value) and same(seen[i], value.to(dtype))


@pytest.mark.parametrize("codes", ["int8", "fp8", "none"])
def test_slots_outside(gpu, codes):
    """Negative slots and slots past the pool are not written and read as zeros."""
    from powershard_amd import ops
    k, v, ks, vs = make_pools(2, 2, 16, 64, codes, torch.bfloat16, gpu, fill=1)
    x = torch.randn(4, 2, 64, generator=seeded(1)).to(torch.bfloat16).to(gpu)
    slots = torch.tensor([-1, 31, 32, -(1 << 40)], device=gpu)
    ops.kv_write(x, x, slots, k, v, ks, vs)
    got = by_slot(k.view(torch.uint8) if codes == "fp8" else k)
    assert (got[:31].contiguous().view(torch.uint8) == 1).all()
    a, b = ops.kv_read(slots, k, v, ks, vs)
    assert torch.equal(a, b) and a.dtype == torch.bfloat16
    assert (a[[0, 2, 3]] == 0).all() and ((a[1] - x[1]).abs() <= 0.07 * x[1].abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_rows_of_zeros_nan_and_inf(gpu, codes):
    from powershard_amd import ops
    k, v, ks, vs = make_pools(1, 1, 16, 128, codes, torch.float16, gpu)
    x = torch.randn(5, 1, 128, generator=seeded(2)).half().to(gpu)
    x[1] = 0
    x[2, 0, 5] = float("nan")
    x[3, 0, 127] = float("inf")
    slots = torch.arange(5, device=gpu)
    ops.kv_write(x, x, slots, k, v, ks, vs)
    s = ks[0, 0, :5]
    assert s[1] == 1 and torch.isfinite(s[[0, 1, 4]]).all() and s[2].isnan() and not torch.isfinite(s[3])
    a, _ = ops.kv_read(slots, k, v, ks, vs)
    assert (a[1] == 0).all() and torch.isfinite(a[[0, 1, 4]]).all()
    assert not torch.isfinite(a[2]).any() and not torch.isfinite(a[3]).any()


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_rows_at_the_edge_of_zero(gpu, codes):
    """Rows whose 127 / max or 448 / max is at the end of fp32: zero rows below the limit, the nearest codes from
    there on, and never a code from a product of zero and infinity."""
    from powershard_amd import ops
    k, v, ks, vs = make_pools(1, 1, 16, 64, codes, torch.bfloat16, gpu, fill=0x7F)
    tops = [2.0 ** -121, 2.0 ** -120, 1.5 * 2.0 ** -120, 1.75 * 2.0 ** -120, 2.0 ** -119, 1.5 * 2.0 ** -119, 2.0 ** -110]
    x = torch.zeros(len(tops), 1, 64)
    x[:, 0, 1::3] = torch.tensor(tops)[:, None]
    x[:, 0, 2::3] = -0.25 * torch.tensor(tops)[:, None]
    x = x.to(torch.bfloat16).to(gpu)
    slots = torch.arange(len(tops), device=gpu)
    ops.kv_write(x, x, slots, k, v, ks, vs)
    kind, lim = CODES[codes]
    limit = 2.0 ** -120 if codes == "int8" else 2.0 ** -119
    got = by_slot(k)[slots].float().cpu()
    for i, top in enumerate(tops):
        want = (x[i].float().cpu().double() / top * lim).float() if top >= limit else torch.zeros(1, 64)
        want = want.round() if codes == "int8" else want.to(kind).float()
        assert torch.equal(got[i], want), top
        assert float(by_slot(ks)[i, 0]) == (float(torch.tensor(top) / lim) if top >= limit else 1.0)
    seen, _ = ops.kv_read(slots, k, v, ks, vs, out_dtype=torch.float32)
    assert ((seen - x.float()).abs().cpu() <= torch.tensor([t / 100 if t >= limit else t for t in tops])[:, None, None]).all()


def test_strides_and_empty(gpu):
    """Slices of a fused projection, misaligned rows, broadcast heads, no tokens."""
    from powershard_amd import ops
    T, H, D = 6, 4, 64
    g = seeded(3)
    fused = torch.randn(T, 3 * H * D + 8, generator=g).to(torch.bfloat16).to(gpu)
    x = fused[:, H * D:2 * H * D].view(T, H, D)
    odd = fused[:, 2 * H * D + 1:3 * H * D + 1].view(T, H, D)
    slots = torch.tensor([3, 40, 17, 2, 90, 16], device=gpu)
    pools = make_pools(8, H, 16, D, "int8", torch.bfloat16, gpu)
    ops.kv_write(x, odd, slots, *pools)
    k, v = ops.kv_read(slots, *pools)
    ref = make_pools(8, H, 16, D, "int8", torch.bfloat16, gpu)
    ops.kv_write(x.contiguous(), odd.contiguous(), slots, *ref)
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(pools, ref))
    one = x[:, :1].expand(T, H, D)
    ops.kv_write(one, one, slots, *pools)
    k, v = ops.kv_read(slots, *pools)
    assert torch.equal(k, v) and torch.equal(k, k[:, :1].expand(T, H, D))
    ops.kv_write(x[:0], x[:0], slots[:0], *pools)
    k, v = ops.kv_read(slots[:0], *pools)
    assert k.shape == v.shape == (0, H, D)


def test_refusals(gpu):
    from powershard_amd import ops
    k, v, ks, vs = make_pools(2, 2, 16, 64, "int8", torch.bfloat16, gpu)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    slots = torch.arange(3, device=gpu)
    for error, call in [
            (TypeError, lambda: ops.kv_write(x.float(), x.float(), slots, k, v, ks, vs)),
            (TypeError, lambda: ops.kv_write(x, x.half(), slots, k, v, ks, vs)),
            (TypeError, lambda: ops.kv_write(x, x, slots, k.half(), v.half())),
            (TypeError, lambda: ops.kv_write(x, x, slots, k.float(), v.float())),
            (ValueError, lambda: ops.kv_write(x, x, slots, k, v)),
            (ValueError, lambda: ops.kv_write(x, x, slots, k, v, ks, vs[:, :, :8])),
            (ValueError, lambda: ops.kv_write(x[:, :1], x[:, :1], slots, k, v, ks, vs)),
            (ValueError, lambda: ops.kv_write(x, x, slots.int(), k, v, ks, vs)),
            (ValueError, lambda: ops.kv_write(x, x, slots[:2], k, v, ks, vs)),
            (ValueError, lambda: ops.kv_write(x, x, slots, k.transpose(1, 2), v.transpose(1, 2), ks, vs)),
            (RuntimeError, lambda: ops.kv_write(x.cpu(), x.cpu(), slots.cpu(), k, v, ks, vs)),
            (RuntimeError, lambda: ops.kv_write(x[..., :24], x[..., :24], slots, k[..., :24].contiguous(), v[..., :24].contiguous(), ks, vs)),
            (RuntimeError, lambda: ops.kv_read(slots, k[:, :, :8].contiguous(), v[:, :, :8].contiguous(), ks[:, :, :8].contiguous(),
                                               vs[:, :, :8].contiguous())),
            (TypeError, lambda: ops.kv_read(slots, k, v, ks, vs, out_dtype=torch.int8)),
            (ValueError, lambda: ops.kv_read(slots.view(1, 3), k, v, ks, vs))]:
        with pytest.raises(error):
            call()
