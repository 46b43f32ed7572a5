"""paged_attention against its formula in 64 bits, on caches whose unwritten places hold NaN.

Tolerance, from the arithmetic, per output: the output type's half ulp of |o|, and (2 e + 2^-15) sum p |v|
for the weights, e = (D + 4) 2^-24 scale max_t sum |q k_t| bounding a score's fp32 error (it enters p and
the denominator), 2^-15 the weights' 16-bit pairs, their scales and fp32 sums of up to 2^8 partial sums."""
import math

import pytest
import torch

from conftest import seeded
from test_kv_cache_gpu import CODES

pytestmark = pytest.mark.gpu

U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # unit roundoff: 8 and 11 significant bits


def make(lens, Hq, Hk, D, page, codes, dtype, gpu, seed=0, spare_cols=2):
    """q, pools, scales, table, lengths; unwritten slots and unused pages NaN, unused columns wild."""
    g = torch.Generator(device=gpu).manual_seed(seed + sum(lens) + 7 * D)
    B, cols = len(lens), max(-(-n // page) for n in lens) + spare_cols
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g, device=gpu).tolist()
    table = torch.full((B, cols), 2 ** 31 - 1, dtype=torch.int32)
    table[:, 1::2] = -5
    valid = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        for c in range(held[b]):
            table[b, c] = order[at]
            valid[order[at], :min(page, n - c * page)] = True
            at += 1
    valid = valid.to(gpu)[:, None, :].expand(pages, Hk, page)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(pages, Hk, page, D, generator=g, device=gpu)
        if codes == "none":
            x = x.to(dtype)
            x[~valid] = float("nan")
            pools.append(x)
            scales.append(None)
            continue
        kind, lim = CODES[codes]
        x = (x * lim / 3.5).clamp(-lim, lim)
        x = x.round().to(kind) if codes == "int8" else x.to(kind)
        if codes == "fp8":
            x.view(torch.uint8)[~valid] = 0x7F
        s = (0.3 + 2 * torch.rand(pages, Hk, page, generator=g, device=gpu)) * 3.5 / lim
        s[~valid] = float("nan")
        pools.append(x)
        scales.append(s)
    q = torch.randn(B, Hq, D, generator=g, device=gpu) * torch.linspace(0.3, 4, Hq, device=gpu)[:, None]
    return (q.to(dtype), pools[0], pools[1], table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), scales[0], scales[1])


def formula(q, k, v, table, lengths, ks, vs, scale=None, window=0):
    """(out, bound of the error beside the output's rounding, lse) in 64 bits."""
    B, Hq, D = q.shape
    Hk, page = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, bound = (torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lengths[b])
        lo = max(0, n - window) if window else 0
        if n <= 0:
            continue
        pick = table[b, :-(-n // page)].long()
        for h in range(Hk):
            def tokens(pool, s):
                x = pool[:, h].float().double()[pick].reshape(-1, D)[lo:n]
                return x if s is None else x * s[:, h].double()[pick].reshape(-1)[lo:n, None]
            heads = slice(h * G, (h + 1) * G)
            kk, vv, qq = tokens(k, ks), tokens(v, vs), q[b, heads].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s, -1)
            e = (D + 4) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True)
            out[b, heads] = p @ vv
            bound[b, heads] = (2 * e + 2.0 ** -15) * (p @ vv.abs())
            lse[b, heads] = torch.logsumexp(s, -1)
    return out, bound, lse


def check(got, args, **kw):
    out, bound, _ = formula(*args, **kw)
    assert got.dtype == args[0].dtype
    err = (got.double() - out).abs()
    assert (err <= U16[got.dtype] * out.abs() + 2.0 ** -25 + bound).all(), float((err - bound).max())


TYPES = [("none", torch.bfloat16), ("none", torch.float16), ("int8", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16),
         ("fp8", torch.float16)]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D,page", [(5, 1, 128, 16), (8, 8, 64, 32), (32, 4, 128, 64), (16, 1, 256, 48), (34, 2, 128, 16),
                                          (3, 3, 16, 16), (6, 2, 96, 80), (20, 4, 240, 128), (7, 7, 144, 16), (40, 1, 80, 32), (64, 1, 64, 16),
                                          (33, 1, 256, 32), (96, 2, 128, 64), (130, 1, 48, 16)])
def test_shapes(gpu, codes, dtype, Hq, Hk, D, page):
    """Head layouts, head dims and pages; lengths of none, one, whole and broken tiles and pages."""
    from powershard_amd import ops
    args = make([1, 0, 15, 16, 17, 31, 32, 33, 64, 127, 129, 260], Hq, Hk, D, page, codes, dtype, gpu)
    got, lse = ops.paged_attention(*args, return_lse=True)
    check(got, args)
    want = formula(*args)[2]
    assert (got[1] == 0).all() and (lse[1] == -math.inf).all()
    some = torch.arange(12, device=gpu) != 1
    assert ((lse[some].double() - want[some]).abs() <= 1e-4 + 1e-5 * want[some].abs()).all()


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("max_len", [None, 1, 700, 4096, 200000])
def test_split_over_the_length(gpu, codes, dtype, max_len):
    """Long and ragged lengths, whatever the plan expects."""
    from powershard_amd import ops
    args = make([4096, 1, 3001, 513, 0, 1024], 10, 2, 128, 64, codes, dtype, gpu)
    for _ in range(3):   # the arrival counters are left as they were
        got = ops.paged_attention(*args, max_len=max_len)
    check(got, args)


@pytest.mark.parametrize("B,lens", [(1, [40000]), (1, [777]), (3, [9000, 12, 20001]), (70, None)])
def test_long_and_wide(gpu, B, lens):
    from powershard_amd import ops
    lens = lens or [(b * 37) % 900 for b in range(B)]
    args = make(lens, 40, 8, 128, 32, "int8", torch.bfloat16, gpu, seed=9)
    check(ops.paged_attention(*args), args)


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_units_that_stay_whole(gpu, codes, dtype, D):
    """Runs of more steps than a wave looks up pages for at once (4096 tokens a workgroup)."""
    from powershard_amd import ops
    args = make([13000, 4096, 4097, 8193], 6, 2, D, 16, codes, dtype, gpu, seed=D)
    check(ops.paged_attention(*args, max_len=1), args)
    bad = args[3].clone()
    bad[0, 700] = -1                       # past the first look-up of its workgroup
    got = ops.paged_attention(*args[:3], bad, *args[4:], max_len=1)
    assert got[0].isnan().all() and torch.isfinite(got[1:]).all()
    assert ops.paged_attention(*args[:3], bad, *args[4:])[0].isnan().all()


@pytest.mark.parametrize("B", [256, 257, 300, 1025])
def test_batches_wider_than_a_workgroup(gpu, B):
    """The runs are found from the lengths of the whole batch, several to a thread."""
    from powershard_amd import ops
    g = seeded(B)
    lens = [int(n) for n in torch.randint(0, 700, (B,), generator=g)]
    args = make(lens, 4, 2, 64, 16, "int8", torch.bfloat16, gpu, seed=3)
    got = ops.paged_attention(*args)
    check(got, args)
    assert torch.equal(ops.paged_attention(*args, max_len=1)[0] == 0, got[0] == 0)


def test_more_rounds_than_32_bits_times_runs(gpu):
    """8192 sequences on the same 20000 tokens: 10 million rounds, whose cuts need 64-bit products."""
    from powershard_amd import ops
    B, n = 8192, 20000
    q1, k, v, table, lengths, ks, vs = make([n], 8, 8, 64, 64, "int8", torch.bfloat16, gpu, seed=5)
    q = torch.randn(B, 8, 64, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu).to(torch.bfloat16)
    pick = torch.tensor([0, 1, 4000, 8190, 8191], device=gpu)
    got = ops.paged_attention(q, k, v, table.expand(B, -1), lengths.expand(B), ks, vs)
    few = (q[pick], k, v, table.expand(5, -1), lengths.expand(5), ks, vs)
    out, bound, _ = formula(*few)
    assert ((got[pick].double() - out).abs() <= U16[torch.bfloat16] * out.abs() + 2.0 ** -25 + bound).all()
    half = ops.paged_attention(q[2048:4096], k, v, table.expand(2048, -1), lengths.expand(2048), ks, vs)
    assert ((got[2048:4096].double() - half.double()).abs() <= 2 * U16[torch.bfloat16] * half.double().abs() + 1e-3).all()


@pytest.mark.parametrize("codes,dtype", [("none", torch.float16), ("int8", torch.bfloat16)])
@pytest.mark.parametrize("heads,lens", [(17, [5000, 3]), (24, [31, 32, 33, 777]), (64, [3000, 1, 64]), (100, [2049])])
def test_many_heads_share(gpu, codes, dtype, heads, lens):
    """More heads to a kv head than a wave has, split over the length."""
    from powershard_amd import ops
    args = make(lens, heads, 1, 128, 16, codes, dtype, gpu)
    check(ops.paged_attention(*args), args)
    two = make(lens, 2 * heads, 2, 64, 64, codes, dtype, gpu)
    check(ops.paged_attention(*two, max_len=1), two)


@pytest.mark.parametrize("heads", [17, 20, 31, 33, 47])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
def test_last_tiles_of_few_heads_joined_apart(gpu, heads, D):
    """The second kernel's grid has 16 heads for every tile; the last one of a kv head has fewer."""
    from powershard_amd import _native, ops
    args = make([40000, 5000], heads, 1, D, 16, "int8", torch.bfloat16, gpu)
    assert _native.lib().psq_paged_attention_own_workspace(_native.CODES_I8, 2, heads, 1, D, args[3].shape[1] * 16) == 1
    got, lse = ops.paged_attention(*args, return_lse=True)
    check(got, args)
    want = formula(*args)[2]
    assert ((lse.double() - want).abs() <= 1e-4 + 1e-5 * want.abs()).all()


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("fp8", torch.float16)])
@pytest.mark.parametrize("window", [1, 16, 100, 1000, 100000])
def test_window_and_scale(gpu, codes, dtype, window):
    """Only the last `window` tokens; pages before them may be gone from the table."""
    from powershard_amd import ops
    lens = [1, 99, 100, 101, 2500, 1003]
    args = make(lens, 12, 4, 64, 16, codes, dtype, gpu)
    want = formula(*args, scale=0.05, window=window)
    table = args[3].clone()
    for b, n in enumerate(lens):
        table[b, :max(0, n - window) // 16] = -1
    got = ops.paged_attention(*args[:3], table, *args[4:], scale=0.05, window=window)
    err = (got.double() - want[0]).abs()
    assert (err <= U16[dtype] * want[0].abs() + 2.0 ** -25 + want[1]).all()


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("gap", [11.0, 14.0, 17.0, 17.5, 20.0])
@pytest.mark.parametrize("max_len", [None, 1])
def test_small_probabilities(gpu, codes, dtype, gap, max_len):
    """A first token that takes nearly all weight and has the value 0, before a long tail whose scores are `gap`
    lower: the tail's values are all that the output has."""
    from powershard_amd import ops
    D, page, lens = 64, 16, [5000, 40, 700]
    args = make(lens, 4, 2, D, page, codes, dtype, gpu, seed=int(gap))
    q, k, v, table, lengths, ks, vs = args
    q.zero_()
    q[..., 0] = 8.0
    for t in (k, v):
        if codes != "none":
            t.view(torch.uint8)[:] = torch.where(t.float().isnan(), 0, t.view(torch.uint8))
    k[..., 0] = 0
    for b in range(3):
        first = int(table[b, 0])
        v[first, :, 0] = 0
        k[first, :, 0, 0] = 1
        if ks is not None:
            ks[first, :, 0] = gap
            vs[first, :, 0] = 1.0
        else:
            k[first, :, 0, 0] = gap
    args = (q, k, v.abs() if codes != "int8" else v.clamp(min=0), table, lengths, ks, vs) if codes != "fp8" else \
        (q, k, (v.view(torch.uint8) & 0x7F).view(v.dtype), table, lengths, ks, vs)
    got, lse = ops.paged_attention(*args, max_len=max_len, return_lse=True)
    check(got, args)
    want = formula(*args)[2]
    assert ((lse.double() - want).abs() <= 1e-4 + 1e-5 * want.abs()).all()


def test_values_that_are_not_finite(gpu):
    """A NaN in a token's key or value reaches its kv head's outputs and no others; scores of -inf get no
    weight; a sequence of only such scores is NaN, as softmax is."""
    from powershard_amd import ops
    args = make([70, 70, 70, 40], 4, 2, 64, 16, "none", torch.bfloat16, gpu)
    q, k, v, table = args[:4]
    clean = ops.paged_attention(*args)
    k[table[0, 4], 0, 3, 9] = float("nan")
    v[table[1, 0], 1, 2, 5] = float("inf")
    q[2] = q[2].abs() + 0.1
    k[table[2, 1], :, 7] = float("-inf")
    for c in range(3):
        k[table[3, c], 1] = float("-inf")
    q[3] = q[3].abs() + 0.1
    got = ops.paged_attention(*args)
    assert got[0, :2].isnan().all() and torch.equal(got[0, 2:], clean[0, 2:])
    assert torch.equal(got[1, :2], clean[1, :2]) and torch.isinf(got[1, 2:, 5]).all()
    assert torch.isfinite(got[1, 2:, torch.arange(64, device=gpu) != 5]).all()
    want = formula(*args)
    assert (got[2].double() - want[0][2]).abs().le(U16[torch.bfloat16] * want[0][2].abs() + 1e-3).all() and torch.isfinite(got[2]).all()
    assert got[3, 2:].isnan().all() and torch.isfinite(got[3, :2]).all()


@pytest.mark.parametrize("codes,dtype", [t for t in TYPES if t[0] != "int8"])
@pytest.mark.parametrize("D", [64, 96, 128, 144, 256])
@pytest.mark.parametrize("max_len", [None, 1])
def test_sums_beside_an_infinite_one(gpu, codes, dtype, D, max_len):
    """An infinite value (e4m3, which has none: a NaN) in one dim of a token: that dim is infinite, and the other
    dims are as near to the formula as ever."""
    from powershard_amd import ops
    args = make([300, 5000, 33], 6, 2, D, 16, codes, dtype, gpu, seed=D)
    v, table = args[2], args[3]
    for b, (token, dim) in enumerate([(200, 5), (4999, D - 1), (0, 0)]):
        at = v[table[b, token // 16], 1, token % 16]
        if codes == "fp8":
            at.view(torch.uint8)[dim] = 0x7F
        else:
            at[dim] = float("-inf") if b == 1 else float("inf")
    got = ops.paged_attention(*args, max_len=max_len).double()
    out, bound, _ = formula(*args)
    wild = torch.zeros_like(out, dtype=torch.bool)
    for b, dim in enumerate([5, D - 1, 0]):
        wild[b, 3:, dim] = True
    assert torch.equal(~torch.isfinite(got), wild)
    if codes != "fp8":
        assert torch.equal(got[wild], out[wild])
    err = (got - out).abs()
    assert (err <= U16[dtype] * out.abs() + 2.0 ** -25 + bound)[~wild].all()


def test_tables_that_lead_nowhere(gpu):
    """A page outside the pool, or a length past the table, makes its sequence NaN and touches nothing else."""
    from powershard_amd import ops
    args = make([70, 70, 2000, 5], 4, 2, 128, 16, "int8", torch.bfloat16, gpu)
    clean = ops.paged_attention(*args)
    table, lengths = args[3].clone(), args[4].clone()
    table[1, 2] = -1
    table[2, 100] = args[1].shape[0]
    lengths[3] = table.shape[1] * 16 + 1
    got, lse = ops.paged_attention(*args[:3], table, lengths, *args[5:], return_lse=True)
    assert torch.equal(got[0], clean[0]) and torch.isfinite(lse[0]).all()
    assert got[1:].isnan().all() and lse[1:].isnan().all()


def test_same_bits_every_time(gpu):
    from powershard_amd import ops
    args = make([5000, 333, 2048], 40, 8, 128, 16, "int8", torch.bfloat16, gpu)
    first = ops.paged_attention(*args)
    for _ in range(30):
        assert torch.equal(ops.paged_attention(*args), first)


def test_strides_streams_and_empty_batches(gpu):
    from powershard_amd import ops
    args = make([300, 4, 1000], 8, 2, 128, 16, "fp8", torch.bfloat16, gpu)
    q, k, v, table, lengths, ks, vs = args
    ref = ops.paged_attention(*args)
    fused = torch.zeros(3, 8 * 128 + 264, dtype=q.dtype, device=gpu)
    fused[:, 8:8 + 1024] = q.reshape(3, -1)
    odd = torch.zeros(3 * 1024 + 1, dtype=q.dtype, device=gpu)[1:].view(3, 8, 128)
    odd.copy_(q)
    wide = torch.zeros(3, 2 * table.shape[1], dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    apart = torch.zeros(3, table.shape[1], 2, dtype=torch.int32, device=gpu)
    apart[..., 0] = table
    for qq in (fused[:, 8:8 + 1024].view(3, 8, 128), odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        for tt in (wide[:, :table.shape[1]], apart[..., 0]):
            assert torch.equal(ops.paged_attention(qq, k, v, tt, lengths, ks, vs), ref)
    same = ops.paged_attention(q, k, v, table[2:3].expand(3, -1), lengths[2:3].expand(3), ks, vs)
    assert torch.equal(same[2], ref[2])
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        got = ops.paged_attention(*args)
    side.synchronize()
    assert torch.equal(got, ref)
    none = ops.paged_attention(q[:0], k, v, table[:0], lengths[:0], ks, vs)
    assert none.shape == (0, 8, 128)
    assert (ops.paged_attention(q, k, v, table[:, :0], lengths * 0, ks, vs) == 0).all()


def test_offsets_past_32_bits(gpu):
    """Pages whose bytes and elements lie past 4 GiB of the pool."""
    from powershard_amd import ops
    pages, page, D = 1100000, 16, 256
    k, v = (torch.zeros(pages, 1, page, D, dtype=torch.int8, device=gpu) for _ in range(2))
    ks, vs = (torch.zeros(pages, 1, page, device=gpu) for _ in range(2))
    x = torch.randn(40, 2, 1, D, generator=seeded(4)).to(torch.bfloat16).to(gpu)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=gpu)
    slots = (table[0].long()[:, None] * page + torch.arange(page, device=gpu)).view(-1)[:40]
    ops.kv_write(x[:, 0], x[:, 1], slots, k, v, ks, vs)
    a, b = ops.kv_read(slots, k, v, ks, vs)
    assert ((a - x[:, 0]).abs() <= 0.01 * x[:, 0].abs().amax(-1, keepdim=True)).all()
    q = torch.randn(1, 4, D, generator=seeded(5)).to(torch.bfloat16).to(gpu)
    got = ops.paged_attention(q, k, v, table, torch.tensor([40], dtype=torch.int32, device=gpu), ks, vs)
    few = [torch.cat([t[-2:], t[3:4]]) for t in (k, v, ks, vs)]
    small = (q, few[0], few[1], torch.tensor([[1, 2, 0]], dtype=torch.int32, device=gpu), torch.tensor([40], dtype=torch.int32, device=gpu),
             few[2], few[3])
    check(got, small)


def test_refusals(gpu):
    from powershard_amd import ops
    args = make([30, 20], 8, 2, 64, 16, "int8", torch.bfloat16, gpu)
    q, k, v, table, lengths, ks, vs = args
    for error, call in [
            (TypeError, lambda: ops.paged_attention(q.float(), *args[1:])),
            (TypeError, lambda: ops.paged_attention(q, k.half(), v.half(), table, lengths)),
            (ValueError, lambda: ops.paged_attention(q, k, v, table, lengths)),
            (ValueError, lambda: ops.paged_attention(q[:, :7], *args[1:])),
            (ValueError, lambda: ops.paged_attention(q[..., :32], *args[1:])),
            (ValueError, lambda: ops.paged_attention(q, k, v, table.long(), lengths, ks, vs)),
            (ValueError, lambda: ops.paged_attention(q, k, v, table[:1], lengths, ks, vs)),
            (ValueError, lambda: ops.paged_attention(q, k, v, table, lengths.long(), ks, vs)),
            (ValueError, lambda: ops.paged_attention(q, k, v, table, lengths[:1], ks, vs)),
            (ValueError, lambda: ops.paged_attention(*args, window=-1)),
            (RuntimeError, lambda: ops.paged_attention(q, k, v, table.cpu(), lengths, ks, vs)),
            (RuntimeError, lambda: ops.paged_attention(q[..., :24], k[..., :24].contiguous(), v[..., :24].contiguous(), table, lengths, ks, vs))]:
        with pytest.raises(error):
            call()
