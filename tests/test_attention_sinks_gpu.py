"""paged_attention with a window and sinks against its formula in 64 bits (tolerance as without sinks)."""
import pytest
import torch

from test_block_attention_gpu import rows_of
from test_paged_attention_gpu import TYPES, U16, make

pytestmark = pytest.mark.gpu


def check(args, window, sinks, **options):
    """Against 64 bits; the weights' pairs hold 16 bits, so the bound of one 16-bit number is taken out."""
    from powershard_amd import ops
    q, lengths = args[0], args[4]
    got, lse = ops.paged_attention(*args, window=window, sinks=sinks, return_lse=True, **options)
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(max(n, 0), device=q.device)[None]
        seen = (at >= n - window) | (at < sinks)
        out, bound, want = rows_of(q[b:b + 1], args[1:], b, seen)
        if n <= 0:
            assert (got[b] == 0).all() and (lse[b] == -float("inf")).all()
            continue
        codes = args[5] is not None
        u = 0.0 if codes and q.dtype == torch.float16 else U16[torch.bfloat16 if codes else q.dtype]
        hk = q.shape[1] // args[1].shape[1]
        pick = args[3][b, :-(-n // args[1].shape[2])].long()
        for h in range(q.shape[1]):      # sum p |v| of the head, to take u of it off the bound
            def tokens(pool, s):
                x = pool[:, h // hk].float().double()[pick].reshape(-1, q.shape[2])[:n]
                return x if s is None else x * s[:, h // hk].double()[pick].reshape(-1)[:n, None]
            s = (q[b, h].double() @ tokens(args[1], args[5]).T / q.shape[2] ** 0.5).masked_fill(~seen[0], -float("inf"))
            bound[0, h] -= u * (torch.softmax(s, -1) @ tokens(args[2], args[6]).abs())
        err = (got[b].double() - out[0]).abs()
        assert (err <= U16[got.dtype] * out[0].abs() + 2.0 ** -25 + bound[0] + 2.0 ** -40).all(), b
        assert ((lse[b].double() - want[0]).abs() <= 1e-4 + 1e-5 * want[0].abs()).all()
    return got


LENS = [1, 0, 5, 16, 17, 100, 129, 500, 1031, 3000]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 16), (7, 33), (64, 4), (100, 128), (128, 200), (1000, 129), (5000, 3)])
def test_windows_and_sinks(gpu, codes, dtype, window, sinks):
    args = make(LENS, 6, 2, 64, 16, codes, dtype, gpu, seed=window)
    for max_len in (None, 1, 4000):
        check(args, window, sinks, max_len=max_len)


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16)])
@pytest.mark.parametrize("Hq,Hk,D,page", [(40, 8, 128, 16), (16, 1, 256, 48), (34, 2, 96, 80), (5, 5, 16, 32)])
def test_shapes(gpu, codes, dtype, Hq, Hk, D, page):
    args = make([700, 33, 0, 2050], Hq, Hk, D, page, codes, dtype, gpu, seed=1)
    check(args, 300, 20)
    check(args, 1900, 64)


@pytest.mark.parametrize("codes,dtype", TYPES)
def test_long_and_many(gpu, codes, dtype):
    args = make([30000, 4097, 9000, 1], 8, 2, 128, 64, codes, dtype, gpu, seed=2)
    check(args, 4096, 64)
    check(args, 20000, 1000)
    args = make([(b * 37) % 700 for b in range(80)], 4, 2, 64, 32, codes, dtype, gpu, seed=3)
    check(args, 100, 5)


def test_no_sinks_is_the_window(gpu):
    from powershard_amd import ops
    for codes, dtype in TYPES:
        args = make(LENS, 6, 2, 64, 16, codes, dtype, gpu)
        for window in (0, 5, 64, 700):
            assert torch.equal(ops.paged_attention(*args, window=window, sinks=0), ops.paged_attention(*args, window=window))
        # sinks that reach the window hide nothing
        a, b = ops.paged_attention(*args, window=16, sinks=10 ** 6), ops.paged_attention(*args)
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max()


def test_pages_between_are_not_followed(gpu):
    """Pages that the window hides and that hold no sinks may be gone, and what they hold does not matter."""
    from powershard_amd import ops
    q, k, v, table, lengths, ks, vs = make([500, 330], 4, 2, 64, 16, "none", torch.bfloat16, gpu)
    want = ops.paged_attention(q, k, v, table, lengths, window=100, sinks=20)
    gone = table.clone()
    gone[0, 2:25], gone[1, 2:14] = -1, 2 ** 31 - 1
    assert torch.equal(ops.paged_attention(q, k, v, gone, lengths, window=100, sinks=20), want)
    for col in (0, 1, 25, 31):
        bad = table.clone()
        bad[0, col] = -1
        got = ops.paged_attention(q, k, v, bad, lengths, window=100, sinks=20)
        assert got[0].isnan().all() and torch.equal(got[1], want[1])
    k[table[0, 3].long()] = float("nan")
    v[table[0, 1].long(), :, 4:] = float("inf")      # tokens 20 .. 31: hidden, on a page of sinks
    assert torch.equal(ops.paged_attention(q, k, v, table, lengths, window=100, sinks=20), want)


def test_refusals(gpu):
    from powershard_amd import ops
    args = make([50], 4, 2, 64, 16, "none", torch.bfloat16, gpu)
    for bad in (dict(sinks=4), dict(window=4, sinks=-1), dict(window=4, sinks=None), dict(window=0, sinks=1)):
        with pytest.raises(ValueError):
            ops.paged_attention(*args, **bad)
