"""paged_prompt_attention and paged_tree_attention where sequences are split over their length (the key tiles cut into runs, their
parts joined by a second kernel).  Each call's split is asked for, so that these cases stay what they are.  Tolerances as in
test_block_attention_gpu."""
import math

import pytest
import torch

from powershard_amd import _native
from test_block_attention_gpu import causal, check_prompts, prompts
from test_paged_attention_gpu import TYPES

pytestmark = pytest.mark.gpu

KIND = {"none": _native.CODES_NONE, "int8": _native.CODES_I8, "fp8": _native.CODES_E4M3}


def split(codes, T, B, N, Hq, Hk, D, window=0, sinks=0, max_len=0):
    return _native.lib().psq_paged_block_workspace_bytes(KIND[codes], T, B, N, Hq, Hk, D, window, sinks, max_len) > 0


def table_holds(pools):
    return pools[2].shape[1] * pools[0].shape[2]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("new", [[0, 0, 1, 0, 0], [1, 0, 0, 0, 0], [0, 2, 0, 0, 1, 0, 0]])
def test_fewer_rows_than_sequences(gpu, codes, dtype, new):
    shapes = [(n, 3000 + 171 * b) for b, n in enumerate(new)]
    q, pools, starts = prompts(shapes, 10, 2, 128, 64, codes, dtype, gpu, seed=12)
    assert split(codes, len(q), len(new), 0, 10, 2, 128, max_len=table_holds(pools))
    check_prompts(shapes, q, pools, starts)


def poisoned(pool, scales, where, dim, value):
    """The pool's or the scales' place is `value` in a copy."""
    pool, scales = pool.clone(), None if scales is None else scales.clone()
    if scales is None:
        pool[where][dim] = value
    else:
        scales[where] = value
    return pool, scales


CUTS = [dict(), dict(window=2000), dict(window=2000, sinks=1500)]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("kw", CUTS, ids=str)
def test_values_that_are_not_finite(gpu, codes, dtype, value, kw):
    """One in a middle part: the rows that see it have it in their sums, and they alone.  Both of its kinds in two parts: NaN."""
    from powershard_amd import ops
    new, n, D, page, dim = 90, 3000, 64, 16, 37
    q, pools, starts = prompts([(new, n)], 4, 2, D, page, codes, dtype, gpu, seed=16)
    k, v, table, lengths, ks, vs = pools
    assert split(codes, new, 1, 0, 4, 2, D, kw.get("window", 0), kw.get("sinks", 0), table_holds(pools))
    call = lambda v, vs: ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, return_lse=True, **kw)   # noqa: E731
    place = lambda t: (int(table[0, t // page]), 1, t % page)   # noqa: E731
    sees = causal(new, n, kw.get("window", 0), kw.get("sinks", 0), gpu)
    for token in (1333, 950, n - 20):        # seen by all rows, with the window alone by those up to 2949, by those from 2980 on
        rows = sees[:, token]
        assert rows.any()
        clean, sums = call(v, vs)
        got, lse = call(*poisoned(v, vs, place(token), dim, value))
        assert torch.equal(got[:, :2], clean[:, :2]) and torch.equal(got[~rows], clean[~rows]) and torch.equal(lse, sums)
        mine = got[rows][:, 2:].float()
        if codes == "none":
            hit = mine[..., dim]
            assert hit.isnan().all() if math.isnan(value) else (hit == value).all()
            rest = torch.arange(D, device=gpu) != dim
            assert torch.equal(got[rows][:, 2:][..., rest], clean[rows][:, 2:][..., rest])
        else:
            # an infinite scale: each dim of the token's values is infinite, by its code's sign, or NaN (0 times infinity)
            x = v[place(token)].float() * value
            assert ((mine == x) | (mine.isnan() & x.isnan())).all()
    if not math.isnan(value) and not kw:
        other = poisoned(*poisoned(v, vs, place(200), dim, -value), place(1333), dim, value)
        got, _ = call(*other)
        assert got[:, 2:, dim].isnan().all() if codes == "none" else not got[:, 2:].isfinite().any()
        assert torch.equal(got[:, :2], clean[:, :2])
