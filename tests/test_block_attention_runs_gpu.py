"""paged_prompt_attention and paged_tree_attention where sequences are split over their length (the key tiles cut into runs, their
parts joined by a second kernel): few rows on long texts, batches wider than a wave, lengths past the table, values that are not
finite.  Each call's split is asked for, so that these cases stay what they are.  Tolerances as in test_block_attention_gpu."""
import math

import pytest
import torch

from powershard_amd import _native
from test_block_attention_gpu import causal, check, check_lse, check_prompts, check_trees, prompts, rows_of
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


@pytest.mark.parametrize("codes,dtype", TYPES)
def test_batches_wider_than_a_wave(gpu, codes, dtype):
    """130 sequences of uneven lengths, some with no rows: runs begin in all of a scan's chunks."""
    shapes = [((b * 7) % 4, (b * 7) % 4 + 40 * (b % 3) + 1900 * (b % 11 == 5) + 2900 * (b == 129)) for b in range(130)]
    T = sum(n for n, _ in shapes)
    q, pools, starts = prompts(shapes, 4, 1, 64, 16, codes, dtype, gpu, tail=3, seed=13)
    for window, sinks in ((0, 0), (1500, 70)):
        assert split(codes, T + 3, 130, 0, 4, 1, 64, window, sinks, table_holds(pools))
        check_prompts(shapes, q, pools, starts, window, sinks)
    lens = [3 + 35 * (b % 5) + 1500 * (b % 9 == 4) for b in range(70)]
    assert split(codes, 210, 70, 3, 4, 1, 64, max_len=1608)
    check_trees(lens, 3, 4, 1, 64, 16, codes, dtype, gpu, seed=14, max_len=1608)


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("far", [300, 2 ** 30, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 70])
def test_lengths_past_the_table(gpu, codes, dtype, far, new):
    """NaN in the rows that see past the table and in their sums, the other sequences right; split, and whole."""
    from powershard_amd import ops
    shapes = [(new, 2500), (new, 2050), (new, 130)]
    q, (k, v, table, lengths, ks, vs), starts = prompts(shapes, 8, 2, 64, 64, codes, dtype, gpu, seed=15)
    table, lengths = table[:, :40].contiguous(), lengths.clone()            # 2560 tokens
    pools = (k, v, table, lengths, ks, vs)
    wants = [rows_of(q[b * new:(b + 1) * new], pools, b, causal(new, n, 0, 0, gpu)) for b, (_, n) in enumerate(shapes)]
    lengths[0] = min(2560 + far, 2 ** 31 - 1)
    parents = torch.full((3, 1), -1, dtype=torch.int32, device=gpu)
    for max_len in (None, 64):
        assert split(codes, 3 * new, 3, 0, 8, 2, 64, max_len=max_len or 2560) == (max_len is None)
        assert split(codes, 3, 3, 1, 8, 2, 64, max_len=max_len or 2560) == (max_len is None)
        got, lse = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, max_len=max_len, return_lse=True)
        tree, sums = ops.paged_tree_attention(q.view(3, new, 8, 64)[:, -1:], k, v, table, lengths, parents, ks, vs, max_len=max_len, return_lse=True)
        assert got[:new].isnan().all() and lse[:new].isnan().all() and tree[0].isnan().all() and sums[0].isnan().all()
        for b in (1, 2):
            out, bound, want = wants[b]
            check(got[b * new:(b + 1) * new], out, bound)
            check_lse(lse[b * new:(b + 1) * new], want)
            check(tree[b], out[-1:], bound[-1:])
            check_lse(sums[b], want[-1:])


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


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("kw", CUTS, ids=str)
@pytest.mark.parametrize("n", [170, 3000])
def test_keys_that_are_not_finite(gpu, codes, dtype, value, kw, n):
    """A score of +infinity or NaN: NaN in the row; of -infinity: the row without the token.  Whole units and cut ones."""
    from powershard_amd import ops
    new, D, page, dim = 90, 64, 16, 37
    token = 3 * n // 5 if n > 1000 else 130
    q, pools, starts = prompts([(new, n)], 4, 2, D, page, codes, dtype, gpu, seed=17)
    k, v, table, lengths, ks, vs = pools
    window, sinks = kw.get("window", 0), kw.get("sinks", 0)
    assert split(codes, new, 1, 0, 4, 2, D, window, sinks, table_holds(pools)) == (n > 1000)
    call = lambda k, ks: ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, return_lse=True, **kw)   # noqa: E731
    where = (int(table[0, token // page]), 1, token % page)
    seen = causal(new, n, window, sinks, gpu)
    rows = seen[:, token].clone()
    clean, sums = call(k, ks)
    got, lse = call(*poisoned(k, ks, where, dim, value))
    assert torch.equal(got[:, :2], clean[:, :2]) and torch.equal(got[~rows], clean[~rows]) and torch.equal(lse[~rows], sums[~rows])
    s = (q[:, 2:, dim].double() if codes == "none" else (q[:, 2:].double() @ k[where].float().double())) * value     # the token's score
    without = seen.clone()
    without[:, token] = False
    out, bound, want = rows_of(q, pools, 0, without)
    for head in (0, 1):
        gone = rows & ~(s[:, head] == -math.inf)
        left = rows & (s[:, head] == -math.inf)
        assert got[gone][:, 2 + head].isnan().all() and not lse[gone][:, 2 + head].isfinite().any()
        assert math.isnan(value) or (gone.any() and left.any()) or not rows.any()
        check(got[left][:, 2 + head], out[left][:, 2 + head], bound[left][:, 2 + head])
        check_lse(lse[left][:, 2 + head], want[left][:, 2 + head])


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("none", torch.float16), ("int8", torch.float16), ("fp8", torch.bfloat16)])
@pytest.mark.parametrize("kw", [dict(), dict(window=1800, sinks=40)], ids=str)
def test_bad_pages(gpu, codes, dtype, kw):
    """A row that sees a token whose page is not there gets NaN, the others what they had: of prompts and of trees."""
    from powershard_amd import ops
    new, n, page, N = 100, 3000, 32, 12
    q, pools, starts = prompts([(new, n), (30, 2064)], 4, 2, 128, page, codes, dtype, gpu, seed=18)
    k, v, table, lengths, ks, vs = pools
    window, sinks = kw.get("window", 0), kw.get("sinks", 0)
    assert split(codes, 130, 2, 0, 4, 2, 128, window, sinks, table_holds(pools)) and split(codes, 2 * N, 2, N, 4, 2, 128, window, sinks, table_holds(pools))
    parents = torch.full((2, N), -1, dtype=torch.int32, device=gpu)
    parents[:, 1:] = torch.arange(N - 1, device=gpu) // 2                # a heap: draft i at depth log2(i + 1)
    drafts = q[:2 * N].view(2, N, 4, 128)
    depth = (torch.arange(N, device=gpu) + 1).float().log2().floor().long()

    def call(table):
        return (ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, **kw),
                ops.paged_tree_attention(drafts, k, v, table, lengths, parents, ks, vs, **kw))
    clean, tree = call(table)
    assert not clean.isnan().any() and not tree.isnan().any()
    for col in (0, 1, 40, 92, 93):
        at = torch.arange(col * page, min((col + 1) * page, n), device=gpu)
        seen = causal(new, n, window, sinks, gpu)[:, at].any(1)
        text, pos = at[at < n - N], n - N + depth[:, None]
        hit = ((text > pos - window) | (text < sinks)).any(1) if window else torch.full((N,), len(text) > 0, device=gpu)
        for i in range(N):                                               # a draft's own way, whatever of it lies in the page
            way, j = [], i
            while j >= 0:
                way.append(j)
                j = (j + 1) // 2 - 1
            hit[i] |= any(n - N + j >= col * page and n - N + j < (col + 1) * page for j in way)
        for bad in (-1, k.shape[0], 2 ** 31 - 1):
            broken = table.clone()
            broken[0, col] = bad
            got, other = call(broken)
            assert got[:new][seen].isnan().all() and torch.equal(got[:new][~seen], clean[:new][~seen]) and torch.equal(got[new:], clean[new:])
            assert other[0][hit].isnan().all() and torch.equal(other[0][~hit], tree[0][~hit]) and torch.equal(other[1], tree[1])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4, 3.0])
@pytest.mark.parametrize("codes,dtype", [("none", torch.float16), ("int8", torch.bfloat16)])
def test_scales(gpu, scale, codes, dtype):
    shapes = [(70, 2500), (3, 1000)]
    q, pools, starts = prompts(shapes, 4, 2, 64, 16, codes, dtype, gpu, seed=19)
    assert split(codes, 73, 2, 0, 4, 2, 64, max_len=table_holds(pools))
    check_prompts(shapes, q, pools, starts, scale=scale)


def test_more_rows_than_tokens(gpu):
    """The rows in front of position 0 get zeros, in a call that is split for the longest text that its table could hold."""
    from powershard_amd import ops
    for codes, dtype in TYPES:
        q, pools, starts = prompts([(20, 2500)], 4, 2, 64, 16, codes, dtype, gpu, seed=20)
        k, v, table, _, ks, vs = pools
        assert split(codes, 20, 1, 0, 4, 2, 64, max_len=table_holds(pools))
        for n in (7, 1, 0, -5):
            lengths = torch.tensor([n], dtype=torch.int32, device=gpu)
            got, lse = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, return_lse=True)
            some = max(n, 0)
            out, bound, want = rows_of(q[20 - some:], pools, 0, causal(some, some, 0, 0, gpu))
            check(got[20 - some:], out, bound)
            check_lse(lse[20 - some:], want)
            assert (got[:20 - some] == 0).all() and (lse[:20 - some] == -math.inf).all()
