"""paged_prompt_attention and paged_tree_attention against their formula in 64 bits, on caches whose unwritten
places hold NaN and whose unused table columns are wild.

Tolerance, from the arithmetic, per output: the output type's half step of |o|, and (2 e + u + 2^-15) sum p |v| for
the weights: e = (D + 4) 2^-24 |scale| max_t sum |q k_t| bounds a score's fp32 error (it enters p and the
denominator), u is half a step of the 16-bit type of the probabilities (bf16; f16 for f16 rows on 16-bit caches;
none for f16 rows on codes, which enter as pairs), 2^-15 the scales, fp32 sums and the pairs.  f16 probabilities
end at 2^-31 of the largest: n 2^-31 max |v| more.  Sums over long texts of more terms than 2^8: their error grows
like the square root and stays below that 2^-15."""
import math

import pytest
import torch

from conftest import seeded
from test_paged_attention_gpu import TYPES, U16, make

pytestmark = pytest.mark.gpu


def rows_of(q, pools, b, seen, scale=None):
    """(out, bound, lse) of q [rows, heads, dim] on sequence b, in 64 bits; seen [rows, tokens] bool."""
    k, v, table, lengths, ks, vs = pools
    n, H, D = q.shape
    Hk, page, L = k.shape[1], k.shape[2], seen.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    pick = table[b, :-(-L // page)].long()
    codes = ks is not None
    u = 0.0 if codes and q.dtype == torch.float16 else U16[torch.bfloat16 if codes else q.dtype]
    out, bound = (torch.zeros(n, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    if n == 0 or L == 0:
        return out, bound, lse
    some = seen.any(1)
    for h in range(H):
        hk = h // (H // Hk)
        def tokens(pool, s):
            x = pool[:, hk].float().double()[pick].reshape(-1, D)[:L]
            return x if s is None else x * s[:, hk].double()[pick].reshape(-1)[:L, None]
        kk, vv, qq = tokens(k, ks), tokens(v, vs), q[:, h].double()
        s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
        p = torch.where(some[:, None], torch.softmax(s, -1), 0.0)
        size = (qq.abs() @ kk.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        e = (D + 4) * 2.0 ** -24 * abs(scale) * size
        out[:, h] = p @ vv
        bound[:, h] = (2 * e + u + 2.0 ** -15) * (p @ vv.abs()) + L * 2.0 ** -31 * vv.abs().max()
        lse[:, h] = torch.logsumexp(s, -1)
    return out, bound, lse


def check(got, out, bound):
    err = (got.double() - out).abs()
    assert not got.isnan().any()
    assert (err <= U16[got.dtype] * out.abs() * (1 + 2.0 ** -7) + 2.0 ** -25 + bound).all(), float((err - bound).max())


def check_lse(lse, want):
    none = want == -math.inf
    assert (lse[none] == -math.inf).all()
    assert ((lse[~none].double() - want[~none]).abs() <= 1e-4 + 1e-5 * want[~none].abs()).all()


def prompts(shapes, Hq, Hk, D, page, codes, dtype, gpu, seed=0, tail=0):
    """(q [tokens + tail, ...], pools, starts) of sequences of (new, all) tokens."""
    args = make([n for _, n in shapes], Hq, Hk, D, page, codes, dtype, gpu, seed=seed)
    starts = [0]
    for new, _ in shapes:
        starts.append(starts[-1] + new)
    g = torch.Generator(device=gpu).manual_seed(seed + 1)
    q = torch.randn(starts[-1] + tail, Hq, D, generator=g, device=gpu) * torch.linspace(0.3, 4, Hq, device=gpu)[:, None]
    return q.to(dtype), args[1:], torch.tensor(starts, dtype=torch.int32, device=gpu)


def causal(new, n, window, sinks, gpu):
    at, pos = torch.arange(n, device=gpu), (n - new + torch.arange(new, device=gpu))[:, None]
    seen = at <= pos
    return seen & ((at > pos - window) | (at < sinks)) if window else seen


def check_prompts(shapes, q, pools, starts, window=0, sinks=0, scale=None, **options):
    from powershard_amd import ops
    k, v, table, lengths, ks, vs = pools
    got, lse = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, window=window, sinks=sinks, scale=scale, return_lse=True, **options)
    assert got.shape == q.shape and got.dtype == q.dtype
    at = 0
    for b, (new, n) in enumerate(shapes):
        out, bound, want = rows_of(q[at:at + new], pools, b, causal(new, n, window, sinks, q.device), scale)
        check(got[at:at + new], out, bound)
        check_lse(lse[at:at + new], want)
        at += new
    assert (got[at:] == 0).all() and (lse[at:] == -math.inf).all()
    return got


SHAPES = [(1, 1), (0, 5), (15, 15), (16, 40), (1, 64), (65, 65), (64, 129), (130, 131), (3, 300), (0, 0), (77, 200)]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D,page", [(5, 1, 128, 16), (8, 8, 64, 32), (16, 4, 128, 64), (16, 1, 256, 48), (3, 3, 16, 16), (6, 2, 96, 80),
                                          (10, 2, 240, 128), (7, 7, 144, 16), (40, 1, 80, 32), (64, 1, 32, 16), (130, 2, 48, 16)])
def test_prompt_shapes(gpu, codes, dtype, Hq, Hk, D, page):
    """Head layouts, head dims and pages; sequences of no, one and many new tokens; rows behind the last one."""
    q, pools, starts = prompts(SHAPES, Hq, Hk, D, page, codes, dtype, gpu, tail=5)
    check_prompts(SHAPES, q, pools, starts)


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 64), (64, 4), (100, 200), (129, 65), (1000, 7)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_windows(gpu, codes, dtype, D, window, sinks):
    shapes = [(300, 700), (1, 513), (257, 257), (40, 2000), (0, 9), (2, 3)]
    q, pools, starts = prompts(shapes, 6, 2, D, 32, codes, dtype, gpu, seed=window)
    check_prompts(shapes, q, pools, starts, window, sinks)


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("max_len", [None, 1, 3000, 10 ** 6])
def test_prompt_long(gpu, codes, dtype, max_len):
    """Few rows on long texts, whatever the plan expects."""
    shapes = [(33, 9001), (1, 4096), (0, 800), (5, 5)]
    q, pools, starts = prompts(shapes, 10, 2, 128, 64, codes, dtype, gpu, seed=3)
    check_prompts(shapes, q, pools, starts, max_len=max_len)


def test_prompt_many_rows(gpu):
    """More tiles of rows than a chip has CUs, and more sequences than a wave has lanes."""
    shapes = [(1500, 1500), (600, 1000)]
    q, pools, starts = prompts(shapes, 20, 4, 64, 16, "none", torch.bfloat16, gpu)
    check_prompts(shapes, q, pools, starts)
    shapes = [(b % 7, b % 7 + b) for b in range(150)]
    q, pools, starts = prompts(shapes, 8, 2, 64, 16, "int8", torch.bfloat16, gpu, tail=3)
    check_prompts(shapes, q, pools, starts)
    check_prompts(shapes, q, pools, starts, window=20, sinks=3)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4, 3.0])
def test_prompt_scales(gpu, scale):
    shapes = [(70, 100)]
    for codes, dtype in (("none", torch.float16), ("int8", torch.bfloat16)):
        q, pools, starts = prompts(shapes, 4, 2, 64, 16, codes, dtype, gpu)
        check_prompts(shapes, q, pools, starts, scale=scale)


# ------------------------------------------------------------------------------- trees
def ways(parents, count):
    """path [N][N] bool and depths of a tree given by its parents."""
    N = len(parents)
    path, depth = torch.zeros(N, N, dtype=torch.bool), [0] * N
    for i in range(count):
        p = parents[i]
        if 0 <= p < i:
            path[i], depth[i] = path[p], depth[p] + 1
        path[i, i] = True
    return path, depth


def check_trees(lens, N, Hq, Hk, D, page, codes, dtype, gpu, window=0, sinks=0, drafts=None, parents=None, seed=0, **options):
    from powershard_amd import ops
    args = make(lens, Hq, Hk, D, page, codes, dtype, gpu, seed=seed)
    pools, B, g = args[1:], len(lens), seeded(seed + N)
    k, v, table, lengths, ks, vs = pools
    q = (torch.randn(B, N, Hq, D, generator=g) * torch.linspace(0.3, 4, Hq)[:, None]).to(dtype).to(gpu)
    if parents is None:
        parents = [[int(torch.randint(-1, i + 1, (1,), generator=g)) if i % 3 else i - 1 for i in range(N)] for _ in range(B)]
    given = None if drafts is None else torch.tensor(drafts, dtype=torch.int32, device=gpu)
    got, lse = ops.paged_tree_attention(q, k, v, table, lengths, torch.tensor(parents, dtype=torch.int32, device=gpu).reshape(B, N), ks, vs,
                                        drafts=given, window=window, sinks=sinks, return_lse=True, **options)
    assert got.shape == q.shape and got.dtype == dtype
    for b, n in enumerate(lens):
        count = min(N, N if drafts is None else drafts[b], n)
        text = n - count
        path, depth = ways(parents[b], count)
        pos = torch.tensor([text + d for d in depth], dtype=torch.int64)
        at = torch.cat([torch.arange(text), pos[:count]])
        seen = torch.cat([torch.ones(N, text, dtype=torch.bool), path[:, :count]], 1)
        if window:
            seen &= (at > pos[:, None] - window) | (at < sinks)
        seen[count:] = False
        out, bound, want = rows_of(q[b], pools, b, seen.to(gpu))
        check(got[b], out, bound)
        check_lse(lse[b], want)
        assert (got[b, count:] == 0).all()
    return got


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D,page,N", [(5, 1, 128, 16, 16), (8, 8, 64, 32, 7), (16, 4, 128, 64, 1), (16, 1, 256, 48, 33), (3, 3, 16, 16, 64),
                                            (6, 2, 96, 80, 24), (10, 2, 240, 128, 12), (40, 1, 80, 32, 3), (64, 1, 32, 16, 64)])
def test_tree_shapes(gpu, codes, dtype, Hq, Hk, D, page, N):
    lens = [N, N + 1, N + 16, N + 63, 64 * 3, N + 200, 128 - N % 3, 0, max(1, N // 2)]
    check_trees(lens, N, Hq, Hk, D, page, codes, dtype, gpu)


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (5, 300), (64, 4), (300, 65)])
def test_tree_windows(gpu, codes, dtype, window, sinks):
    """A window shorter than the ways through the tree, sinks that reach into it."""
    check_trees([24, 40, 300, 700, 64, 65], 24, 6, 2, 64, 16, codes, dtype, gpu, window=window, sinks=sinks)


def test_tree_counts(gpu):
    """Fewer drafts than rows, none, more than the sequence has; a chain, all from the text, parents that are none."""
    N = 20
    drafts = [20, 7, 0, 1, 20, 64]
    lens = [100, 90, 130, 1, 5, 33]
    for codes, dtype in (("none", torch.float16), ("int8", torch.bfloat16)):
        check_trees(lens, N, 6, 2, 64, 16, codes, dtype, gpu, drafts=drafts)
        for parents in ([i - 1 for i in range(N)], [-1] * N, [-7, 1, 2, 50, 2 ** 31 - 1, -2 ** 31] + [0] * (N - 6)):
            check_trees(lens, N, 6, 2, 64, 16, codes, dtype, gpu, drafts=drafts, parents=[parents] * 6)
            check_trees(lens, N, 6, 2, 64, 16, codes, dtype, gpu, window=4, sinks=2, parents=[parents] * 6)


@pytest.mark.parametrize("codes,dtype", TYPES)
def test_tree_long(gpu, codes, dtype):
    check_trees([9000, 64, 4097, 5000], 64, 10, 2, 128, 64, codes, dtype, gpu, seed=5)
    check_trees([20000], 5, 8, 1, 64, 16, codes, dtype, gpu, seed=6)


def test_chain_is_the_prompt(gpu):
    """A tree that is one chain has a prompt's rows and the single token's."""
    from powershard_amd import ops
    N, lens = 9, [200, 9, 70]
    for codes, dtype in TYPES:
        q, k, v, table, lengths, ks, vs = make(lens, 8, 2, 128, 16, codes, dtype, gpu, seed=8)
        rows = torch.randn(3, N, 8, 128, generator=seeded(2)).to(dtype).to(gpu)
        chain = torch.arange(-1, N - 1, dtype=torch.int32, device=gpu).repeat(3, 1)
        starts = torch.arange(4, dtype=torch.int32, device=gpu) * N
        for kw in ({}, dict(window=33, sinks=5)):
            a = ops.paged_tree_attention(rows, k, v, table, lengths, chain, ks, vs, **kw)
            b = ops.paged_prompt_attention(rows.view(-1, 8, 128), k, v, table, starts, lengths, ks, vs, **kw)
            assert torch.equal(a.view(-1, 8, 128), b)


# ------------------------------------------------------------------------------- what masks hide
@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_masks_hide_reaches_nobody(gpu, codes, dtype, value):
    """Keys and values of a token that are not finite reach the rows that see it, and them alone."""
    from powershard_amd import ops
    new, n, D, page = 90, 170, 64, 16
    q, pools, starts = prompts([(new, n)], 4, 2, D, page, codes, dtype, gpu, seed=4)
    k, v, table, lengths, ks, vs = pools
    token, dim = 130, 37                                 # seen from position 130 on, with a window to 149
    pg, off = int(table[0, token // page]), token % page
    call = lambda **kw: ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, **kw)
    for kw, sees in ((dict(), lambda p: p >= token), (dict(window=20), lambda p: token <= p < token + 20),
                     (dict(window=20, sinks=131), lambda p: p >= token), (dict(window=20, sinks=130), lambda p: token <= p < token + 20)):
        clean = call(**kw)
        rows = torch.tensor([sees(n - new + i) for i in range(new)], device=gpu)
        assert rows.any() and not rows.all()
        for which in ("k", "v"):
            pool, scales = (k, ks) if which == "k" else (v, vs)
            where = (pg, 1, off)
            if codes == "none":
                old = pool[where].clone()
                pool[where][dim] = value
            else:
                old = scales[where].clone()
                scales[where] = value
            got = call(**kw)
            if codes == "none":
                pool[where] = old
            else:
                scales[where] = old
            assert torch.equal(got[:, :2], clean[:, :2])              # of the other kv head
            assert torch.equal(got[~rows], clean[~rows])
            mine = got[rows][:, 2:].float()
            if which == "v" and codes == "none":
                hit = mine[..., dim]
                assert hit.isnan().all() if math.isnan(value) else (hit == value).all()
                rest = torch.arange(D, device=gpu) != dim
                assert torch.equal(got[rows][:, 2:][..., rest], clean[rows][:, 2:][..., rest])
            elif which == "v":
                assert not mine.isfinite().all(-1).any()


@pytest.mark.parametrize("codes,dtype", [("none", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16)])
def test_bad_pages(gpu, codes, dtype):
    """A row that sees a token whose page is not there gets NaN, the others what they had."""
    from powershard_amd import ops
    new, n, page = 100, 400, 32
    q, pools, starts = prompts([(new, n), (30, 64)], 4, 2, 128, page, codes, dtype, gpu, seed=6)
    k, v, table, lengths, ks, vs = pools
    for kw in (dict(), dict(window=40, sinks=3)):
        clean = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, **kw)
        for col in (0, 10, 11, 12):
            for bad in (-1, k.shape[0], 2 ** 31 - 1):
                broken = table.clone()
                broken[0, col] = bad
                seen = causal(new, n, kw.get("window", 0), kw.get("sinks", 0), gpu)[:, col * page:(col + 1) * page].any(1)
                got = ops.paged_prompt_attention(q, k, v, broken, starts, lengths, ks, vs, **kw)
                assert got[:new][seen].isnan().all() and torch.equal(got[:new][~seen], clean[:new][~seen])
                assert torch.equal(got[new:], clean[new:])
    cut = table[:, :12].contiguous()                     # tokens past the table
    got = ops.paged_prompt_attention(q, k, v, cut, starts, lengths, ks, vs)
    clean = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs)
    seen = torch.arange(new, device=gpu) + n - new >= 12 * page
    assert got[:new][seen].isnan().all() and torch.equal(got[:new][~seen], clean[:new][~seen]) and torch.equal(got[new:], clean[new:])
    none = torch.empty((2, 0), dtype=torch.int32, device=gpu)
    assert ops.paged_prompt_attention(q, k, v, none, starts, lengths, ks, vs).isnan().all()


def test_lengths_and_starts_that_do_not_fit(gpu):
    """More rows than tokens: those in front of the text get zeros; starts and lengths out of range stay in bounds."""
    from powershard_amd import ops
    q, pools, starts = prompts([(20, 50)], 4, 2, 64, 16, "none", torch.bfloat16, gpu)
    k, v, table, lengths, _, _ = pools
    clean = ops.paged_prompt_attention(q, k, v, table, starts, lengths)
    short = ops.paged_prompt_attention(q, k, v, table, starts, torch.tensor([7], dtype=torch.int32, device=gpu))
    assert (short[:13] == 0).all() and not short.isnan().any() and (short[13:] != 0).any(-1).all()
    for lens in (0, -5):
        assert (ops.paged_prompt_attention(q, k, v, table, starts, torch.tensor([lens], dtype=torch.int32, device=gpu)) == 0).all()
    got = ops.paged_prompt_attention(q, k, v, table, torch.tensor([0, 99], dtype=torch.int32, device=gpu), lengths)
    assert torch.equal(got, clean)
    got = ops.paged_prompt_attention(q, k, v, table, torch.tensor([5, 2], dtype=torch.int32, device=gpu), lengths)
    assert got.shape == q.shape


@pytest.mark.parametrize("codes,dtype", [("none", torch.float16), ("int8", torch.bfloat16)])
def test_layouts(gpu, codes, dtype):
    """Strided and misaligned queries, strided tables, lengths and starts."""
    from powershard_amd import ops
    shapes = [(20, 50), (3, 3)]
    q, pools, starts = prompts(shapes, 4, 2, 64, 16, codes, dtype, gpu)
    k, v, table, lengths, ks, vs = pools
    clean = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs)
    two = lambda t: torch.stack([t, t], -1).flatten(-2)[..., ::2]
    odd = torch.cat([torch.zeros(1, dtype=dtype, device=gpu), q.reshape(-1)])[1:].view(q.shape)
    for other in (two(q), odd, q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([q, q], 1)[:, 4:]):
        assert torch.equal(ops.paged_prompt_attention(other, k, v, two(table), two(starts), two(lengths), ks, vs), clean)
    wide = torch.cat([table, table], 1)[:, :table.shape[1]]
    assert torch.equal(ops.paged_prompt_attention(q, k, v, wide, starts, lengths, ks, vs), clean)
    assert ops.paged_prompt_attention(q[:0], k, v, table, torch.zeros(3, dtype=torch.int32, device=gpu), lengths, ks, vs).shape == (0, 4, 64)
    assert ops.paged_prompt_attention(q[:, :0], k, v, table, starts, lengths, ks, vs).shape == (23, 0, 64)
    nobody = ops.paged_prompt_attention(q, k, v, table[:0], starts[:1], lengths[:0], ks, vs)
    assert (nobody == 0).all()
    rows = torch.randn(2, 3, 4, 64, generator=seeded(1)).to(dtype).to(gpu)
    parents = torch.tensor([[-1, 0, 0], [-1, -1, 1]], dtype=torch.int32, device=gpu)
    tree = ops.paged_tree_attention(rows, k, v, table, lengths, parents, ks, vs)
    assert torch.equal(ops.paged_tree_attention(rows.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, lengths, two(parents), ks, vs), tree)
    assert ops.paged_tree_attention(rows[:, :0], k, v, table, lengths, parents[:, :0], ks, vs).shape == (2, 0, 4, 64)
    assert ops.paged_tree_attention(rows[:0], k, v, table[:0], lengths[:0], parents[:0], ks, vs).shape == (0, 3, 4, 64)


def test_refusals(gpu):
    from powershard_amd import ops
    q, pools, starts = prompts([(20, 50)], 4, 2, 64, 16, "int8", torch.bfloat16, gpu)
    k, v, table, lengths, ks, vs = pools

    def prompt(q=q, k=k, v=v, table=table, starts=starts, lengths=lengths, ks=ks, vs=vs, **kw):
        return ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, **kw)

    parents = torch.full((1, 20), -1, dtype=torch.int32, device=gpu)

    def tree(q=q[None], k=k, v=v, table=table, lengths=lengths, parents=parents, ks=ks, vs=vs, **kw):
        return ops.paged_tree_attention(q, k, v, table, lengths, parents, ks, vs, **kw)
    prompt(), tree()
    for call, bad in ((prompt, dict(q=q.float())), (tree, dict(q=q[None].float())), (prompt, dict(k=k.bfloat16(), v=v))):
        with pytest.raises(TypeError):
            call(**bad)
    for call, bad in [(prompt, dict(q=q[None])), (prompt, dict(q=q[:, :3])), (prompt, dict(q=q[..., :32])), (prompt, dict(starts=starts.long())),
                      (prompt, dict(starts=starts[:1])), (prompt, dict(lengths=lengths.long())), (prompt, dict(table=table.long())),
                      (prompt, dict(table=table[0])), (prompt, dict(window=-1)), (prompt, dict(sinks=4)), (prompt, dict(window=4, sinks=-1)),
                      (prompt, dict(ks=None)), (tree, dict(q=q)), (tree, dict(parents=parents.long())), (tree, dict(parents=parents[:, :3])),
                      (tree, dict(drafts=lengths.long())), (tree, dict(drafts=parents[0])), (tree, dict(lengths=torch.cat([lengths, lengths]))),
                      (tree, dict(q=q.new_zeros(1, 65, 4, 64), parents=parents.new_zeros(1, 65))), (tree, dict(sinks=1))]:
        with pytest.raises(ValueError):
            call(**bad)
    for call, bad in [(prompt, dict(starts=starts.cpu())), (prompt, dict(table=table.cpu())), (prompt, dict(k=k.cpu())), (prompt, dict(q=q.cpu())),
                      (tree, dict(parents=parents.cpu())), (tree, dict(drafts=lengths.cpu()))]:
        with pytest.raises(RuntimeError):
            call(**bad)
