"""The rotary write, the prompts', the steps' and the trees' attention together: through the cache and the decoder layer,
captured into graphs, on streams side by side; and lengths past the table."""
import threading

import pytest
import torch
from torch import nn

from conftest import heavy_rows
from test_block_attention_gpu import check_prompts, prompts
from test_decoder_gpu import DIM, HEADS, HIDDEN, KV, ROT, decoder
from test_paged_attention_gpu import TYPES

pytestmark = pytest.mark.gpu

WAYS = [([-1, 0, 0, 2, -1, 1], [0, 2, 3]), ([-1, -1, 1, 2, 0, 0], [1, 2])]    # trees of six drafts, the way that is kept


def rotary(kind):
    from powershard_amd.decoder import Rotary
    if kind == "axes":
        return Rotary(DIM, base=300.0, axes=[0] * 8 + [1] * 12 + [2] * 12)
    return Rotary(48, base=1e6, interleaved=True) if kind == "part" else Rotary(DIM)


def forward(layers, form, x, cache, slots, *where, **options):
    h = None
    for i, layer in enumerate(layers):
        x, h = getattr(layer, form)(x, h, cache, i, *((where[0], slots) if form == "prompt" else (slots, where[0])), **options)
    return x.float() + h.float()


def run_prompts(layers, cache, seqs, texts):
    slots = cache.extend(seqs, [len(t) for t in texts])
    y = forward(layers, "prompts", torch.cat(texts), cache, slots, cache.prompts(seqs, [len(t) for t in texts]))
    return y.split([len(t) for t in texts])


def run_step(layers, cache, seqs, x):
    slots = cache.extend(seqs, 1)
    return forward(layers, "step", x, cache, slots, cache.table(seqs))


def run_drafts(layers, cache, seqs, x, parents):
    slots = cache.extend(seqs, x.shape[1])
    return forward(layers, "drafts", x.reshape(-1, x.shape[-1]), cache, slots, cache.drafts(seqs, parents)).view(x.shape)


def whole_run(layers, cache, texts, tail):
    """[(outputs, rows of the inputs they are of)] of: ragged prompts, a second part of them, two steps, a tree of drafts of
    which one way stays, a step, and the first sequence's prompt by itself."""
    seqs, said = [cache.open() for _ in texts], [[] for _ in texts]
    def saw(i, y, rows):
        said[i].append((y, list(rows)))
    cut = [n - 7 - 3 * i for i, n in enumerate(len(t) - tail for t in texts)]
    for a, b in ((0, 0), (0, 1)):
        part = [t[:c] if b == 0 else t[c:len(t) - tail] for t, c in zip(texts, cut)]
        for i, y in enumerate(run_prompts(layers, cache, seqs, part)):
            at = 0 if b == 0 else cut[i]
            saw(i, y, range(at, at + len(y)))
    at = [len(t) - tail for t in texts]
    for _ in range(2):
        y = run_step(layers, cache, seqs, torch.stack([t[a] for t, a in zip(texts, at)]))
        for i in range(len(seqs)):
            saw(i, y[i:i + 1], [at[i]])
            at[i] += 1
    n = len(WAYS[0][0])
    x = torch.stack([t[a] for t, a in zip(texts, at)])[:, None].repeat(1, n, 1).flip(0)    # (wrong drafts are other rows)
    for i, (_, way) in enumerate(WAYS):
        for d, k in enumerate(way):
            x[i, k] = texts[i][at[i] + d]
    y = run_drafts(layers, cache, seqs, x, [p for p, _ in WAYS])
    for i, (_, way) in enumerate(WAYS):
        cache.accept(seqs[i], n, way)
        saw(i, y[i, way], range(at[i], at[i] + len(way)))
        at[i] += len(way)
    y = run_step(layers, cache, seqs, torch.stack([t[a] for t, a in zip(texts, at)]))
    for i in range(len(seqs)):
        saw(i, y[i:i + 1], [at[i]])
    slots = cache.extend(seqs[:1], 2)
    saw(0, forward(layers, "prompt", texts[0][at[0] + 1:at[0] + 3], cache, slots, seqs[0]), [at[0] + 1, at[0] + 2])
    return said


def formula(layers, weights, x):
    """The layers on one text, in 64 bits."""
    n = len(x)
    h, y, at = torch.zeros(n, HIDDEN, dtype=torch.float64), x.double().cpu(), torch.arange(n)
    for layer, w in zip(layers, weights):
        def norm(t, g):
            return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g
        rot = layer.rotary
        freq, _ = rot.on(torch.device("cpu"))
        t = at[:, None, None] * freq

        def turn(r):
            a, b = (r[..., 0:rot.dim:2], r[..., 1:rot.dim:2]) if rot.interleaved else (r[..., :rot.dim // 2], r[..., rot.dim // 2:rot.dim])
            a, b = a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()
            ab = torch.stack([a, b], -1).flatten(-2) if rot.interleaved else torch.cat([a, b], -1)
            return torch.cat([ab, r[..., rot.dim:]], -1)
        h = h + y
        rows = norm(h, w["norm1"])
        q, k, v = ((rows @ w[m + "_proj"].T).reshape(n, -1, DIM) for m in "qkv")
        q, k = turn(q), turn(k)
        seen = at <= at[:, None]
        if layer.window:
            seen &= (at > at[:, None] - layer.window) | (at < layer.sinks)
        out = torch.zeros(n, HEADS, DIM, dtype=torch.float64)
        for i in range(HEADS):
            s = (q[:, i] @ k[:, i * KV // HEADS].T / DIM ** 0.5).masked_fill(~seen, float("-inf"))
            out[:, i] = torch.softmax(s, -1) @ v[:, i * KV // HEADS]
        h = h + out.reshape(n, -1) @ w["o_proj"].T
        gate, up = (norm(h, w["norm2"]) @ w["up_proj"].T).chunk(2, -1)
        y = (nn.functional.silu(gate) * up) @ w["down_proj"].T
    return h + y


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("kind", ["whole", "part", "axes"])
def test_run_against_64_bits(gpu, kind, window, sinks):
    """Weight-only layers on a 16-bit cache: only bf16 roundings (about 20 a layer on the way, 2^-9 rms each, so
    sqrt(40) 2^-9 of the norm, 1.3%; bound 2^-5) separate the run from the formula."""
    from powershard_amd.kv_cache import PagedKVCache
    layers, weights = decoder("int4", {"group_size": 128}, gpu)
    for layer in layers:
        layer.rotary, layer.window, layer.sinks = rotary(kind), window, sinks
    texts = [heavy_rows(n, HIDDEN, 60 + n, outlier_frac=0).to(gpu) for n in (49, 90)]
    with torch.no_grad():
        said = whole_run(layers, PagedKVCache(2, 12, 16, KV, DIM, device=gpu), texts, 9)
    for t, parts in zip(texts, said):
        want = formula(layers, weights, t)
        for y, rows in parts:
            assert (y.double().cpu() - want[rows]).norm() <= 2.0 ** -5 * want[rows].norm(), rows


@pytest.mark.parametrize("codes", [None, "int8", "fp8"])
@pytest.mark.parametrize("fmt,opts", [("int8", ROT), ("fp8", {})])
def test_run_equals_the_prompt(gpu, fmt, opts, codes):
    """All forms against all of the text as one prompt.  They see the same codes in the cache and differ in the order of
    fp32 sums, so in the roundings of attention outputs that this turns over, and in the codes that those turn over:
    bound 2 layers x 4 linears x 2^-8 of the rows' norm for int8 rows, whose half step is 2^-8 of a row's maximum.
    A row of e4m3 codes has errors of at most half a step, 2^-4 of each value, 2^-4 / sqrt(3) rms.  What is turned over
    behind a first linear turns over more (a change of d of a value's size crosses an edge with d / step and is then a
    step: d becomes sqrt(d step), which grows to the step's own size), so by the end the two runs' roundings are as good as
    independent: sqrt(2 / 3) 2^-4 of the row's norm for each of 2 x 4 linears, whose own roundings are independent too:
    sqrt(8) sqrt(2 / 3) 2^-4 in all, as no branch is larger than the sum that it goes into."""
    from powershard_amd.kv_cache import PagedKVCache
    layers, _ = decoder(fmt, opts, gpu)
    bound = 2.0 ** -5 if fmt == "int8" else (16 / 3) ** 0.5 * 2.0 ** -4
    for layer in layers:
        layer.rotary, layer.window, layer.sinks = rotary("whole"), 40, 2
    texts = [heavy_rows(n, HIDDEN, 80 + n, outlier_frac=0).to(gpu) for n in (49, 90)]
    with torch.no_grad():
        said = whole_run(layers, PagedKVCache(2, 12, 16, KV, DIM, codes=codes, device=gpu), texts, 9)
        cache = PagedKVCache(2, 12, 16, KV, DIM, codes=codes, device=gpu)
        wants = run_prompts(layers, cache, [cache.open() for _ in texts], texts)
    for want, parts in zip(wants, said):
        for y, rows in parts:
            assert (y - want[rows]).norm() <= bound * want[rows].norm(), rows


def test_positions_of_several_axes(gpu):
    """Positions given to a layer: its prompt equals the one by its parts, and differs from that of the places."""
    from powershard_amd.kv_cache import PagedKVCache
    layers, _ = decoder("int4", {"group_size": 128}, gpu)
    for layer in layers:
        layer.rotary = rotary("axes")
    x = heavy_rows(24, HIDDEN, 9, outlier_frac=0).to(gpu)
    p = torch.stack([torch.zeros(24), torch.arange(24) // 6, torch.arange(24) % 6]).int().to(gpu)
    with torch.no_grad():
        def run(parts, positions):
            cache = PagedKVCache(2, 4, 16, KV, DIM, device=gpu)
            seq, out = cache.open(), []
            for a, b in parts:
                slots = cache.extend([seq], b - a)
                where = cache.prompts([seq], [b - a])
                out.append(forward(layers, "prompts", x[a:b], cache, slots, where, positions=positions and p[:, a:b]))
            return torch.cat(out)
        whole, parts, places = run([(0, 24)], True), run([(0, 10), (10, 24)], True), run([(0, 24)], None)
    assert (whole - parts).norm() <= 2.0 ** -5 * whole.norm() and (whole - places).norm() > 2.0 ** -5 * whole.norm()


def test_plain_layer_is_unchanged(gpu):
    """A layer without a rotary runs the operations that it ran: the same bits, whatever another layer has."""
    from powershard_amd.decoder import prompt_attention, rope
    from powershard_amd.kv_cache import PagedKVCache
    (layer,), _ = decoder("int8", ROT, gpu, layers=1)
    x = heavy_rows(20, HIDDEN, 4, outlier_frac=0).to(gpu)
    with torch.no_grad():
        cache, other = (PagedKVCache(1, 4, 16, KV, DIM, codes="int8", device=gpu) for _ in range(2))
        seq = cache.open()
        slots = cache.extend([seq], 20)
        y, h = layer.prompt(x, None, cache, 0, seq, slots)
        q, k, v, r = layer._unturned(x, None)
        at = torch.arange(20, device=gpu)
        other.write(0, rope(k, at), v, slots)
        want, s = layer._rest(prompt_attention(rope(q, at), *other.read(0, slots, torch.float32), 0), r)
    assert torch.equal(y, want) and torch.equal(h, s) and torch.equal(cache.k, other.k)


def make_calls(gpu, codes, seed):
    """(caches, inputs, call): append, prompts' attention over split key tiles, trees' attention and a step's."""
    from powershard_amd.kv_cache import PagedKVCache
    B, H, D, N, new = 3, 8, 128, 5, 9
    g = torch.Generator(device=gpu).manual_seed(seed)
    freq = 10000.0 ** (-torch.arange(D // 2, device=gpu, dtype=torch.float64) / (D // 2))
    inputs = dict(q=torch.zeros(B * new, H, D, device=gpu).bfloat16(), k=torch.zeros(B * new, 2, D, device=gpu).bfloat16(),
                  v=torch.zeros(B * new, 2, D, device=gpu).bfloat16(), slots=torch.full((B * new,), -1, dtype=torch.int64, device=gpu),
                  table=torch.full((B, 80), -1, dtype=torch.int32, device=gpu), lengths=torch.zeros(B, dtype=torch.int32, device=gpu),
                  positions=torch.zeros(B * new, dtype=torch.int32, device=gpu),
                  parents=torch.full((B, N), -1, dtype=torch.int32, device=gpu),
                  starts=torch.arange(0, B * new + 1, new, dtype=torch.int32, device=gpu))

    def cache():
        c = PagedKVCache(1, 240, 16, 2, D, codes=codes, device=gpu)
        past, seqs = torch.Generator(device=gpu).manual_seed(seed), [c.open() for _ in range(B)]
        for s, n in zip(seqs, (1000, 0, 333)):
            x = torch.randn(n, 2, 2, D, generator=past, device=gpu).bfloat16()
            c.write(0, x[:, 0], x[:, 1], c.extend([s], n))
        return c, seqs

    def fill(c, seqs):
        slots = c.extend(seqs, new)
        for name in ("q", "k", "v"):
            inputs[name].normal_(generator=g)
        where = c.prompts(seqs, [new] * B)
        inputs["slots"].copy_(slots)
        inputs["table"][:, :where.block_table.shape[1]] = where.block_table
        inputs["lengths"].copy_(where.lengths)
        inputs["positions"].copy_(where.positions)
        inputs["parents"].copy_((torch.rand(B, N, device=gpu, generator=g) * torch.arange(N + 1, device=gpu)[1:]).int() - 1)

    def call(c):
        from powershard_amd.kv_cache import Drafts, Prompts
        i = inputs
        where = Prompts(i["table"], i["lengths"], 1280, i["starts"], i["positions"])
        q = c.append(0, i["q"], i["k"], i["v"], i["positions"], freq, i["slots"])
        prompt = c.attend_prompts(0, q, where, return_lse=True)
        tree = c.attend_drafts(0, q.view(B, new, H, D)[:, new - N:], Drafts(i["table"], i["lengths"], 1280, i["parents"], None), window=300, sinks=70)
        step = c.attend(0, q.view(B, new, H, D)[:, -1], i["table"], i["lengths"], 1280, window=300, sinks=7)
        return (q, *prompt, tree, step)
    return cache, fill, call


@pytest.mark.parametrize("codes", [None, "int8", "fp8"])
def test_run_in_a_graph(gpu, codes):
    """Captured once and replayed as the texts grow, with eager work in between: every replay has the eager call's bits."""
    cache, fill, call = make_calls(gpu, codes, 1)
    (c0, s0), (c1, s1) = cache(), cache()
    stream = torch.cuda.Stream(gpu)
    stream.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(stream):
        call(c0)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = call(c0)
    for _ in range(5):
        fill(c0, s0)
        c1.extend(s1, 9)
        graph.replay()
        got = [t.clone() for t in captured]
        want = call(c1)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b) and not a.isnan().any()
        assert torch.equal(c0.k.view(torch.uint8), c1.k.view(torch.uint8))


def test_side_by_side(gpu):
    """Two host threads with a stream each, and two graphs of the same calls replayed side by side: the bits of one alone."""
    made = [make_calls(gpu, "int8", seed) for seed in (1, 2)]
    caches = [m[0]() for m in made]
    for m, (c, s) in zip(made, caches):
        m[1](c, s)
    want = [[t.clone() for t in m[2](c)] for m, (c, _) in zip(made, caches)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(gpu) for _ in made], [None, None]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i] = made[i][2](caches[i][0])
        streams[i].synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in made], []
    for graph, stream, m, (c, _) in zip(graphs, streams, made, caches):
        with torch.cuda.graph(graph, stream=stream):
            outs.append(m[2](c))
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
            for x in a:
                x.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("far", [300, 2 ** 30, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 70])
def test_lengths_past_the_table(gpu, codes, dtype, far, new):
    """A length past the table: NaN in the rows that see past it (all of those whose token is there), the others right:
    two ways of cutting the keys, each within 2^-8 sum p |v| + 2^-8 |o| of the formula, so 2^-6 of the largest value."""
    from powershard_amd import ops
    shapes = [(new, 300), (new, 250)]
    q, (k, v, table, lengths, ks, vs), starts = prompts(shapes, 8, 2, 64, 64, codes, dtype, gpu)
    lengths = lengths.clone()
    table = table[:, :5].contiguous()      # 320 tokens
    want = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs).float()
    near = 2.0 ** -6 * float((v.float() if vs is None else v.float() * vs[..., None]).nan_to_num(0, 0, 0).abs().max())
    lengths[0] = min(320 + far, 2 ** 31 - 1)
    for max_len in (None, 64):             # (cut into runs, and whole)
        got, lse = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs, max_len=max_len, return_lse=True)
        assert got[:new].isnan().all() and lse[:new].isnan().logical_or(lse[:new] == -torch.inf).all()
        assert ((got[new:].float() - want[new:]).abs() <= near).all()
        tree = ops.paged_tree_attention(q.view(2, new, 8, 64)[:, -1:], k, v, table, lengths, torch.full((2, 1), -1, dtype=torch.int32, device=gpu), ks, vs,
                                        max_len=max_len)
        assert tree[0].isnan().all() and ((tree[1, 0].float() - want[-1]).abs() <= near).all()
    lengths[0] = 325                       # the last five tokens past the table, the twenty in front of them NaN in the cache
    got = ops.paged_prompt_attention(q, k, v, table, starts, lengths, ks, vs)
    assert got[max(new - 25, 0):new].isnan().all() and not got[:max(new - 25, 0)].isnan().any()


@pytest.mark.parametrize("codes", [torch.bfloat16, torch.int8])
def test_pools_past_4_gib(gpu, codes):
    """Pages whose bytes lie past 2^32: the bits of the same pages at the pool's start."""
    from powershard_amd import ops
    H, Hk, D, page, n = 8, 8, 128, 64, 9
    pages = 2 ** 33 // (Hk * page * D * codes.itemsize) // 2 * 9 // 8        # 4.5 GiB
    g = torch.Generator(device=gpu).manual_seed(3)
    small = [torch.zeros(n, Hk, page, D, dtype=codes, device=gpu) for _ in range(2)]
    small += [None, None] if codes is torch.bfloat16 else [torch.ones(n, Hk, page, device=gpu) for _ in range(2)]
    large = [t if t is None else torch.empty((pages,) + t.shape[1:], dtype=t.dtype, device=gpu) for t in small]
    q, k, v = (torch.randn(n * page, h, D, generator=g, device=gpu).bfloat16() for h in (H, Hk, Hk))
    at, freq = torch.arange(n * page, dtype=torch.int32, device=gpu), 100.0 ** (-torch.arange(64, device=gpu).double() / 64)
    table = torch.randperm(n, generator=g, device=gpu)[None].int()
    slots = table[0].long().repeat_interleave(page) * page + torch.arange(page, device=gpu).repeat(n)
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([n * page], [0, 100]))
    parents = torch.arange(-1, 15, dtype=torch.int32, device=gpu)[None]
    got = []
    for pools, first in ((small, 0), (large, pages - n)):
        turned = ops.rope_kv_write(q, k, v, at, freq, slots + first * page, *pools)
        where = table + first
        got.append([turned, *ops.kv_read(slots + first * page, *pools),
                    ops.paged_prompt_attention(turned[-100:], *pools[:2], where, starts, lengths, *pools[2:]),
                    ops.paged_tree_attention(turned[-16:][None], *pools[:2], where, lengths, parents, *pools[2:]),
                    ops.paged_attention(turned[-1:], *pools[:2], where, lengths, *pools[2:], window=100, sinks=70)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and not a.isnan().any()
