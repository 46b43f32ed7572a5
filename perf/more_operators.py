"""The measured operators of a text decoder's attention over its paged key-value cache beyond one new
token: keys turned to their positions as they are appended (with the queries), prompts that attend to the
cache, trees of drafted tokens, and windows whose first tokens stay visible.

A case is one call that a decoder makes per layer.  ``run`` computes it either with the package's operators
(``own``) or in plain torch operations in 32 bits (angles in 64).

Layouts: caches [pages, kv heads, page size, head dim], their scales [pages, kv heads, page size], one page
table row per sequence, slot = page * page size + offset.  Everything past a sequence's length, and every
page that no sequence holds, is NaN (garbage, for int8 codes), as memory that nobody has written may be.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
DEVICE = "cuda:0"
GOLDEN = 0.6180339887498949


def _append(name, tokens, first, heads, kv_heads, dim, page, dtype, codes, rotary=0, axes=1, interleaved=False):
    """tokens at positions first, first + 1, ... (axes 3: of images of 32 x 48 patches in a video, in turn)."""
    return dict(name=name, kind="append", tokens=tokens, first=first, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, rotary=rotary or dim, axes=axes, interleaved=interleaved)


def _step(name, batch, max_len, heads, kv_heads, dim, page, dtype, codes, window, sinks):
    return dict(name=name, kind="step", batch=batch, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, window=window, sinks=sinks)


def _prompt(name, batch, new, past, heads, kv_heads, dim, page, dtype, codes="none", window=0, sinks=0):
    """batch sequences of up to `new` new tokens after up to `past` cached ones."""
    return dict(name=name, kind="prompt", batch=batch, new=new, past=past, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, window=window, sinks=sinks)


def _tree(name, batch, drafts, max_len, heads, kv_heads, dim, page, dtype, codes="none", window=0, sinks=0):
    """batch sequences of up to max_len tokens, the last `drafts` of which are a tree."""
    return dict(name=name, kind="tree", batch=batch, drafts=drafts, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, codes=codes, window=window, sinks=sinks)


def listed():
    return [
        # the next token of one user, far into a text, onto an int8 cache: latency
        _append("append_i8_token_t1", 1, 100003, 40, 8, 128, 16, "bf16", "int8"),
        # the frames of a short video in a prompt: time, height and width turn a part of the dims each
        _append("append_f16_video_t4095", 4095, 77, 64, 16, 64, 32, "f16", "none", axes=3, interleaved=True),
        # a whole prompt onto an fp8 cache
        _append("append_fp8_prompt_t8191", 8191, 0, 40, 8, 128, 64, "bf16", "fp8"),
        # a batch of users of a layer that sees the last 1024 tokens and the first 4
        _step("step_f16_window_b16", 16, 8192, 64, 16, 64, 32, "f16", "none", 1024, 4),
        # many users, a wide window and 64 tokens of instructions that all of them keep
        _step("step_i8_window_b64", 64, 16384, 40, 8, 128, 16, "bf16", "int8", 4096, 64),
        # one short prompt, as many kv heads as heads: latency
        _prompt("prompt_bf16_short_t77", 1, 77, 0, 40, 40, 128, 16, "bf16"),
        # prompts of ragged lengths that go on from cached ones, in a layer with a window and sinks
        _prompt("prompt_f16_window_b7", 7, 4095, 2000, 64, 16, 64, 32, "f16", window=1024, sinks=4),
        # one long prompt, all of it at once
        _prompt("prompt_bf16_long_t8191", 1, 8191, 0, 40, 8, 128, 64, "bf16"),
        # the last chunk of a very long prompt on an int8 cache
        _prompt("prompt_i8_chunk_t512", 1, 512, 64977, 40, 8, 128, 64, "f16", "int8"),
        # a small tree of drafts of one user: latency
        _tree("tree_bf16_n16", 1, 16, 4000, 40, 8, 128, 16, "bf16"),
        # trees of a batch of users of ragged lengths
        _tree("tree_i8_b61_n24", 61, 24, 4096, 40, 8, 128, 16, "bf16", "int8"),
        # a large tree deep in a very long text
        _tree("tree_fp8_long_n64", 1, 64, 131071, 40, 8, 128, 64, "bf16", "fp8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 8192 new tokens of 1 to 128 sequences after up to 131072 cached ones, trees of 1 to
    64 drafts, windows with 0 to 256 sinks; head dims of 16 to 256, 1 to 64 heads, shared or not; every type."""
    kind = rng.choice(["append", "step", "prompt", "prompt", "tree", "tree"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    codes = rng.choice(["int8", "fp8", "none", "none"])
    dim = rng.choice([64, 128, 128, 128, 256, 16 * rng.randint(1, 16)])
    page = rng.choice([16, 32, 64, 128, 16 * rng.randint(1, 16)])
    kv_heads = rng.choice([1, 2, 4, 8, 8, rng.randint(1, 40)])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16, rng.randint(1, 64)])
    group = max(1, min(group, 64 // kv_heads))
    heads = group * kv_heads
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        while tokens * (heads + 2 * kv_heads) * dim > 8191 * 56 * 128:
            tokens = max(1, tokens // 2)
        rotary = dim if rng.random() < 0.7 else 16 * rng.randint(1, dim // 16)
        return dict(kind=kind, tokens=tokens, first=rng.choice([0, _log(rng, 1, 131072)]), heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, dtype=dtype, codes=codes, rotary=rotary, axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.4)
    window = _log(rng, 1, 8192) if kind == "step" or rng.random() < 0.3 else 0
    sinks = rng.choice([0, 1, 4, 64, rng.randint(0, 256)]) if window else 0
    if kind == "step":
        batch, max_len = _log(rng, 1, 128), _log(rng, 1, 131072)
        # no more cache than the largest listed case
        while batch * max_len * kv_heads * dim > 64 * 16384 * 8 * 128:
            batch, max_len = (max(1, batch // 2), max_len) if batch > 1 else (batch, max_len // 2)
        return dict(kind=kind, batch=batch, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                    codes=codes, window=window, sinks=sinks)
    if kind == "prompt":
        batch, new, past = _log(rng, 1, 16), _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 65536)])
        # no more products (nor cache) than the largest listed case, as if there were no window
        while batch * new * (new / 2 + past) * heads * dim > 8191 * 4096 * 40 * 128 or batch * (new + past) * kv_heads * dim > 131072 * 8 * 128:
            if batch > 1:
                batch //= 2
            elif past > new:
                past //= 2
            else:
                new = max(1, new // 2)
        return dict(kind=kind, batch=batch, new=new, past=past, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                    codes=codes, window=window, sinks=sinks)
    drafts = _log(rng, 1, 64)
    batch, max_len = _log(rng, 1, 128), _log(rng, drafts, 131072)
    while batch * max_len * heads * dim * drafts > 8191 * 4096 * 40 * 128 or batch * max_len * kv_heads * dim > 4 * 131072 * 8 * 128:
        batch, max_len = (max(1, batch // 2), max_len) if batch > 1 else (batch, max(drafts, max_len // 2))
    return dict(kind=kind, batch=batch, drafts=drafts, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, window=window, sinks=sinks)


# ------------------------------------------------------------------------------- inputs
def _ragged(longest, batch, least=0):
    """Ragged lengths that the case alone sets: spread evenly over least .. longest, the longest among them."""
    return [longest if b == 0 else least + int((longest - least) * ((b * GOLDEN) % 1.0)) for b in range(batch)]


def _shapes(case):
    """[(new tokens, all tokens)] of the sequences."""
    if case["kind"] == "prompt":
        new, past = _ragged(case["new"], case["batch"]), _ragged(case["past"], case["batch"])
        return [(n, n + p) for n, p in zip(new, past[::-1])]
    if case["kind"] == "tree":
        return [(case["drafts"], n) for n in _ragged(case["max_len"], case["batch"], case["drafts"])]
    return [(min(n, 1), n) for n in _ragged(case["max_len"], case["batch"])]


def _unwritten(x, valid):
    """x with every row that valid leaves out set to what unwritten memory may hold."""
    if x.dtype != torch.int8:
        one = x.element_size() == 1
        x.view(torch.uint8 if one else torch.int16).masked_fill_(~valid.unsqueeze(-1), 0x7F if one else 0x7FFF)
    return x


def _pools(case, g, pages, valid):
    """K and V pools with their scales; valid [pages, page size]: the slots that hold tokens."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    valid = valid.unsqueeze(1).expand(shape[:3])
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32 if case["codes"] != "none" else DTYPES[case["dtype"]])
        if case["codes"] == "none":
            pools.append(_unwritten(x, valid))
            scales.append(None)
            continue
        code, limit = CODES[case["codes"]]
        x = x.mul_(limit / 3.5).clamp_(-limit, limit)
        pools.append(_unwritten(x.round_().to(code) if code == torch.int8 else x.to(code), valid))
        s = (0.5 + 1.5 * torch.rand(shape[:3], generator=g, device=DEVICE)) * (3.5 / limit)
        scales.append(s.masked_fill_(~valid, float("nan")))
    return dict(k=pools[0], v=pools[1], ks=scales[0], vs=scales[1])


def _cache(case, g, lengths):
    """Pools and page table of sequences of these lengths (on the host)."""
    page, lens = case["page"], torch.tensor(lengths, device=DEVICE)
    held = (lens + page - 1) // page
    pages = sum(-(-n // page) for n in lengths) + 1
    order = torch.randperm(pages, generator=g, device=DEVICE)
    col = torch.arange(max(1, -(-max(lengths) // page)), device=DEVICE)
    first = torch.cumsum(held, 0) - held
    used = col < held.unsqueeze(1)
    # the columns past a sequence's pages hold nothing that may be followed
    table = torch.where(used, order[(first.unsqueeze(1) + col).clamp(max=pages - 1)], -1)
    valid = torch.zeros(pages, page, dtype=torch.bool, device=DEVICE)
    fill = (lens.unsqueeze(1) - col * page).clamp(0, page)
    valid[table[used]] = torch.arange(page, device=DEVICE) < fill[used].unsqueeze(1)
    return dict(_pools(case, g, pages, valid), table=table.to(torch.int32), lengths=lens.to(torch.int32))


def _positions(case):
    """[axes, tokens] int64."""
    at = torch.arange(case["tokens"], device=DEVICE)
    if case["axes"] == 1:
        return (case["first"] + at).unsqueeze(0)
    return case["first"] + torch.stack([at // (32 * 48), at // 48 % 32, at % 48])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed % (1 << 60))
    dtype = DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["kind"] == "append":
        T, page, pairs = case["tokens"], case["page"], case["rotary"] // 2
        pages = -(-T // page) + 1
        order = torch.randperm(pages, generator=g, device=DEVICE)
        at = torch.arange(T, device=DEVICE)
        # queries, keys and values as a fused projection leaves them, some channels of the keys larger
        qkv = normal(T, H + 2 * Hk, D)
        qkv[:, H:H + Hk] *= torch.where(torch.rand(D, generator=g, device=DEVICE) < 0.05, 8.0, 1.0)
        qkv = qkv.to(dtype)
        pair = torch.arange(pairs, device=DEVICE)
        # (time has the first quarter of the pairs, height and width the rest)
        axis = None if case["axes"] == 1 else torch.where(pair < pairs // 4, 0, 1 + (pair - pairs // 4) * 2 // max(1, pairs - pairs // 4)).to(torch.int32)
        positions = _positions(case)
        return dict(_pools(case, g, pages, torch.zeros(pages, page, dtype=torch.bool, device=DEVICE)), case=case,
                    q=qkv[:, :H], new_k=qkv[:, H:H + Hk], new_v=qkv[:, H + Hk:], positions=positions if case["axes"] > 1 else positions[0],
                    freq=10000.0 ** (-pair.double() / pairs), axis=axis, slots=order[at // page] * page + at % page)
    shapes = _shapes(case)
    pick = torch.randperm(len(shapes), generator=g, device=DEVICE).tolist()
    shapes = [shapes[i] for i in pick]
    state = dict(_cache(case, g, [n for _, n in shapes]), case=case, shapes=shapes)
    rows = case["batch"] if case["kind"] == "step" else sum(n for n, _ in shapes)
    # heads from flat to peaked
    state["q"] = (normal(rows, H, D) * torch.linspace(0.5, 3.0, H, device=DEVICE).unsqueeze(1)).to(dtype)
    if case["kind"] == "prompt":
        starts = [0]
        for n, _ in shapes:
            starts.append(starts[-1] + n)
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    if case["kind"] == "tree":
        B, N = case["batch"], case["drafts"]
        state["q"] = state["q"].view(B, N, H, D)
        # half of the drafts go on from the one before, the others from any earlier one or from the text
        at = torch.arange(N, device=DEVICE)
        back = (torch.rand(B, N, generator=g, device=DEVICE) * (at + 1)).long() - 1
        chain = torch.rand(B, N, generator=g, device=DEVICE) < 0.5
        state["parents"] = torch.where(chain, at - 1, back.minimum(at - 1)).to(torch.int32)
    return state


# ------------------------------------------------------------------------------- the operators
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-powershard_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from powershard_amd import ops
    return ops


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _append_own(s):
    ops = _ops()
    q = ops.rope_kv_write(s["q"], s["new_k"], s["new_v"], s["positions"], s["freq"], s["slots"], s["k"], s["v"], s["ks"], s["vs"],
                          axes=s["axis"], interleaved=s["case"]["interleaved"])
    # the codes as the values that they stand for
    k, v = ops.kv_read(s["slots"], s["k"], s["v"], s["ks"], s["vs"], out_dtype=q.dtype)
    return {"q": q, "k": k, "v": v}


def _step_own(s):
    case = s["case"]
    return _ops().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["ks"], s["vs"], window=case["window"],
                                  sinks=case["sinks"], max_len=case["max_len"])


def _prompt_own(s):
    case = s["case"]
    return _ops().paged_prompt_attention(s["q"], s["k"], s["v"], s["table"], s["starts"], s["lengths"], s["ks"], s["vs"],
                                         window=case["window"], sinks=case["sinks"], max_len=case["new"] + case["past"])


def _tree_own(s):
    case = s["case"]
    return _ops().paged_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["parents"], s["ks"], s["vs"],
                                       window=case["window"], sinks=case["sinks"], max_len=case["max_len"])


_run_own = {"append": _append_own, "step": _step_own, "prompt": _prompt_own, "tree": _tree_own}


# ------------------------------------------------------------------------------- plain forms
def _bits(pool):
    return pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)


def _turned(x, cos, sin, interleaved):
    """The first 2 * pairs dims of x [tokens, heads, dim] turned; cos, sin [tokens, 1, pairs]."""
    n = 2 * cos.shape[-1]
    head, rest = x[..., :n], x[..., n:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), rest], -1)


def _append_plain(s):
    case = s["case"]
    page = case["page"]
    at = s["positions"].reshape(-1, case["tokens"]).double()
    at = at[0].unsqueeze(1) if s["axis"] is None else at[s["axis"].long()].T
    angle = (at * s["freq"]).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    dtype = s["q"].dtype
    out = {"q": _turned(s["q"].float(), cos, sin, case["interleaved"]).to(dtype)}
    pg, pos = s["slots"] // page, s["slots"] % page
    rows = {"k": _turned(s["new_k"].float(), cos, sin, case["interleaved"]), "v": s["new_v"].float()}
    for name, x in rows.items():
        pool, scales = s[name], s[name + "s"]
        if scales is None:
            pool.transpose(1, 2)[pg, pos] = x.to(dtype)
            out[name] = pool.transpose(1, 2)[pg, pos]
            continue
        limit = CODES[case["codes"]][1]
        amax = x.abs().amax(-1, keepdim=True)
        scale = torch.where(amax == 0, 1.0, amax / limit)
        y = x / scale
        code = (y.round().clamp(-127, 127) if case["codes"] == "int8" else y.clamp(-448, 448)).to(pool.dtype)
        pool.transpose(1, 2).view(torch.int8)[pg, pos] = code.view(torch.int8)
        scales.transpose(1, 2)[pg, pos] = scale.squeeze(-1)
        codes = pool.transpose(1, 2).view(torch.int8)[pg, pos].view(pool.dtype).float()
        out[name] = (codes * scales.transpose(1, 2)[pg, pos].unsqueeze(-1)).to(dtype)
    return out


def _step_plain(s):
    case = s["case"]
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    table, lens = s["table"].long().clamp(min=0), s["lengths"].long().unsqueeze(1)
    L = table.shape[1] * case["page"]
    at = torch.arange(L, device=DEVICE)
    valid = (at < lens) & ((at >= lens - case["window"]) | (at < case["sinks"]))

    def dense(pool, scales):   # [B, Hk, L, D] in 32 bits, zero where no token is seen
        x = _bits(pool)[table].view(pool.dtype).transpose(1, 2).reshape(B, Hk, L, D).float()
        if scales is not None:
            x = x * scales[table].transpose(1, 2).reshape(B, Hk, L, 1)
        return x.masked_fill_(~valid.view(B, 1, L, 1), 0.0)

    scores = s["q"].float().view(B, Hk, H // Hk, D) @ dense(s["k"], s["ks"]).transpose(2, 3) / math.sqrt(D)
    scores = scores.masked_fill_(~valid.view(B, 1, 1, L), float("-inf"))
    return _weighted(scores, dense(s["v"], s["vs"])).view(B, H, D).to(s["q"].dtype)


def _weighted(scores, values):
    """softmax(scores) values; a row that sees nothing: zeros."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ values) / torch.where(total == 0, 1.0, total)


def _sequence_plain(s, b, q, seen):
    """Attention of q [rows, H, D] on sequence b's cache in 32 bits; seen(first row, rows): [rows, tokens] bool."""
    case, n = s["case"], s["shapes"][b][1]
    Hk, D = case["kv_heads"], case["dim"]
    pages = s["table"][b, :-(-n // case["page"])].long()

    def dense(pool, scales):   # [Hk, n, D]
        x = _bits(pool)[pages].view(pool.dtype).transpose(0, 1).reshape(Hk, -1, D)[:, :n].float()
        return x if scales is None else x * scales[pages].transpose(0, 1).reshape(Hk, -1, 1)[:, :n]

    k, v = dense(s["k"], s["ks"]).transpose(1, 2), dense(s["v"], s["vs"])
    group, out = q.shape[1] // Hk, torch.empty_like(q)
    rows = max(1, (1 << 27) // (q.shape[1] * n))
    for a in range(0, q.shape[0], rows):
        part = q[a:a + rows].float()
        m = part.shape[0]
        part = part.view(m, Hk, group, D).permute(1, 2, 0, 3).reshape(Hk, group * m, D)
        scores = (part @ k / math.sqrt(D)).view(Hk, group, m, n)
        scores = scores.masked_fill_(~seen(a, m), float("-inf")).view(Hk, group * m, n)
        out[a:a + rows] = _weighted(scores, v).view(Hk, group, m, D).permute(2, 0, 1, 3).reshape(m, -1, D).to(q.dtype)
    return out


def _near(case, position, at):
    """Whether tokens at `at` are in the window of `position` or among the sinks."""
    return (at > position - case["window"]) | (at < case["sinks"]) if case["window"] else torch.ones_like(at > position)


def _prompt_plain(s):
    case, out, first = s["case"], torch.empty_like(s["q"]), 0
    for b, (new, n) in enumerate(s["shapes"]):
        at = torch.arange(n, device=DEVICE)

        def seen(a, m):
            position = (n - new + a + torch.arange(m, device=DEVICE)).unsqueeze(1)
            return (at <= position) & _near(case, position, at)
        if new:
            out[first:first + new] = _sequence_plain(s, b, s["q"][first:first + new], seen)
        first += new
    return out


def _tree_plain(s):
    case, N = s["case"], s["case"]["drafts"]
    out, parents = torch.empty_like(s["q"]), s["parents"].long()
    # path[b, i, j]: draft j is i or before it on its way from the text
    path = torch.zeros(case["batch"], N, N, dtype=torch.bool, device=DEVICE)
    for i in range(N):
        p = parents[:, i]
        path[:, i] = torch.where((p >= 0).unsqueeze(1), path[torch.arange(case["batch"], device=DEVICE), p.clamp(min=0)], False)
        path[:, i, i] = True
    depth = path.sum(-1) - 1
    for b, (_, n) in enumerate(s["shapes"]):
        text = n - N
        at = torch.cat([torch.arange(text, device=DEVICE), text + depth[b]])   # the tokens' positions

        def seen(a, m):
            position = (text + depth[b, a:a + m]).unsqueeze(1)
            on_way = torch.cat([torch.ones(m, text, dtype=torch.bool, device=DEVICE), path[b, a:a + m]], 1)
            return on_way & _near(case, position, at)
        out[b] = _sequence_plain(s, b, s["q"][b], seen)
    return out


_run_plain = {"append": _append_plain, "step": _step_plain, "prompt": _prompt_plain, "tree": _tree_plain}


# ------------------------------------------------------------------------------- in 64 bits
def _nearest(x, codes):
    if codes == "int8":
        return torch.round(x).clamp(-127, 127)
    # e4m3: three fraction bits, exponents from -6 up, so steps of 2^(max(e, -6) - 3)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _append_exact(s):
    case, f = s["case"], torch.float64
    T, pairs = case["tokens"], case["rotary"] // 2
    position = _positions(case).to(f)
    turn = torch.empty(T, pairs, dtype=torch.complex128, device=DEVICE)
    for i in range(pairs):
        axis = 0 if s["axis"] is None else int(s["axis"][i])
        angle = position[axis] * s["freq"][i]
        turn[:, i] = torch.complex(angle.cos(), angle.sin())

    def rotated(x):
        x = x.to(f).clone()
        i = torch.arange(pairs, device=DEVICE)
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
        z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
        x[..., a], x[..., b] = z.real, z.imag
        return x

    out = {"q": rotated(s["q"])}
    for name, x in (("k", rotated(s["new_k"])), ("v", s["new_v"].to(f))):
        if case["codes"] != "none":
            amax = x.abs().max(-1, keepdim=True).values
            scale = torch.where(amax == 0, torch.ones_like(amax), amax / CODES[case["codes"]][1])
            x = _nearest(x / scale, case["codes"]) * scale
        out[name] = x
    return out


def _seen_exact(s, b, draft_parents, i):
    """The tokens that row i of sequence b attends to, as indices."""
    case, (new, n) = s["case"], s["shapes"][b]
    if case["kind"] == "tree":
        way = []
        while i >= 0:
            way.append(i)
            i = draft_parents[i]
        position, chosen = n - new + len(way) - 1, []
        for depth, j in enumerate(reversed(way)):
            p = n - new + depth
            if not case["window"] or p > position - case["window"] or p < case["sinks"]:
                chosen.append(n - new + j)
        limit = n - new
    else:
        position, chosen, limit = n - new + i, [], n - new + i + 1
    if not case["window"]:
        spans = [(0, limit)]
    else:
        low = max(0, position - case["window"] + 1)
        spans = [(0, min(case["sinks"], limit, low)), (low, limit)]
    return spans, chosen


def _attention_exact(s):
    case, f = s["case"], torch.float64
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q = s["q"].reshape(-1, H, D)
    out, first = torch.zeros(q.shape, dtype=f, device=DEVICE), 0
    for b, (new, n) in enumerate(s["shapes"]):
        if case["kind"] == "step":
            first = b
        if new == 0:
            continue
        pages = torch.tensor(s["table"][b, :-(-n // page)].tolist(), device=DEVICE)
        parents = s["parents"][b].tolist() if case["kind"] == "tree" else None
        seen = torch.zeros(new, n, dtype=torch.bool)
        for i in range(new):
            spans, chosen = _seen_exact(s, b, parents, i)
            for lo, hi in spans:
                seen[i, lo:hi] = True
            seen[i, chosen] = True
        hidden = ~seen.to(DEVICE)
        for h in range(Hk):
            def tokens(pool, scales):
                x = _bits(pool[:, h].contiguous())[pages].view(pool.dtype).float().to(f).reshape(-1, D)[:n]
                return x if scales is None else x * scales[:, h][pages].to(f).reshape(-1)[:n, None]
            k, v = tokens(s["k"], s["ks"]), tokens(s["v"], s["vs"])
            for j in range(h * (H // Hk), (h + 1) * (H // Hk)):
                for a in range(0, new, 4096):
                    rows = slice(first + a, first + min(new, a + 4096))
                    scores = q[rows, j].to(f) @ k.T / math.sqrt(D)
                    scores[hidden[a:a + 4096]] = -math.inf
                    out[rows, j] = torch.softmax(scores, -1) @ v
        first += new
    return out.view(s["q"].shape)


def exact(case, seed):
    s = prepare(case, seed)
    return _append_exact(s) if case["kind"] == "append" else _attention_exact(s)


# ------------------------------------------------------------------------------- work
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    element = 2 if case["codes"] == "none" else 1
    per = Hk * (2 * D * element + (0 if case["codes"] == "none" else 8))   # a cached token
    if case["kind"] == "append":
        T = case["tokens"]
        # queries in and out, keys and values in, their codes written and read again for the values that come back
        return {"bytes": T * (4 * H * D + 4 * Hk * D + 2 * per + 4 * Hk * D + 8 * case["axes"] + 16) + 12 * case["rotary"],
                "flops": T * (3 * (H + Hk) * case["rotary"] + (6 * Hk * D if element == 1 else 0))}
    window, sinks = case["window"], case["sinks"]
    rows = cached = products = 0

    def span(position):   # tokens up to and with this position that are seen
        n = position + 1
        return n if not window or n <= window else window + min(sinks, n - window)
    for new, n in _shapes(case):
        rows += new
        if new == 0:
            continue
        first = n - new
        if case["kind"] == "tree":   # (each draft with the text and itself, whatever the tree is)
            products += new * span(first)
            cached += min(span(first) + new - 1, n)
        else:
            products += sum(span(p) for p in range(first, n))
            low = max(0, first - window + 1) if window else 0
            cached += n - low + min(sinks, low)
    rows = case["batch"] if case["kind"] == "step" else rows
    tables = 4 * sum(-(-n // case["page"]) for _, n in _shapes(case)) + 4 * case["batch"]
    extra = {"step": 0, "prompt": 4 * (case["batch"] + 1), "tree": 4 * rows}[case["kind"]]
    return {"bytes": cached * per + 4 * rows * H * D + tables + extra, "flops": 4 * products * H * D}
