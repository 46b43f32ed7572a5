"""The measured operators of a text decoder's layer around the quantized linears: the norm that makes
their 8-bit rows, the paged key-value cache that is quantized as it is written, its read-back, and the
attention of one new token over it.

A case is one call that a decoder makes per layer (cache cases: the write of the new tokens and the
read of the tokens that the prompt's attention needs).  ``run`` computes it either with the package's
operators (``own``) or in plain torch operations in 32 bits.

Layouts: caches [pages, kv heads, page size, head dim], their scales [pages, kv heads, page size],
one page table row per sequence, slot = page * page size + offset.  Everything past a sequence's
length, and every page that no sequence holds, is NaN (garbage, for int8 codes), as memory that
nobody has written may be.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
DEVICE = "cuda:0"
EPS = 1e-6


def _norm(name, M, K, dtype, codes, rot=0):
    return dict(name=name, kind="norm", M=M, K=K, dtype=dtype, codes=codes, rot=rot)


def _cache(name, new, total, kv_heads, dim, page, dtype, codes):
    return dict(name=name, kind="cache", new=new, total=total, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, codes=codes)


def _attend(name, batch, max_len, heads, kv_heads, dim, page, dtype, codes="none", window=0):
    return dict(name=name, kind="attend", batch=batch, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, window=window)


def listed():
    return [
        # the next token of one user, into an int8 ConvRot projection: latency
        _norm("norm_i8_token_m1", 1, 5120, "bf16", "int8", rot=256),
        # the next tokens of a batch of users, into an fp8 projection
        _norm("norm_fp8_batch_m61", 61, 5376, "f16", "fp8"),
        # the tokens of long prompts, into an int8 ConvRot projection
        _norm("norm_i8_prompt_m8191", 8191, 5120, "bf16", "int8", rot=256),
        # one new token of each of 64 users
        _cache("cache_i8_tokens_t64", 64, 64, 8, 128, 16, "bf16", "int8"),
        # a whole prompt that ends inside a page
        _cache("cache_fp8_prompt_t4095", 4095, 4095, 8, 128, 64, "bf16", "fp8"),
        # the last chunk of a very long prompt, whose attention reads all of it
        _cache("cache_i8_chunk_t65489", 512, 65489, 8, 128, 64, "f16", "int8"),
        # one user right after a short prompt, as many kv heads as heads: latency
        _attend("attend_bf16_short", 1, 77, 40, 40, 128, 16, "bf16"),
        # a batch of users of ragged lengths on an int8 cache, shared kv heads
        _attend("attend_i8_batch", 61, 4096, 40, 8, 128, 16, "bf16", "int8"),
        # one user deep in a very long text: split over the length
        _attend("attend_fp8_long", 1, 131071, 40, 8, 128, 64, "bf16", "fp8"),
        # a layer that attends to the last 1024 tokens only, narrow heads
        _attend("attend_f16_window", 16, 8192, 64, 16, 64, 32, "f16", window=1024),
        # one kv head shared by all heads, wide heads, pages that are no power of two
        _attend("attend_i8_shared_d256", 8, 6000, 16, 1, 256, 48, "f16", "int8"),
        # the largest batch: the cache fills gigabytes
        _attend("attend_bf16_large", 128, 8192, 64, 8, 128, 64, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 8192 rows of 512 to 14336 columns; 1 to 65536 cached tokens; batches of 1 to
    128 with lengths up to 131072; head dims of 16 to 256, 1 to 64 heads, shared or not; every type."""
    kind = rng.choice(["norm", "cache", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "norm":
        K = 256 * _log(rng, 2, 56)
        codes = rng.choice(["int8", "int8", "fp8"])
        M = _log(rng, 1, max(1, 8192 * 5120 // max(K, 5120)))
        return dict(kind=kind, M=M, K=K, dtype=dtype, codes=codes, rot=rng.choice([0, 256]) if codes == "int8" else 0)
    dim = rng.choice([64, 128, 128, 128, 256, 16 * rng.randint(1, 16)])
    page = rng.choice([16, 32, 64, 128, 16 * rng.randint(1, 16)])
    codes = rng.choice(["int8", "fp8"] if kind == "cache" else ["int8", "fp8", "none"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, rng.randint(1, 40)])
    if kind == "cache":
        total = _log(rng, 1, 65536)
        while total * kv_heads * dim > 65489 * 8 * 128:
            total = max(1, total // 2)
        new = total if rng.random() < 0.5 else _log(rng, 1, total)
        return dict(kind=kind, new=new, total=total, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, codes=codes)
    group = rng.choice([1, 2, 4, 5, 7, 8, 16, rng.randint(1, 64)])
    group = max(1, min(group, 64 // kv_heads))
    batch, max_len = _log(rng, 1, 128), _log(rng, 1, 131072)
    # no more cache, and no more products, than the largest listed case
    while batch * max_len * kv_heads * dim * max(1, group / 8) > 128 * 8192 * 8 * 128:
        batch, max_len = (max(1, batch // 2), max_len) if batch > 1 else (batch, max_len // 2)
    window = _log(rng, 1, max_len) if rng.random() < 0.2 else 0
    return dict(kind=kind, batch=batch, max_len=max_len, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, codes=codes, window=window)


# ------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Ragged lengths that the case alone sets: spread evenly over 0 .. max_len, the longest among them."""
    B, longest = case["batch"], case["max_len"]
    return [longest if b == 0 else int(longest * ((b * 0.6180339887498949) % 1.0)) for b in range(B)]


def _unwritten(k, codes, valid):
    """k with every row that valid leaves out set to what unwritten memory may hold."""
    if k.dtype == torch.int8:
        return k
    bits = k.view(torch.uint8 if k.element_size() == 1 else torch.int16)
    bits.masked_fill_(~valid.unsqueeze(-1), 0x7F if codes == "fp8" else 0x7FFF)
    return k


def _pools(case, g, pages, valid):
    """K and V pools with their scales; valid [pages, page size]: the slots that hold tokens."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    valid = valid.unsqueeze(1).expand(shape[:3])
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32 if case["codes"] != "none" else DTYPES[case["dtype"]])
        if case["codes"] == "none":
            pools.append(_unwritten(x, "none", valid))
            scales.append(None)
            continue
        code, limit = CODES[case["codes"]]
        x = x.mul_(limit / 3.5).clamp_(-limit, limit)
        pools.append(_unwritten(x.round_().to(code) if code == torch.int8 else x.to(code), case["codes"], valid))
        s = (0.5 + 1.5 * torch.rand(shape[:3], generator=g, device=DEVICE)) * (3.5 / limit)
        scales.append(s.masked_fill_(~valid, float("nan")))
    return pools[0], pools[1], scales[0], scales[1]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed % (1 << 60))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["kind"] == "norm":
        M, K = case["M"], case["K"]
        # activations and residual stream: normal, a hundredth of the channels twenty times larger
        outlier = torch.where(torch.rand(K, generator=g, device=DEVICE) < 0.01, 20.0, 1.0)
        return dict(case=case, x=(normal(M, K) * outlier).to(dtype), residual=(2.0 * normal(M, K) * outlier).to(dtype),
                    weight=(1.0 + 0.1 * normal(K)).to(dtype))
    page = case["page"]
    if case["kind"] == "cache":
        total, new = case["total"], case["new"]
        pages = -(-total // page) + 1
        order = torch.randperm(pages, generator=g, device=DEVICE)
        at = torch.arange(total, device=DEVICE)
        slots = order[at // page] * page + at % page
        valid = torch.zeros(pages * page, dtype=torch.bool, device=DEVICE)
        valid[slots[:total - new]] = True
        k, v, ks, vs = _pools(case, g, pages, valid.view(pages, page))
        # the keys and values as a fused projection leaves them: rows of k heads, then v heads
        kv = normal(new, 2, case["kv_heads"], case["dim"])
        kv[:, 0] *= torch.where(torch.rand(case["dim"], generator=g, device=DEVICE) < 0.05, 8.0, 1.0)
        kv = kv.to(dtype)
        return dict(case=case, new_k=kv[:, 0], new_v=kv[:, 1], new_slots=slots[total - new:].clone(), slots=slots, k=k, v=v, ks=ks, vs=vs)
    lens = torch.tensor(_lengths(case), device=DEVICE)
    B = case["batch"]
    lens = lens[torch.randperm(B, generator=g, device=DEVICE)]
    per = -(-case["max_len"] // page)
    held = (lens + page - 1) // page
    pages = sum(-(-n // page) for n in _lengths(case)) + 1
    order = torch.randperm(pages, generator=g, device=DEVICE)
    col = torch.arange(per, device=DEVICE)
    first = torch.cumsum(held, 0) - held
    used = col < held.unsqueeze(1)
    # the columns past a sequence's pages hold nothing that may be followed
    table = torch.where(used, order[(first.unsqueeze(1) + col).clamp(max=pages - 1)], -1)
    valid = torch.zeros(pages, page, dtype=torch.bool, device=DEVICE)
    fill = (lens.unsqueeze(1) - col * page).clamp(0, page)
    valid[table[used]] = torch.arange(page, device=DEVICE) < fill[used].unsqueeze(1)
    k, v, ks, vs = _pools(case, g, pages, valid)
    # heads from flat to peaked
    q = normal(B, case["heads"], case["dim"]) * torch.linspace(0.5, 3.0, case["heads"], device=DEVICE).unsqueeze(1)
    return dict(case=case, q=q.to(dtype), k=k, v=v, ks=ks, vs=vs, table=table.to(torch.int32), lengths=lens.to(torch.int32))


# ------------------------------------------------------------------------------- the operators
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-powershard_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from powershard_amd import ops
    return ops


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _norm_own(s):
    ops, case = _ops(), s["case"]
    q, scale, total = ops.add_rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], codes=case["codes"], rot_group=case["rot"])
    # int8 codes as the values they stand for; e4m3 codes are a floating tensor already
    values = q if case["codes"] == "fp8" else ops.dequant_i8_rows(q, scale)
    return {"sum": total, "values": values, "scale": scale}


def _cache_own(s):
    ops = _ops()
    ops.kv_write(s["new_k"], s["new_v"], s["new_slots"], s["k"], s["v"], s["ks"], s["vs"])
    k, v = ops.kv_read(s["slots"], s["k"], s["v"], s["ks"], s["vs"], out_dtype=s["new_k"].dtype)
    return {"k": k, "v": v}


def _attend_own(s):
    case = s["case"]
    return _ops().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["ks"], s["vs"], window=case["window"],
                                  max_len=case["max_len"])


_run_own = {"norm": _norm_own, "cache": _cache_own, "attend": _attend_own}


# ------------------------------------------------------------------------------- plain forms
def _rounded(x, codes):
    """x rounded to whole numbers in -127 .. 127, or to e4m3."""
    if codes == "int8":
        return x.round().clamp(-127, 127)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _hadamard(size, dtype):
    """The regular Hadamard matrix of a power of four, normalized."""
    h4 = torch.ones(4, 4, dtype=dtype, device=DEVICE) - 2 * torch.eye(4, dtype=dtype, device=DEVICE).flip(0)
    h = h4 / 2
    return h if size == 4 else torch.kron(h, _hadamard(size // 4, dtype))


def _norm_plain(s):
    case = s["case"]
    limit = CODES[case["codes"]][1]
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    h = total.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if case["rot"]:
        y = (y.view(-1, case["rot"]) @ _hadamard(case["rot"], torch.float32)).view(y.shape)
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.where(amax == 0, 1.0, amax / limit)
    values = _rounded(y / scale, case["codes"])
    if case["codes"] == "int8":
        values = (values * scale).to(torch.bfloat16)
    return {"sum": total, "values": values, "scale": scale.squeeze(-1)}


def _flat(pool):
    """[pages, heads, page, ...] as [slots, heads, ...]."""
    return pool.transpose(1, 2)


def _cache_plain(s):
    case = s["case"]
    limit, page = CODES[case["codes"]][1], case["page"]
    at, pos = s["new_slots"] // page, s["new_slots"] % page
    seen = []
    for new, pool, scales in ((s["new_k"], s["k"], s["ks"]), (s["new_v"], s["v"], s["vs"])):
        x = new.float()
        amax = x.abs().amax(-1, keepdim=True)
        scale = torch.where(amax == 0, 1.0, amax / limit)
        code = _rounded(x / scale, case["codes"]).to(pool.dtype)
        _flat(pool).view(torch.int8)[at, pos] = code.view(torch.int8)
        _flat(scales)[at, pos] = scale.squeeze(-1)
        a, b = s["slots"] // page, s["slots"] % page
        codes = _flat(pool).view(torch.int8)[a, b].view(pool.dtype).float()
        seen.append((codes * _flat(scales)[a, b].unsqueeze(-1)).to(new.dtype))
    return {"k": seen[0], "v": seen[1]}


def _attend_plain(s):
    case = s["case"]
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    q, table, lens = s["q"], s["table"].long().clamp(min=0), s["lengths"].long()
    L = table.shape[1] * case["page"]
    at = torch.arange(L, device=q.device)
    valid = at < lens.unsqueeze(1)
    if case["window"]:
        valid &= at >= (lens - case["window"]).unsqueeze(1)

    def dense(pool, scales):   # [B, Hk, L, D] in 32 bits, zero where no token is
        x = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)[table].view(pool.dtype).transpose(1, 2).reshape(B, Hk, L, D).float()
        if scales is not None:
            x = x * scales[table].transpose(1, 2).reshape(B, Hk, L, 1)
        return x.masked_fill_(~valid.view(B, 1, L, 1), 0.0)

    scores = q.float().view(B, Hk, H // Hk, D) @ dense(s["k"], s["ks"]).transpose(2, 3) / math.sqrt(D)
    scores = scores.masked_fill_(~valid.view(B, 1, 1, L), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    weight = p.sum(-1, keepdim=True)
    out = (p @ dense(s["v"], s["vs"])) / torch.where(weight == 0, 1.0, weight)   # a sequence of no tokens: zeros
    return out.view(B, H, D).to(q.dtype)


_run_plain = {"norm": _norm_plain, "cache": _cache_plain, "attend": _attend_plain}


# ------------------------------------------------------------------------------- in 64 bits
def _nearest(x, codes):
    if codes == "int8":
        return torch.round(x).clamp(-127, 127)
    # e4m3: three fraction bits, exponents from -6 up, so steps of 2^(max(e, -6) - 3)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["kind"] == "norm":
        limit = CODES[case["codes"]][1]
        total = s["x"].to(f) + s["residual"].to(f)
        h = total.to(s["x"].dtype).to(f)
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["K"] + EPS) * s["weight"].to(f)
        if case["rot"]:
            y = torch.matmul(y.unflatten(-1, (-1, case["rot"])), _hadamard(case["rot"], f)).flatten(-2)
        scale = y.abs().max(-1, keepdim=True).values / limit
        scale[scale == 0] = 1.0
        values = _nearest(y / scale, case["codes"])
        return {"sum": total, "values": values * scale if case["codes"] == "int8" else values, "scale": scale[:, 0]}
    if case["kind"] == "cache":
        limit, total, new, page = CODES[case["codes"]][1], case["total"], case["new"], case["page"]
        out = {}
        for name, x, pool, scales in (("k", s["new_k"], s["k"], s["ks"]), ("v", s["new_v"], s["v"], s["vs"])):
            seen = torch.empty(total, case["kv_heads"], case["dim"], dtype=f, device=DEVICE)
            old = s["slots"][:total - new]
            for h in range(case["kv_heads"]):
                codes = pool[:, h].float().to(f).reshape(-1, case["dim"])
                seen[:total - new, h] = codes[old] * scales[:, h].to(f).reshape(-1)[old, None]
            amax = x.to(f).abs().max(-1, keepdim=True).values
            scale = torch.where(amax == 0, torch.ones_like(amax), amax / limit)
            seen[total - new:] = _nearest(x.to(f) / scale, case["codes"]) * scale
            out[name] = seen
        return out
    B, H, Hk, D, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(B, H, D, dtype=f, device=DEVICE)
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = s["table"][b, :-(-n // page)].tolist()
        pick = torch.tensor(pages, device=DEVICE)
        for h in range(Hk):
            def tokens(pool, scales):
                x = pool[:, h].view(torch.uint8 if pool.element_size() == 1 else torch.int16)[pick].view(pool.dtype).float().to(f).reshape(-1, D)[first:n]
                return x if scales is None else x * scales[:, h][pick].to(f).reshape(-1)[first:n, None]
            queries = s["q"][b, h * (H // Hk):(h + 1) * (H // Hk)].to(f)
            p = torch.softmax(queries @ tokens(s["k"], s["ks"]).T / math.sqrt(D), -1)
            out[b, h * (H // Hk):(h + 1) * (H // Hk)] = p @ tokens(s["v"], s["vs"])
    return out


# ------------------------------------------------------------------------------- work
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["kind"] == "norm":
        n = case["M"] * case["K"]
        # x, the residual and the sum in 16 bits; the codes, which are what the path makes, 8 bits; int8
        # codes are read again for the values that come back, 16 bits
        per = 2 + 2 + 2 + 1 + (3 if case["codes"] == "int8" else 0)
        return {"bytes": n * per + 2 * case["K"] + 4 * case["M"], "flops": 8 * n}
    row = case["kv_heads"] * case["dim"]
    if case["kind"] == "cache":
        # new keys and values read and written as codes with scales; all tokens read and given back
        write = case["new"] * (2 * row * 3 + 8 * case["kv_heads"] + 8)
        read = case["total"] * (2 * row * 3 + 8 * case["kv_heads"] + 8)
        return {"bytes": write + read, "flops": 6 * case["new"] * row + 2 * case["total"] * row}
    lens = [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]
    tokens = sum(lens)
    per = 2 * row * (2 if case["codes"] == "none" else 1) + (0 if case["codes"] == "none" else 8 * case["kv_heads"])
    ends = 2 * 2 * case["batch"] * case["heads"] * case["dim"]   # queries in, outputs out
    return {"bytes": tokens * per + ends + 4 * case["batch"] + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 4 * tokens * case["heads"] * case["dim"]}
