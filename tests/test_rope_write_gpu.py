"""Keys appended to the paged cache turned to their positions, and the turned queries, against 64 bits.

Errors of the kernel in front of the last rounding, as fractions of |a| + |b| (a pair's elements): the
angle's remainder is rounded to fp32 once in turns (2^-25 turns: 2^-22.3), the two series and their
products add a few fp32 roundings (2^-24 each): below 2^-21 together, and the reference's own angle
(a product in 64 bits) 2^-52 of the position.  A 16-bit result adds half a step.  A row's maximum is off by
less than sqrt(2) 2 2^-21 of itself, so codes are the nearest ones to a quotient off by 2^-18 of the largest code."""
import pytest
import torch

from conftest import seeded
from test_kv_cache_gpu import CODES, by_slot, make_pools, same

pytestmark = pytest.mark.gpu


def turned(x, positions, freq, axes=None, interleaved=False):
    """(x turned in 64 bits, what |a| + |b| of each element's pair is)."""
    x, pairs = x.double().cpu(), freq.shape[0]
    at = positions.double().cpu()
    at = at[:, None].expand(-1, pairs) if axes is None else at[axes.long().cpu()].T
    angle = (at * freq.double().cpu())[:, None]
    i = torch.arange(pairs)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    y[..., b] = x[..., b] * angle.cos() + x[..., a] * angle.sin()
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def check(got, y, size, dtype, far):
    """got, 16 bits, against y; far: the largest position."""
    bound = y.abs() * torch.finfo(dtype).eps / 2 + size * (2.0 ** -21 + far * 2.0 ** -52) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got.double().cpu() - y).abs() <= bound).all()


def check_codes(codes, pool, scales, slots, y, far):
    loose = 2.0 ** -18 + far * 2.0 ** -51
    lim = CODES[codes][1]
    amax = y.abs().amax(-1)
    s = by_slot(scales)[slots].double().cpu()
    assert ((s - amax / lim).abs() <= amax / lim * loose).all()
    u = y / (amax / lim)[..., None]
    q = by_slot(pool.view(torch.int8))[slots].view(pool.dtype).double().cpu()
    step = torch.full_like(u, 0.5) if codes == "int8" else torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 4)
    assert ((q - u).abs() <= step * (1 + 2.0 ** -10) + lim * loose).all()   # (e4m3: half a step may be that of the binade above)


def freqs(pairs, gpu):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=gpu) / pairs)


@pytest.mark.parametrize("codes", ["none", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,H,D,page,rotary,axes,interleaved", [
    (1, 40, 8, 128, 16, 128, 1, False), (1, 1, 1, 16, 16, 16, 1, True), (7, 6, 3, 48, 16, 32, 1, False), (61, 10, 5, 80, 48, 80, 3, True),
    (130, 4, 4, 256, 64, 256, 2, False), (33, 7, 1, 240, 16, 16, 1, True), (300, 8, 2, 64, 32, 48, 3, False), (4200, 3, 1, 32, 112, 32, 1, True)])
def test_against_64_bits(gpu, codes, dtype, T, Hq, H, D, page, rotary, axes, interleaved):
    from powershard_amd import ops
    g = seeded(T + D)
    pages = -(-T // page) + 2
    k, v, ks, vs = make_pools(pages, H, page, D, codes, dtype, gpu, fill=0x7F)
    k2, v2, ks2, vs2 = make_pools(pages, H, page, D, codes, dtype, gpu, fill=0x7F)
    qkv = (torch.randn(T, Hq + 2 * H, D, generator=g) * torch.exp2(torch.randint(-4, 5, (T, Hq + 2 * H, 1), generator=g).float())).to(dtype).to(gpu)
    q, nk, nv = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    slots = torch.randperm(pages * page, generator=g)[:T].to(gpu)
    pairs, far = rotary // 2, 131071
    positions = torch.randint(-far, far, (axes, T), generator=g).to(torch.int32 if axes == 2 else torch.int64).to(gpu)
    axis = None if axes == 1 else torch.randint(0, axes, (pairs,), generator=g).to(torch.int32).to(gpu)
    if axes == 1:
        positions = positions[0]
    freq = freqs(pairs, gpu)
    before = qkv.clone()
    out = ops.rope_kv_write(q, nk, nv, positions, freq, slots, k, v, ks, vs, axes=axis, interleaved=interleaved)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous() and same(qkv, before)
    check(out, *turned(q, positions, freq, axis, interleaved), dtype, far)
    ops.kv_write(nk, nv, slots, k2, v2, ks2, vs2)      # values are written as without positions
    assert same(v, v2) and (vs is None or same(vs, vs2))
    y, size = turned(nk, positions, freq, axis, interleaved)
    if codes == "none":
        check(by_slot(k)[slots], y, size, dtype, far)
    else:
        check_codes(codes, k, ks, slots, y, far)
    others = torch.ones(pages * page, dtype=torch.bool, device=gpu)
    others[slots] = False
    raw, raw2 = (by_slot(t.view(torch.uint8)) for t in (k, k2))
    assert torch.equal(raw[others], raw2[others]) and (ks is None or by_slot(ks)[others].isnan().all())
    # position 0 turns nothing
    out = ops.rope_kv_write(q, nk, nv, torch.zeros_like(positions), freq, slots, k, v, ks, vs, axes=axis, interleaved=interleaved)
    assert torch.equal(out, q) and same(k, k2) and (ks is None or same(ks, ks2))


@pytest.mark.parametrize("at", [2 ** 31 - 1, -2 ** 31, 1000003])
def test_far_positions(gpu, at):
    from powershard_amd import ops
    k, v, _, _ = make_pools(1, 1, 16, 128, "none", torch.float16, gpu)
    x = torch.randn(1, 3, 128, generator=seeded(3)).half().to(gpu)
    freq = freqs(64, gpu)
    for kind in (torch.int32, torch.int64):
        pos = torch.tensor([at], dtype=kind, device=gpu)
        out = ops.rope_kv_write(x, x[:, :1], x[:, 1:2], pos, freq, torch.zeros(1, dtype=torch.int64, device=gpu), k, v)
        check(out, *turned(x, pos, freq), torch.float16, abs(at))


@pytest.mark.parametrize("codes", ["none", "int8", "fp8"])
def test_layouts_and_edges(gpu, codes):
    """Strided and misaligned inputs, fp32 frequencies, strided axes and positions, skipped slots, zero, NaN and
    infinite rows, no tokens, no queries."""
    from powershard_amd import ops
    g = seeded(9)
    T, Hq, H, D, page, dtype = 6, 4, 2, 64, 16, torch.bfloat16
    x = torch.randn(T, Hq + 2 * H, D, generator=g)
    x[1, Hq] = 0
    x[2, Hq + 1, 5] = float("nan")
    x[3, Hq + 1, 40] = float("inf")
    x = x.to(dtype).to(gpu)
    q, nk, nv = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    freq, slots = freqs(32, gpu), torch.tensor([3, 17, 30, -1, 2, 1 << 40], device=gpu)
    pos = torch.arange(2 * T, device=gpu).view(2, T)
    axis = (torch.arange(32, device=gpu) % 2).to(torch.int32)
    want = make_pools(2, H, page, D, codes, dtype, gpu, fill=0)
    out = ops.rope_kv_write(q, nk, nv, pos, freq, slots, *want, axes=axis)
    check(out, *turned(q, pos, freq, axis), dtype, 100)
    if codes == "none":
        check(by_slot(want[0])[slots[:2]], *[t[:2] for t in turned(nk, pos, freq, axis)], dtype, 100)
    else:
        s = by_slot(want[2])
        assert s[17, 0] == 1 and (by_slot(want[0].float())[17, 0] == 0).all() and s[30, 1].isnan() and not s[30, 0].isnan()
    def other(t):     # elements two apart
        return torch.stack([t, t], -1).flatten(-2)[..., ::2]
    odd = torch.cat([torch.zeros(1, dtype=dtype, device=gpu), nv.reshape(-1)])[1:].view(nv.shape)   # 2 bytes off
    got = make_pools(2, H, page, D, codes, dtype, gpu, fill=0)
    out2 = ops.rope_kv_write(q.transpose(0, 1).contiguous().transpose(0, 1), other(nk), odd, torch.stack([pos, pos], -1).flatten(1)[:, ::2],
                             other(freq), other(slots), *got, axes=other(axis))
    assert same(out, out2) and all(a is None or same(a, b) for a, b in zip(want, got))
    one = ops.rope_kv_write(q, nk, nv, pos[0], freq.float(), slots, *got)
    check(one, *turned(q, pos[0], freq.float()), dtype, 100)
    wild = torch.full_like(axis, 7)     # (outside the axes: the last one)
    out3 = ops.rope_kv_write(q, nk, nv, pos, freq, slots, *got, axes=wild)
    assert same(out3, ops.rope_kv_write(q, nk, nv, pos[1], freq, slots, *got))
    assert ops.rope_kv_write(q[:0], nk[:0], nv[:0], pos[0, :0], freq, slots[:0], *got).shape == (0, Hq, D)
    before = [None if t is None else t.clone() for t in got]
    assert ops.rope_kv_write(q[:, :0], nk, nv, pos[1], freq, slots, *got).shape == (T, 0, D)   # writes what the last call with all of it wrote
    assert all(a is None or same(a, b) for a, b in zip(before, got))


def test_refusals(gpu):
    from powershard_amd import ops
    k, v, ks, vs = make_pools(2, 2, 16, 64, "int8", torch.bfloat16, gpu)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    pos, slots, freq = torch.arange(3, device=gpu), torch.arange(3, device=gpu), freqs(32, gpu)
    axis = torch.zeros(32, dtype=torch.int32, device=gpu)

    def call(q=x, nk=x, nv=x, positions=pos, freq=freq, slots=slots, k=k, v=v, ks=ks, vs=vs, **options):
        return ops.rope_kv_write(q, nk, nv, positions, freq, slots, k, v, ks, vs, **options)
    call()
    for bad in (dict(q=x.float()), dict(nk=x.half()), dict(nv=x.half()), dict(k=k.float(), v=v.float())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(q=x[:2]), dict(q=x[..., :32]), dict(q=x[0]), dict(nk=x[:, :1]), dict(nv=x[:2]), dict(freq=freq[:12]), dict(freq=freq[:0]),
                dict(freq=freqs(40, gpu)), dict(freq=freq.view(4, 8)), dict(positions=pos.float()), dict(positions=pos[:2]), dict(positions=pos[None]),
                dict(axes=axis), dict(positions=pos[None], axes=axis[:8]), dict(positions=pos[None], axes=axis.long()), dict(positions=pos[None][:0], axes=axis),
                dict(slots=slots.int()), dict(slots=slots[:2]), dict(ks=None), dict(ks=ks.half())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(q=x.cpu()), dict(nv=x.cpu()), dict(positions=pos.cpu()), dict(freq=freq.cpu()), dict(slots=slots.cpu()), dict(k=k.cpu()),
                dict(positions=pos[None], axes=axis.cpu())):
        with pytest.raises(RuntimeError):
            call(**bad)


def test_streams_and_graph(gpu):
    """On a stream of its own and captured: positions, slots and rows are read at every replay."""
    from powershard_amd import ops
    T, Hq, H, D = 5, 8, 2, 128
    pools = [make_pools(4, H, 16, D, "fp8", torch.bfloat16, gpu, fill=0) for _ in range(2)]
    freq = freqs(64, gpu)
    x = torch.zeros(T, Hq + 2 * H, D, dtype=torch.bfloat16, device=gpu)
    pos, slots = torch.zeros(T, dtype=torch.int32, device=gpu), torch.full((T,), -1, dtype=torch.int64, device=gpu)

    def step(p):
        return ops.rope_kv_write(x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:], pos, freq, slots, *p)
    stream = torch.cuda.Stream(gpu)
    stream.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(stream):
        step(pools[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(pools[0])
    for i in range(5):
        x.copy_(torch.randn(x.shape, generator=seeded(i)))
        pos.copy_(torch.randint(0, 5000, (T,), generator=seeded(i)))
        slots.copy_(torch.randperm(64, generator=seeded(i))[:T])
        want = step(pools[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want) and all(same(a, b) for a, b in zip(*pools))
