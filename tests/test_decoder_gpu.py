"""The decoder layer: quantized rows handed from the norm to the linears, and a text decoded through the
paged cache, prompt and single tokens, against the same text as one prompt and against 64 bits."""
import pytest
import torch
from torch import nn

from conftest import heavy_rows, seeded
from test_quant_linear_gpu import make_layer

pytestmark = pytest.mark.gpu

ROT = {"convrot": True, "convrot_groupsize": 256}
Q8 = [("int8", ROT), ("int8", {"convrot": False}), ("fp8", {})]


@pytest.mark.parametrize("fmt,opts", Q8)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 5, 300])
@pytest.mark.parametrize("activation,N", [(None, 320), ("gelu_tanh", 96), ("silu_gate", 256), ("silu_gate", 96)])
def test_forward_codes_has_the_forwards_values(gpu, fmt, opts, dtype, M, activation, N):
    from powershard_amd import ops
    from powershard_amd.quant_linear import QuantizedRows
    layer, _, _ = make_layer(512, N, fmt, opts, dtype, True, gpu, seed=5, bias=activation is None)
    x = heavy_rows(M, 512, 6, dtype=dtype).to(gpu).reshape(1, M, 512)
    kind, group = layer.input_codes()
    assert (kind, group) == (fmt, 256 if opts.get("convrot") else 0)
    q, scale = ops.quantize_rows(x[0], fp8=fmt == "fp8", rot_group=group)
    rows = QuantizedRows(q, scale, group, tuple(x.shape), dtype)
    want = (layer(x) if activation is None else layer.forward_act(x, activation)).to(dtype)
    got = layer.forward_codes(rows, activation)
    assert got.dtype == dtype and torch.equal(got.view(torch.int16), want.view(torch.int16))
    slow = layer.forward_codes(rows._replace(dtype=torch.float32), activation)     # the general path
    assert torch.equal(slow.view(torch.int16), want.view(torch.int16))


def test_input_codes_and_refusals(gpu):
    from powershard_amd.norm import rows_for
    from powershard_amd.quant_linear import QuantizedRows
    def layer(fmt, opts, native=True, K=512):
        return make_layer(K, 64, fmt, opts, torch.bfloat16, native, gpu, seed=7)[0]
    int8, rot, fp8, int4 = layer("int8", {"convrot": False}), layer("int8", ROT), layer("fp8", {}), layer("int4", {"group_size": 128})
    assert int4.input_codes() is None and layer("fp8", {}, native=False).input_codes() is None
    assert layer("int8", {"convrot": False}, K=448).input_codes() is None
    assert rows_for([rot, rot]) == ("int8", 256) and rows_for([int8, rot]) is None and rows_for([rot, int4]) is None
    assert rows_for([nn.Linear(4, 4)]) is None
    full = layer("fp8", {})
    full._ps_full_precision = True
    assert full.input_codes() is None
    codes = torch.zeros(3, 512, dtype=torch.int8, device=gpu)
    rows = QuantizedRows(codes, torch.ones(3, device=gpu), 0, (3, 512), torch.bfloat16)
    assert int8.forward_codes(rows).shape == (3, 64)
    for module in (rot, fp8, int4, full):
        with pytest.raises(ValueError):
            module.forward_codes(rows)
    with pytest.raises(ValueError):
        int8.forward_codes(rows._replace(codes=codes[:, :384].contiguous()))


@pytest.mark.parametrize("fmt,opts", Q8 + [("int4", {"group_size": 128})])
def test_norm_hands_rows_to_the_linears(gpu, fmt, opts):
    from powershard_amd import ops
    from powershard_amd.norm import RMSNorm, linear
    from powershard_amd.quant_linear import QuantizedRows
    layers = [make_layer(512, n, fmt, opts, torch.bfloat16, True, gpu, seed=8 + n)[0] for n in (64, 128)]
    norm = RMSNorm(512, device=gpu)
    norm.weight.data = 1 + 0.1 * torch.randn(512, generator=seeded(1)).to(gpu).bfloat16()
    x, r = (heavy_rows(6, 512, 20 + i).to(gpu).reshape(2, 3, 512) for i in range(2))
    rows, h = norm(x, r, layers)
    assert isinstance(rows, QuantizedRows) == (fmt != "int4") and h.shape == x.shape
    plain, h2 = norm(x, r)
    assert plain.shape == x.shape and torch.equal(h, h2) and torch.equal(h, x + r)
    first, h3 = norm(x)
    assert h3 is x and first.shape == x.shape
    for module in layers:
        y = linear(module, rows)
        if fmt == "int4":
            assert torch.equal(y, module(plain))
        else:
            q, s, _ = ops.add_rms_norm(x.reshape(6, 512), norm.weight, residual=r.reshape(6, 512), codes=fmt, rot_group=rows.rot_group)
            w = module.forward_codes(QuantizedRows(q, s, rows.rot_group, (2, 3, 512), torch.bfloat16))
            assert y.shape == (2, 3, module.out_features) and torch.equal(y, w)


HIDDEN, HEADS, KV, DIM, MLP = 512, 8, 2, 64, 768


def decoder(fmt, opts, gpu, layers=2, dtype=torch.bfloat16):
    """Layers with quantized weights; [{name: dequantized weight}]."""
    from powershard_amd.decoder import DecoderLayer
    from powershard_amd.quant_linear import install_quant_linears, pack, quantized_from_float
    g, made, weights = seeded(3), [], []
    for _ in range(layers):
        layer = DecoderLayer(HIDDEN, HEADS, KV, DIM, MLP, dtype=dtype, device=gpu)
        names = [n for n, m in layer.named_modules() if isinstance(m, nn.Linear)]
        shapes = {n: tuple(layer.get_submodule(n).weight.shape) for n in names}
        tensors = {n + ".weight": {"key": n + ".weight", "dtype": "BF16", "shape": list(shapes[n])} for n in names}
        install_quant_linears(layer, tensors, fmt, "native", None, dtype, gpu, quant_options=opts)
        deq = {}
        for n in names:
            module = layer.get_submodule(n)
            w = (torch.randn(shapes[n], generator=g) * shapes[n][1] ** -0.5).to(torch.bfloat16)
            qt = quantized_from_float(w, module._ps_qplan.fmt, **opts)
            module.qbytes = nn.Parameter(pack(qt, module._ps_qplan, gpu), requires_grad=False)
            deq[n] = qt.dequantize().double()
        for n in ("norm1", "norm2"):
            module = getattr(layer, n)
            module.weight.data = (1 + 0.1 * torch.randn(HIDDEN, generator=g)).to(dtype).to(gpu)
            deq[n] = module.weight.double().cpu()
        made.append(layer)
        weights.append(deq)
    return made, weights


def run_prompt(layers, cache, seq, x):
    slots, h = cache.extend([seq], x.shape[0]), None
    for i, layer in enumerate(layers):
        x, h = layer.prompt(x, h, cache, i, seq, slots)
    return x.float() + h.float()


def run_step(layers, cache, seqs, x):
    slots, h = cache.extend(seqs, 1), None
    table = cache.table(seqs)
    for i, layer in enumerate(layers):
        x, h = layer.step(x, h, cache, i, slots, table)
    return x.float() + h.float()


@pytest.mark.parametrize("codes", [None, "int8", "fp8"])
@pytest.mark.parametrize("fmt,opts", [("int8", ROT), ("fp8", {}), ("int4", {"group_size": 128})])
def test_tokens_one_by_one_equal_the_prompt(gpu, fmt, opts, codes):
    """Two sequences of ragged lengths: a prompt, then token by token, against all of it as a prompt.

    Both forms see the same codes in the cache and differ in the order of fp32 sums, so in the roundings of
    attention outputs that this turns over, and in the codes that those turn over: bound 2 layers x 4
    linears x 2^-8 of the rows' norm."""
    from powershard_amd.kv_cache import PagedKVCache
    layers, _ = decoder(fmt, opts, gpu)
    texts = [heavy_rows(n, HIDDEN, 40 + n, outlier_frac=0).to(gpu) for n in (45, 70)]
    with torch.no_grad():
        ref = PagedKVCache(2, 12, 16, KV, DIM, codes=codes, device=gpu)
        want = [run_prompt(layers, ref, ref.open(), t) for t in texts]
        cache = PagedKVCache(2, 12, 16, KV, DIM, codes=codes, device=gpu)
        seqs = [cache.open(), cache.open()]
        steps = 12
        for s, t in zip(seqs, texts):
            got = run_prompt(layers, cache, s, t[:len(t) - steps])
            part = want[seqs.index(s)][:len(t) - steps]
            assert (got - part).norm() <= 2.0 ** -5 * part.norm()
        for k in range(steps):
            y = run_step(layers, cache, seqs, torch.stack([t[len(t) - steps + k] for t in texts]))
            w = torch.stack([x[len(t) - steps + k] for x, t in zip(want, texts)])
            assert (y - w).norm() <= 2.0 ** -5 * w.norm(), k
    assert all(m._ps_native for layer in layers for m in layer.modules() if hasattr(m, "_ps_native"))


def test_against_64_bits(gpu):
    """Weight-only layers on a 16-bit cache: only bf16 roundings (about 20 a layer on the way, 2^-9 rms
    each, so sqrt(40) 2^-9 of the norm, 1.3%; bound 2^-5) separate them from the formula."""
    from powershard_amd.decoder import rope
    from powershard_amd.kv_cache import PagedKVCache
    layers, weights = decoder("int4", {"group_size": 128}, gpu)
    x = heavy_rows(33, HIDDEN, 50, outlier_frac=0).to(gpu)
    with torch.no_grad():
        cache = PagedKVCache(2, 8, 16, KV, DIM, device=gpu)
        seq = cache.open()
        run_prompt(layers, cache, seq, x[:20])
        got = torch.cat([run_step(layers, cache, [seq], x[t:t + 1]) for t in range(20, 33)]).double().cpu()
    h, y = torch.zeros(33, HIDDEN, dtype=torch.float64), x.double().cpu()
    at = torch.arange(33)
    for w in weights:
        def norm(t, g):
            return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g
        h = h + y
        rows = norm(h, w["norm1"])
        q, k, v = (rows @ w[n + "_proj"].T for n in "qkv")
        q, k = (rope(t.float().reshape(33, -1, DIM), at).double() for t in (q, k))
        v = v.reshape(33, KV, DIM)
        out = torch.zeros(33, HEADS, DIM, dtype=torch.float64)
        for i in range(HEADS):
            s = (q[:, i] @ k[:, i * KV // HEADS].T / DIM ** 0.5).masked_fill(at > at[:, None], float("-inf"))
            out[:, i] = torch.softmax(s, -1) @ v[:, i * KV // HEADS]
        h = h + out.reshape(33, -1) @ w["o_proj"].T
        gate, up = (norm(h, w["norm2"]) @ w["up_proj"].T).chunk(2, -1)
        y = (nn.functional.silu(gate) * up) @ w["down_proj"].T
    want = (h + y)[20:]
    assert (got - want).norm() <= 2.0 ** -5 * want.norm()


def test_step_in_a_graph(gpu):
    """Norm, cache write, attention and read-back captured once and replayed as the text grows, with eager
    work in between: every replay has the eager call's bits."""
    from powershard_amd import ops
    from powershard_amd.kv_cache import PagedKVCache
    B, H, D, K = 5, 10, 128, 1280
    caches = [PagedKVCache(1, 200, 16, 2, D, codes="int8", device=gpu) for _ in range(2)]
    g = torch.Generator(device=gpu).manual_seed(1)
    seqs = [[c.open() for _ in range(B)] for c in caches]
    past = [torch.randn(n, 2, 2, D, generator=g, device=gpu).bfloat16() for n in (300, 0, 17, 511, 1)]
    for c, ids in zip(caches, seqs):
        for s, p in zip(ids, past):
            c.write(0, p[:, 0], p[:, 1], c.extend([s], len(p)))
    x = torch.zeros(B, K, dtype=torch.bfloat16, device=gpu)
    r, w = torch.zeros_like(x), torch.ones(K, device=gpu)
    kv = torch.zeros(B, 2, 2, D, dtype=torch.bfloat16, device=gpu)
    slots = torch.full((B,), -1, dtype=torch.int64, device=gpu)
    table = torch.full((B, 40), -1, dtype=torch.int32, device=gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)

    def step(cache):
        q, scale, h = ops.add_rms_norm(x, w, residual=r, codes="int8", rot_group=256)
        cache.write(0, kv[:, 0], kv[:, 1], slots)
        out = cache.attend(0, h.view(B, H, D), table, lengths, 640)
        return (q, scale, h, out) + cache.read(0, slots)

    stream = torch.cuda.Stream(gpu)
    stream.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(stream):       # the stream's workspace is made, and zeroed, before the capture
        step(caches[0])
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = step(caches[0])
    for _ in range(5):
        x.normal_(generator=g)
        r.normal_(generator=g)
        kv.normal_(generator=g)
        new = [c.extend(ids, 1) for c, ids in zip(caches, seqs)]
        assert torch.equal(new[0], new[1])
        slots.copy_(new[0])
        t, n, _ = caches[0].table(seqs[0])
        table[:, :t.shape[1]] = t
        lengths.copy_(n)
        graph.replay()
        got = [t.clone() for t in captured]
        want = step(caches[1])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt,opts", Q8)
def test_forward_codes_of_rows_in_other_layouts(gpu, fmt, opts):
    """Codes and scales that are slices, broadcasts or off 16 bytes have the values of dense ones."""
    from powershard_amd import ops
    from powershard_amd.quant_linear import QuantizedRows
    layer, _, _ = make_layer(512, 96, fmt, opts, torch.bfloat16, True, gpu, seed=5)
    kind, group = layer.input_codes()
    x = heavy_rows(7, 512, 6).to(gpu)
    q, scale = ops.quantize_rows(x, fp8=fmt == "fp8", rot_group=group)
    rows = QuantizedRows(q, scale, group, (7, 512), torch.bfloat16)
    want = layer.forward_codes(rows)
    wide = torch.zeros(7, 1024, dtype=torch.uint8, device=gpu)
    wide[:, 512:] = q.view(torch.uint8)
    odd = torch.zeros(7 * 512 + 1, dtype=torch.uint8, device=gpu)[1:].view(7, 512)
    odd.copy_(q.view(torch.uint8))
    for codes in (wide[:, 512:].view(q.dtype), odd.view(q.dtype)):
        assert torch.equal(layer.forward_codes(rows._replace(codes=codes)), want)
    apart = torch.zeros(14, device=gpu)
    apart[::2] = scale
    assert torch.equal(layer.forward_codes(rows._replace(scale=apart[::2])), want)
    one = rows._replace(codes=q[:1].expand(7, 512), scale=scale[:1].expand(7))
    assert torch.equal(layer.forward_codes(one), want[:1].expand(7, 96))


@pytest.mark.parametrize("fmt,opts", Q8)
@pytest.mark.parametrize("activation", [None, "silu_gate"])
def test_forward_codes_follows_the_rows_dtype(gpu, fmt, opts, activation):
    """A text-encoder module gives back the dtype of the rows, as its forward does."""
    from powershard_amd import ops
    from powershard_amd.quant_linear import QuantizedRows
    layer, _, _ = make_layer(512, 256, fmt, opts, torch.bfloat16, True, gpu, seed=5, follow_input=True)
    kind, group = layer.input_codes()
    x = heavy_rows(3, 512, 6).to(gpu)
    q, scale = ops.quantize_rows(x, fp8=fmt == "fp8", rot_group=group)
    for dtype in (torch.float16, torch.float32, torch.bfloat16):
        got = layer.forward_codes(QuantizedRows(q, scale, group, (3, 512), dtype), activation)
        want = layer(x) if activation is None else layer.forward_act(x, activation)
        assert got.dtype is dtype and torch.equal(got, want.to(dtype))
    assert layer._ps_native


def test_layers_and_linears_run_their_hooks(gpu):
    """prompt and step are module calls, and the linears are called as modules with the norm's codes."""
    from powershard_amd.kv_cache import PagedKVCache
    from powershard_amd.quant_linear import QuantizedRows
    layers, _ = decoder("int8", ROT, gpu, layers=1)
    calls, x = [], heavy_rows(5, HIDDEN, 61, outlier_frac=0).to(gpu)
    cache = PagedKVCache(1, 4, 16, KV, DIM, device=gpu)
    seq = cache.open()
    layer = layers[0]
    layer.register_forward_pre_hook(lambda m, args: calls.append("layer"))
    layer.q_proj.register_forward_pre_hook(lambda m, args: calls.append(type(args[0])))
    with torch.no_grad():
        run_prompt(layers, cache, seq, x)
        run_step(layers, cache, [seq], x[:1])
    assert calls == ["layer", QuantizedRows] * 2
    with pytest.raises(ValueError):
        layer(x, None, cache, 0, cache.slots(seq))


def test_int8_scales_are_counted(gpu):
    """A kernel reads one scale per int8 row: fewer are refused (forward_codes: one warning first, as the forward)."""
    from powershard_amd import ops
    from powershard_amd import quant_tensor as qtm
    from powershard_amd.quant_linear import QuantizedRows, QuantPlan, pack
    q = torch.ones(96, 512, dtype=torch.int8, device=gpu)
    with pytest.raises(ValueError):
        ops.dequant_i8_rows(q, torch.ones(1, device=gpu))
    with pytest.raises(ValueError):
        ops.dequant_i8_rows(q, torch.ones(97, 1, device=gpu))
    layer, _, _ = make_layer(512, 96, "int8", {"convrot": False}, torch.bfloat16, True, gpu, seed=5)
    weight = qtm.QuantizedWeight(q, qtm.Int8RowwiseLayout, qtm.Int8RowwiseParams(torch.ones(1, device=gpu)))
    layer._ps_qplan = QuantPlan.of(weight, layer._ps_qplan.fmt, {})
    layer.qbytes = nn.Parameter(pack(weight, layer._ps_qplan, gpu), requires_grad=False)
    rows = QuantizedRows(q[:5].clone(), torch.ones(5, device=gpu), 0, (5, 512), torch.bfloat16)
    with pytest.warns(UserWarning, match="switches to dequantize"), pytest.raises(ValueError):
        layer.forward_codes(rows)
