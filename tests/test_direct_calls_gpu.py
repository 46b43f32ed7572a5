"""The decoder operators' direct calls (csrc/direct.cpp) against the general path of ops.py: the same bits for
arguments that both take, None for those that only the general path takes, the same refusals."""
import pytest
import torch

from powershard_amd import _native, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def raw():
    return torch.cuda.current_stream(DEV).cuda_stream


def general(monkeypatch, call):
    """call() with the direct calls off."""
    with monkeypatch.context() as m:
        m.setattr(_native, "_direct", False)
        return call()


def same(a, b):
    a, b = [(t,) if isinstance(t, torch.Tensor) else t for t in (a, b)]
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype is y.dtype and x.shape == y.shape and x.stride() == y.stride()
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def rand(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def cache(kind, Hk=2, D=64, pages=6, page=16, seed=3):
    """k, v, k_scale, v_scale filled with tokens 0 .. pages * page - 1 at their own slots."""
    n = pages * page
    shape = (pages, Hk, page, D)
    coded = kind in (torch.int8, torch.float8_e4m3fn)
    pools = [torch.zeros(shape, dtype=kind, device=DEV) for _ in range(2)]
    pools += [torch.zeros(shape[:3], device=DEV) if coded else None for _ in range(2)]
    dtype = torch.bfloat16 if coded else kind
    ops.kv_write(rand(n, Hk, D, dtype=dtype, seed=seed), rand(n, Hk, D, dtype=dtype, seed=seed + 1), torch.arange(n, device=DEV), *pools)
    return pools


KINDS = [torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("codes", [None, "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,with_res,rot", [(1, 512, True, 0), (5, 768, False, 256), (0, 64, True, 0)])
def test_norm(monkeypatch, codes, dtype, M, K, with_res, rot):
    x, w, r = rand(M, K, dtype=dtype), rand(K, dtype=torch.float32, seed=1), rand(M, K, dtype=dtype, seed=2) if with_res else None
    done = _native.direct().add_rms_norm(x, w, 1e-6, r, ops.CODES[codes], rot, raw())
    assert done is not None
    call = lambda: ops.add_rms_norm(x, w, 1e-6, residual=r, codes=codes, rot_group=rot)   # noqa: E731
    same(done, general(monkeypatch, call))
    same(call(), done)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("T", [0, 1, 7])
def test_cache(monkeypatch, kind, T):
    pools = cache(kind)
    k, v = [rand(T, 3, 2, 64, dtype=kind if pools[2] is None else torch.float16, seed=s)[:, 1] for s in (5, 6)]   # token strides of 3 rows
    slots = torch.tensor([40, -1, 3, 95, 17, 0, 64][:T], dtype=torch.int64, device=DEV)
    apart = [None if t is None else t.clone() for t in pools]
    assert _native.direct().kv_write(k, v, slots, *pools, raw()) is True
    general(monkeypatch, lambda: ops.kv_write(k, v, slots, *apart))
    same(pools, apart)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        done = _native.direct().kv_read(slots, *pools, ops._DT[out], raw())
        assert done is not None
        same(done, general(monkeypatch, lambda: ops.kv_read(slots, *pools, out_dtype=out)))
    same(ops.kv_read(slots, *pools), general(monkeypatch, lambda: ops.kv_read(slots, *pools)))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("scale,window,max_len", [(None, 0, None), (0.3, 20, 96), (None, 0, 5), (None, 500, -1)])
def test_attention(monkeypatch, kind, lse, scale, window, max_len):
    pools = cache(kind)
    q = rand(3, 12, 64, dtype=kind if pools[2] is None else torch.bfloat16, seed=9)[:, 2:8]     # rows apart
    table = torch.tensor([[0, 3, 1, 2, 9], [5, 4, 0, 1, 9], [2, 2, 2, 2, 9]], dtype=torch.int32, device=DEV)[:, :4]
    lengths = torch.tensor([64, 33, 0], dtype=torch.int32, device=DEV)
    call = lambda: ops.paged_attention(q, pools[0], pools[1], table, lengths, *pools[2:], scale=scale, window=window,   # noqa: E731
                                       max_len=max_len, return_lse=lse)
    want = general(monkeypatch, call)
    done = _native.direct().paged_attention(q, *pools, table, lengths, scale, window, max_len, lse, ops._workspaces.get((0, raw() or None)), raw())
    assert done is not None
    same(done, want)
    same(call(), want)


def test_a_workspace_is_made_where_there_is_none():
    pools = cache(torch.int8, pages=40)
    q = rand(1, 2, 64, seed=9)
    table = torch.arange(40, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor([640], dtype=torch.int32, device=DEV)
    want = ops.paged_attention(q, pools[0], pools[1], table, lengths, *pools[2:])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(DEV)
    args = (q, *pools, table, lengths, None, 0, None, False)
    with torch.cuda.stream(stream):
        assert _native.direct().paged_attention(*args, None, raw()) is None
        got = ops.paged_attention(q, pools[0], pools[1], table, lengths, *pools[2:])
        held = ops._workspaces.get((0, raw()))
        if held is not None:   # (None where this process has used more streams than workspaces are kept for)
            same(_native.direct().paged_attention(*args, held, raw()), got)
            assert _native.direct().paged_attention(*args, held[:64], raw()) is None
    stream.synchronize()
    bound = 4 * 2.0 ** -8 * want.float().abs().max()     # one rounding to bf16 each, of sums in another order
    assert (got.float() - want.float()).abs().max() <= bound


class Named(torch.Tensor):
    pass


def left_alone():
    """(name, a call of ops that has to come out as the general path alone does)."""
    x, w = rand(4, 512), rand(512, seed=1)
    wide = rand(4, 1024)
    pools = cache(torch.int8)
    k = rand(4, 2, 64)
    slots = torch.tensor([1, 99, 5, 99, 9, 99, 11, 99], device=DEV)[::2]
    q, table, lengths = rand(2, 4, 64), torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.tensor([5, 9], dtype=torch.int32, device=DEV)
    attend = lambda *a, **kw: ops.paged_attention(*a, *pools[2:], **kw)   # noqa: E731
    K, V, KS, VS = pools
    return {
        "column slice": lambda: ops.add_rms_norm(wide[:, :512], w, codes="int8"),
        "off 16 bytes": lambda: ops.add_rms_norm(wide.reshape(-1)[1:1 + 2048].view(4, 512), w, codes="int8"),
        "a subclass": lambda: ops.add_rms_norm(x.as_subclass(Named), w, codes="int8"),
        "transposed residual": lambda: ops.add_rms_norm(x, w, residual=rand(512, 4).t(), codes="fp8"),
        "static scale": lambda: ops.add_rms_norm(x, w, codes="int8", static_scale=torch.tensor([0.02])),
        "unknown codes": lambda: ops.add_rms_norm(x, w, codes="int3"),
        "K of 500": lambda: ops.add_rms_norm(rand(4, 500), rand(500)),
        "weight too long": lambda: ops.add_rms_norm(x, rand(513)),
        "residual of another type": lambda: ops.add_rms_norm(x, w, residual=x.half()),
        "f32 rows": lambda: ops.add_rms_norm(x.float(), w),
        "weight on the host": lambda: ops.add_rms_norm(x, w.cpu()),
        "a group of 128": lambda: ops.add_rms_norm(x, w, codes="int8", rot_group=128),
        "a negative eps": lambda: ops.add_rms_norm(x, w, eps=-1.0),
        "slots apart": lambda: ops.kv_read(slots, *pools),
        "int32 slots": lambda: ops.kv_read(slots.int(), *pools),
        "read as int8": lambda: ops.kv_read(slots, *pools, out_dtype=torch.int8),
        "no scales": lambda: ops.kv_read(slots, K, V),
        "scales of another shape": lambda: ops.kv_read(slots, K, V, KS[:-1], VS),
        "pools of two types": lambda: ops.kv_read(slots, K, V.view(torch.float8_e4m3fn), KS, VS),
        "pools sliced": lambda: ops.kv_read(slots, K[:, :1], V[:, :1], KS[:, :1], VS[:, :1]),
        "more keys than slots": lambda: ops.kv_write(k, k, slots[:3], *pools),
        "other heads": lambda: ops.kv_write(rand(4, 3, 64), rand(4, 3, 64), slots, *pools),
        "keys on the host": lambda: ops.kv_write(k, k.cpu(), slots, *pools),
        "f16 values": lambda: ops.kv_write(k, k.half(), slots, *pools),
        "queries with a stride": lambda: attend(rand(2, 4, 128)[..., ::2], K, V, table, lengths),
        "lengths apart": lambda: attend(q, K, V, table, lengths.repeat_interleave(2)[::2]),
        "int64 lengths": lambda: attend(q, K, V, table, lengths.long()),
        "table transposed": lambda: attend(q, K, V, torch.zeros(4, 2, dtype=torch.int32, device=DEV).t(), lengths),
        "one table": lambda: attend(q, K, V, table[:1], lengths),
        "3 heads on 2": lambda: attend(rand(2, 3, 64), K, V, table, lengths),
        "no window": lambda: attend(q, K, V, table, lengths, window=None),
        "a negative window": lambda: attend(q, K, V, table, lengths, window=-3),
        "dim of 128": lambda: attend(rand(2, 4, 128), K, V, table, lengths),
        "f32 queries": lambda: attend(q.float(), K, V, table, lengths),
    }


def test_what_is_left_to_the_general_path(monkeypatch):
    for name, call in left_alone().items():
        print(name, flush=True)
        outcomes = []
        for run in (call, lambda: general(monkeypatch, call)):
            try:
                outcomes.append(run())
            except (TypeError, ValueError, RuntimeError) as error:
                outcomes.append((type(error), str(error)))
        if isinstance(outcomes[0], tuple) and isinstance(outcomes[0][0], type):
            assert outcomes[0] == outcomes[1], name
        else:
            same(*outcomes)


def test_timed_launches_take_the_general_path():
    x, w = rand(4, 512), rand(512, seed=1)
    with ops.kernel_timer() as events:
        ops.add_rms_norm(x, w, codes="int8")
    assert len(events["add_rms_norm"]) == 1


def test_in_a_graph_and_in_inference_mode(monkeypatch):
    x, w, r = rand(4, 512), rand(512, seed=1), rand(4, 512, seed=2)
    want = general(monkeypatch, lambda: ops.add_rms_norm(x, w, residual=r, codes="int8"))
    with torch.inference_mode():
        same(ops.add_rms_norm(x, w, residual=r, codes="int8"), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.add_rms_norm(x, w, residual=r, codes="int8")
    for step in range(3):
        x.copy_(rand(4, 512, seed=10 + step))
        want = general(monkeypatch, lambda: ops.add_rms_norm(x, w, residual=r, codes="int8"))
        graph.replay()
        torch.cuda.synchronize()
        same(got, want)
