"""The direct calls (csrc/direct.cpp) of the rotary write and of the prompts' and trees' attention against the general path
of ops.py: the same bits for what both take, None and the same refusals for the rest."""
import pytest
import torch

from powershard_amd import _native, ops
from test_direct_calls_gpu import DEV, KINDS, cache, general, rand, raw, same

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def setup(kind):
    pools = cache(kind)
    return pools, kind if pools[2] is None else torch.bfloat16


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("T,bits,axes,interleaved", [(0, 32, False, False), (1, 64, False, True), (5, 32, True, False), (5, 64, True, True)])
def test_rope(monkeypatch, kind, T, bits, axes, interleaved):
    pools, dtype = setup(kind)
    q, k, v = rand(T, 8, 64, dtype=dtype, seed=1)[:, 2:], rand(T, 3, 2, 64, dtype=dtype, seed=2)[:, 1], rand(T, 2, 64, dtype=dtype, seed=3)
    positions = torch.arange(3 * T, device=DEV).view(3, T).to(torch.int32 if bits == 32 else torch.int64)
    positions, axis = (positions, i32([0, 1, 2, 2] * 4)) if axes else (positions[1], None)
    freq = 100.0 ** (-torch.arange(16, dtype=torch.float64, device=DEV) / 16)
    slots = torch.tensor([40, -1, 3, 95, 17][:T], dtype=torch.int64, device=DEV)
    apart = [None if t is None else t.clone() for t in pools]
    done = _native.direct().rope_kv_write(q, k, v, positions, freq, slots, *pools, axis, interleaved, raw())
    assert done is not None
    call = lambda p: ops.rope_kv_write(q, k, v, positions, freq, slots, *p, axes=axis, interleaved=interleaved)   # noqa: E731
    same(done, general(monkeypatch, lambda: call(apart)))
    same(pools, apart)
    same(call(pools), done)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("scale,window,sinks,max_len", [(None, 0, 0, None), (0.3, 20, 3, 96), (-1.0, 0, 0, 5), (None, 500, 0, -1)])
def test_blocks(monkeypatch, kind, lse, scale, window, sinks, max_len):
    pools, dtype = setup(kind)
    table = i32([[0, 3, 1, 2, 9], [5, 4, 0, 1, 9]])[:, :4]
    lengths, starts = i32([64, 33]), i32([0, 7, 10])
    q = rand(10, 12, 64, dtype=dtype, seed=9)[:, 2:8]
    options = dict(scale=scale, window=window, sinks=sinks, max_len=max_len, return_lse=lse)
    call = lambda: ops.paged_prompt_attention(q, *pools[:2], table, starts, lengths, *pools[2:], **options)   # noqa: E731
    want = general(monkeypatch, call)
    done = _native.direct().paged_prompt_attention(q, *pools, table, lengths, starts, None, scale, window, sinks, max_len, lse, raw())
    assert done is not None
    same(done, want)
    same(call(), want)
    tree, parents = q.view(2, 5, 6, 64), i32([[-1, 0, 1, 0, 3], [-1, -1, 1, 1, 0]])
    for drafts in (None, i32([5, 2])):
        call = lambda: ops.paged_tree_attention(tree, *pools[:2], table, lengths, parents, *pools[2:], drafts=drafts, **options)   # noqa: E731,B023
        want = general(monkeypatch, call)
        done = _native.direct().paged_tree_attention(tree, *pools, table, lengths, parents, drafts, scale, window, sinks, max_len, lse, raw())
        assert done is not None
        same(done, want)
        same(call(), want)


def test_what_is_left_to_the_general_path(monkeypatch):
    pools, dtype = setup(torch.int8)
    table, lengths, starts, parents = i32([[0, 3, 1, 2]]), i32([64]), i32([0, 3]), i32([[-1, 0, 0]])
    q, k, v = rand(3, 4, 64, dtype=dtype), rand(3, 2, 64, dtype=dtype), rand(3, 2, 64, dtype=dtype)
    freq, at, slots = torch.ones(16, dtype=torch.float64, device=DEV), i32([0, 1, 2]), torch.arange(3, device=DEV)
    wide = torch.zeros(3, 4, 128, dtype=dtype, device=DEV)[..., ::2]
    wide.copy_(q)
    direct = _native.direct()
    prompt = lambda q=q, table=table, lengths=lengths, starts=starts, window=0, sinks=0: (   # noqa: E731
        (q, *pools, table, lengths, starts, None, None, window, sinks, None, False, raw()),
        lambda: ops.paged_prompt_attention(q, *pools[:2], table, starts, lengths, *pools[2:], window=window, sinks=sinks))
    tree = lambda q=q[None], parents=parents, drafts=None: (                                 # noqa: E731
        (q, *pools, table, lengths, parents, drafts, None, 0, 0, None, False, raw()),
        lambda: ops.paged_tree_attention(q, *pools[:2], table, lengths, parents, *pools[2:], drafts=drafts))
    rope = lambda q=q, k=k, at=at, freq=freq, slots=slots, axes=None: (                       # noqa: E731
        (q, k, v, at, freq, slots, *pools, axes, False, raw()),
        lambda: ops.rope_kv_write(q, k, v, at, freq, slots, *pools, axes=axes))
    spread = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    for name, (args, call) in [("prompt", prompt(q=wide)), ("prompt", prompt(table=torch.stack([table, table], -1)[..., 0])),
                               ("tree", tree(q=wide[None])), ("tree", tree(parents=torch.stack([parents, parents], -1)[..., 0])),
                               ("rope", rope(q=wide)), ("rope", rope(freq=freq.float())),
                               ("rope", rope(at=torch.stack([at, at], -1)[:, 0]))]:
        f = getattr(direct, {"prompt": "paged_prompt_attention", "tree": "paged_tree_attention", "rope": "rope_kv_write"}[name])
        assert f(*args) is None, name
        same(call(), general(monkeypatch, call))
    for name, (args, call) in [("prompt", prompt(q=q.half().float())), ("prompt", prompt(lengths=lengths.long())), ("prompt", prompt(starts=starts[:1])),
                               ("prompt", prompt(sinks=2)), ("prompt", prompt(window=-1)), ("prompt", prompt(lengths=spread[:, 0])),
                               ("prompt", prompt(table=table.cpu())), ("tree", tree(parents=parents[:, :2])), ("tree", tree(drafts=i32([1, 1]))),
                               ("tree", tree(q=rand(1, 65, 4, 64, dtype=dtype), parents=torch.zeros(1, 65, dtype=torch.int32, device=DEV))),
                               ("rope", rope(k=k.half())), ("rope", rope(freq=freq[:4])), ("rope", rope(at=at.float())), ("rope", rope(axes=at)),
                               ("rope", rope(slots=slots[:2])), ("rope", rope(slots=slots.int())), ("rope", rope(at=at.cpu()))]:
        f = getattr(direct, {"prompt": "paged_prompt_attention", "tree": "paged_tree_attention", "rope": "rope_kv_write"}[name])
        assert f(*args) is None, name
        errors = []
        for run in (call, lambda: general(monkeypatch, call)):   # noqa: B023
            with pytest.raises((TypeError, ValueError, RuntimeError)) as e:
                run()
            errors.append((e.type, str(e.value)))
        assert errors[0] == errors[1]
