"""The C entry points of the cache's rotated writes and of the attention of prompts and trees on the CPU: bad arguments are refused before any device is
touched, empty problems are no-ops, tensors that are not on a GPU are refused by the wrappers."""
import pytest
import torch

from powershard_amd import _native, ops

A = 0x10000
ARG, SHAPE = -1, -2


def append(codes=1, q=A, k=A, v=A, dt=0, strides=(512, 64, 256, 64, 256, 64), pos=A, bits=64, axes=1, stride=0, axis=None, freq=A, rotary=64,
           paired=0, slots=A, T=5, Hq=8, H=4, D=64, kc=A, vc=A, ks=A, vs=A, pages=8, page=16, out=A):
    return _native.lib().psq_rope_kv_write(codes, q, k, v, dt, *strides, pos, bits, axes, stride, axis, freq, rotary, paired, slots, T, Hq, H,
                                           D, kc, vc, ks, vs, pages, page, out, None)


def prompt(codes=1, q=A, dt=0, qt=512, qh=64, kc=A, vc=A, ks=A, vs=A, pages=8, page=16, table=A, stride=4, cols=4, starts=A, lens=A, B=2,
           T=9, Hq=8, Hk=4, D=64, scale=0.125, window=0, sinks=0, max_len=64, out=A, lse=None, ws=None, nb=0):
    return _native.lib().psq_paged_prompt_attention(codes, q, dt, qt, qh, kc, vc, ks, vs, pages, page, table, stride, cols, starts, lens, B, T,
                                                    Hq, Hk, D, scale, window, sinks, max_len, out, lse, ws, nb, None)


def tree(codes=1, q=A, dt=0, qt=512, qh=64, kc=A, vc=A, ks=A, vs=A, pages=8, page=16, table=A, stride=4, cols=4, lens=A, parents=A,
         drafts=None, B=2, N=9, Hq=8, Hk=4, D=64, scale=0.125, window=0, sinks=0, max_len=64, out=A, lse=None, ws=None, nb=0):
    return _native.lib().psq_paged_tree_attention(codes, q, dt, qt, qh, kc, vc, ks, vs, pages, page, table, stride, cols, lens, parents, drafts,
                                                  B, N, Hq, Hk, D, scale, window, sinks, max_len, out, lse, ws, nb, None)


BLOCKS = [(code, lambda f=f, bad=bad: f(**bad)) for f in (prompt, tree) for code, bad in [
    (ARG, dict(codes=3)), (ARG, dict(dt=2)), (ARG, dict(B=-1)), (ARG, dict(window=-1)), (ARG, dict(window=4, sinks=-1)), (ARG, dict(sinks=1)),
    (ARG, dict(max_len=-1)), (ARG, dict(nb=-1)), (ARG, dict(q=None)), (ARG, dict(out=None)), (ARG, dict(lens=None)), (ARG, dict(table=None)),
    (ARG, dict(ks=None)), (ARG, dict(Hk=0)), (ARG, dict(cols=-1)), (SHAPE, dict(Hq=6)), (SHAPE, dict(qh=68)), (SHAPE, dict(q=A + 8)),
    (SHAPE, dict(out=A + 8)), (SHAPE, dict(table=A + 2)), (SHAPE, dict(lens=A + 2)), (SHAPE, dict(lse=A + 2)), (SHAPE, dict(D=24)),
    (SHAPE, dict(page=20)), (SHAPE, dict(B=1 << 20)), (SHAPE, dict(cols=1 << 40)), (SHAPE, dict(kc=A + 4)), (SHAPE, dict(ws=A + 64, nb=1 << 20))]]


@pytest.mark.parametrize("code,call", BLOCKS + [
    (ARG, lambda: prompt(starts=None)), (ARG, lambda: prompt(T=-1)), (SHAPE, lambda: prompt(starts=A + 2)), (SHAPE, lambda: prompt(T=1 << 40)),
    (ARG, lambda: tree(parents=None)), (ARG, lambda: tree(N=-1)), (SHAPE, lambda: tree(N=65)), (SHAPE, lambda: tree(parents=A + 2)),
    (SHAPE, lambda: tree(drafts=A + 2)),
    (ARG, lambda: append(codes=3)), (ARG, lambda: append(dt=2)), (ARG, lambda: append(T=-1)), (ARG, lambda: append(Hq=-1)),
    (ARG, lambda: append(bits=16)), (ARG, lambda: append(q=None)), (ARG, lambda: append(k=None)), (ARG, lambda: append(v=None)),
    (ARG, lambda: append(slots=None)), (ARG, lambda: append(pos=None)), (ARG, lambda: append(freq=None)), (ARG, lambda: append(out=None)),
    (ARG, lambda: append(axes=0)), (ARG, lambda: append(axes=3)), (ARG, lambda: append(ks=None)), (ARG, lambda: append(kc=None)),
    (SHAPE, lambda: append(rotary=24)), (SHAPE, lambda: append(rotary=0)), (SHAPE, lambda: append(rotary=80)), (SHAPE, lambda: append(D=72)),
    (SHAPE, lambda: append(page=24)), (SHAPE, lambda: append(q=A + 8)), (SHAPE, lambda: append(out=A + 2)), (SHAPE, lambda: append(pos=A + 4)),
    (SHAPE, lambda: append(freq=A + 4)), (SHAPE, lambda: append(axis=A + 2)), (SHAPE, lambda: append(strides=(512, 64, 256, 60, 256, 64))),
    (SHAPE, lambda: append(T=1 << 31)), (SHAPE, lambda: append(Hq=1 << 16)),
])
def test_refused_without_a_device(code, call):
    assert call() == code
    assert _native.lib().psq_last_error().decode()


def test_empty_problems_are_no_ops():
    assert append(T=0, q=None, k=None, v=None, pos=None, slots=None, freq=None, out=None) == 0
    assert prompt(T=0, q=None, out=None) == 0 and prompt(Hq=0, q=None, out=None) == 0
    assert tree(B=0, q=None, out=None) == 0 and tree(N=0, q=None, out=None) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    at = torch.arange(2)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.paged_prompt_attention(x, pool, pool, one[None], torch.tensor([0, 2], dtype=torch.int32), one)
    with pytest.raises(RuntimeError):
        ops.paged_tree_attention(x[None], pool, pool, one[None], one, torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        ops.rope_kv_write(x, x, x, at, torch.ones(32, dtype=torch.float64), at, pool, pool)
