"""The C entry points of the cache's rotated writes on the CPU: bad arguments are refused before any device is
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


@pytest.mark.parametrize("code,call", [
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


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    at = torch.arange(2)
    with pytest.raises(RuntimeError):
        ops.rope_kv_write(x, x, x, at, torch.ones(32, dtype=torch.float64), at, pool, pool)
