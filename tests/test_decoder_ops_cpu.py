"""The decoder operators' C entry points on the CPU: bad arguments are refused before any device is
touched, empty problems are no-ops, and tensors that are not on a GPU are refused by the wrappers."""
import pytest
import torch

from powershard_amd import _native, ops

A = 0x10000


def norm(codes=1, x=A, dt=0, ldx=512, res=A, ldr=512, w=A, wdt=0, eps=1e-6, h=A, lds=512, rot=0, static=None, out=A, ldo=512, scale=A,
         M=4, K=512):
    return _native.lib().psq_add_rms_norm(codes, x, dt, ldx, res, ldr, w, wdt, eps, h, lds, rot, static, out, ldo, scale, M, K, None)


def write(codes=1, k=A, v=A, dt=0, strides=(256, 64, 256, 64), slots=A, T=5, H=4, D=64, kc=A, vc=A, ks=A, vs=A, pages=8, page=16):
    return _native.lib().psq_kv_write(codes, k, v, dt, *strides, slots, T, H, D, kc, vc, ks, vs, pages, page, None)


def read(codes=1, slots=A, T=5, kc=A, vc=A, cdt=0, ks=A, vs=A, pages=8, page=16, H=4, D=64, k=A, v=A, odt=0):
    return _native.lib().psq_kv_read(codes, slots, T, kc, vc, cdt, ks, vs, pages, page, H, D, k, v, odt, None)


def attend(codes=1, q=A, dt=0, qb=512, qh=64, kc=A, vc=A, ks=A, vs=A, pages=8, page=16, table=A, stride=4, cols=4, lens=A, B=2, Hq=8,
           Hk=4, D=64, scale=0.125, window=0, max_len=64, out=A, lse=None, ws=None, nb=0):
    return _native.lib().psq_paged_attention(codes, q, dt, qb, qh, kc, vc, ks, vs, pages, page, table, stride, cols, lens, B, Hq, Hk, D,
                                             scale, window, max_len, out, lse, ws, nb, None)


ARG, SHAPE = -1, -2


@pytest.mark.parametrize("code,call", [
    (ARG, lambda: norm(codes=3)), (ARG, lambda: norm(x=None)), (ARG, lambda: norm(res=None)), (ARG, lambda: norm(h=None)),
    (ARG, lambda: norm(scale=None)), (ARG, lambda: norm(dt=2)), (ARG, lambda: norm(wdt=3)), (ARG, lambda: norm(eps=-1.0)),
    (ARG, lambda: norm(eps=float("nan"))), (ARG, lambda: norm(M=-1)), (ARG, lambda: norm(codes=0, static=A)),
    (SHAPE, lambda: norm(K=500)), (SHAPE, lambda: norm(K=32784, ldx=32784, ldr=32784, lds=32784, ldo=32784)),
    (SHAPE, lambda: norm(ldx=504)), (SHAPE, lambda: norm(ldr=516)), (SHAPE, lambda: norm(ldo=520)), (SHAPE, lambda: norm(x=A + 8)),
    (SHAPE, lambda: norm(w=A + 2)), (SHAPE, lambda: norm(rot=128)), (SHAPE, lambda: norm(K=96, rot=64)), (SHAPE, lambda: norm(M=1 << 31)),
    (ARG, lambda: write(codes=-1)), (ARG, lambda: write(dt=2)), (ARG, lambda: write(T=-1)), (ARG, lambda: write(k=None)),
    (ARG, lambda: write(slots=None)), (ARG, lambda: write(ks=None)), (ARG, lambda: write(vc=None)), (ARG, lambda: write(page=0)),
    (ARG, lambda: write(H=0)), (ARG, lambda: write(pages=-1)), (SHAPE, lambda: write(D=72)), (SHAPE, lambda: write(D=272)),
    (SHAPE, lambda: write(page=24)), (SHAPE, lambda: write(strides=(256, 60, 256, 64))), (SHAPE, lambda: write(k=A + 2)),
    (SHAPE, lambda: write(kc=A + 8)), (SHAPE, lambda: write(slots=A + 4)), (SHAPE, lambda: write(T=1 << 40)),
    (ARG, lambda: read(odt=4)), (ARG, lambda: read(codes=0, cdt=2, ks=None, vs=None)), (ARG, lambda: read(k=None)),
    (ARG, lambda: read(vs=None)), (SHAPE, lambda: read(v=A + 8)), (SHAPE, lambda: read(D=40)), (SHAPE, lambda: read(T=1 << 40)),
    (ARG, lambda: attend(codes=7)), (ARG, lambda: attend(dt=2)), (ARG, lambda: attend(B=-1)), (ARG, lambda: attend(window=-1)),
    (ARG, lambda: attend(max_len=-1)), (ARG, lambda: attend(q=None)), (ARG, lambda: attend(out=None)), (ARG, lambda: attend(lens=None)),
    (ARG, lambda: attend(table=None)), (ARG, lambda: attend(ks=None)), (ARG, lambda: attend(Hk=0)), (SHAPE, lambda: attend(Hq=6)),
    (SHAPE, lambda: attend(qh=68)), (SHAPE, lambda: attend(q=A + 8)), (SHAPE, lambda: attend(table=A + 2)), (SHAPE, lambda: attend(D=24)),
    (SHAPE, lambda: attend(page=20)), (SHAPE, lambda: attend(B=1 << 20)), (SHAPE, lambda: attend(cols=1 << 40)),
    (SHAPE, lambda: attend(kc=A + 4)), (SHAPE, lambda: attend(ks=A + 4)),
])
def test_refused_without_a_device(code, call):
    assert call() == code
    assert _native.lib().psq_last_error().decode()


def test_empty_problems_are_no_ops():
    assert norm(M=0, x=None, res=None, h=None, out=None, scale=None) == 0
    assert write(T=0, k=None, v=None, slots=None) == 0
    assert write(pages=0, kc=None, vc=None, ks=None, vs=None) == 0
    assert read(T=0, k=None, v=None, slots=None) == 0
    assert attend(B=0, q=None, out=None, lens=None, table=None) == 0
    assert attend(Hq=0, q=None, out=None) == 0


def test_workspace_is_asked_for_without_a_device():
    assert _native.lib().psq_paged_attention_workspace_bytes(1, 0, 8, 4, 64, 1000) == 0
    assert _native.lib().psq_paged_attention_workspace_bytes(1, 2, 8, 4, 64, 0) == 0


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64)
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.add_rms_norm(x, w, codes="int8"),
                 lambda: ops.kv_write(x.view(2, 1, 64), x.view(2, 1, 64), torch.arange(2), pool, pool),
                 lambda: ops.kv_read(torch.arange(2), pool, pool),
                 lambda: ops.paged_attention(x.view(2, 1, 64)[:1], pool, pool, one.view(1, 1), one)):
        with pytest.raises(RuntimeError):
            call()
