"""add_rms_norm against its formula in 64 bits.

Tolerances, from the arithmetic: the sum h is one fp32 addition and one rounding, so it is exact.  In
fp32 the normalized values are within a few ulp of their row's largest (products, at most five transform
stages of adds: 2^-20 of it), the sum of squares within (16 + 6 + 16) 2^-24 of itself (a thread's chunk,
its wave, the waves), so scales are within 4e-6; a code is the nearest to y / scale up to these errors."""
import pytest
import torch

from conftest import heavy_rows, seeded

pytestmark = pytest.mark.gpu

LIMIT = {"int8": 127.0, "fp8": 448.0}
U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # unit roundoff: 8 and 11 significant bits


def _inputs(M, K, dtype, seed, gpu):
    x = heavy_rows(M, K, seed, dtype=dtype).to(gpu)
    r = heavy_rows(M, K, seed + 1, dtype=dtype).to(gpu) * 2
    w = (1 + 0.2 * torch.randn(K, generator=seeded(seed + 2))).to(gpu)
    return x, r, w


def _formula(h, w, eps, rot):
    import oracle
    h, w = h.double().cpu(), w.double().cpu()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w
    if rot:
        y = (y.reshape(len(y), -1, rot) @ oracle.regular_hadamard(rot).double()).reshape(y.shape)
    return y


def _check_codes(q, scale, y, codes, static=None):
    lim = LIMIT[codes]
    amax = y.abs().amax(-1)
    want = torch.where(amax == 0, 1.0, amax / lim) if static is None else torch.full_like(amax, static)
    scale = scale.double().cpu()
    assert ((scale - want).abs() <= 4e-6 * want).all()
    u = (y / scale[:, None]).clamp(-lim, lim)
    step = torch.ones_like(u) if codes == "int8" else \
        torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3)
    assert ((q.float().double().cpu() - u).abs() <= step * 0.5 + 4e-6 * u.abs() + 2.0 ** -20 * lim).all()


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,rot", [(1, 16, 0), (3, 48, 16), (2, 1008, 0), (5, 1024, 4), (4, 1024, 64), (1, 5120, 256), (7, 5376, 256),
                                     (3, 4096, 1024), (2, 16400, 0), (2, 32768, 0), (300, 512, 0)])
def test_codes(gpu, codes, dtype, M, K, rot):
    from powershard_amd import ops
    if codes == "fp8" and rot not in (0, 256):
        rot = 0
    x, r, w = _inputs(M, K, dtype, 11 + M + K, gpu)
    for res in (None, r):
        q, scale, h = ops.add_rms_norm(x, w, 1e-6, residual=res, codes=codes, rot_group=rot)
        assert (h is None) == (res is None)
        h = x if res is None else h
        assert res is None or torch.equal(h, (x.float() + res.float()).to(dtype))
        _check_codes(q, scale, _formula(h, w, 1e-6, rot), codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,rot", [(1, 16, 0), (6, 5120, 0), (2, 2048, 256), (3, 20000, 0)])
def test_16_bit_rows(gpu, dtype, wdtype, M, K, rot):
    from powershard_amd import ops
    x, r, w = _inputs(M, K, dtype, 5 + K, gpu)
    w = w.to(wdtype)
    y, scale, h = ops.add_rms_norm(x, w, 1e-5, residual=r, rot_group=rot)
    assert scale is None and y.dtype == dtype
    want = _formula(h, w, 1e-5, rot)
    tol = (U16[dtype] + 4e-6) * want.abs() + 2.0 ** -25 + (2.0 ** -20 * want.abs().amax(-1, keepdim=True) if rot else 0)
    assert ((y.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_static_scale(gpu, codes):
    from powershard_amd import ops
    x, r, w = _inputs(9, 1024, torch.bfloat16, 3, gpu)
    static = torch.tensor([0.02], device=gpu)
    q, scale, h = ops.add_rms_norm(x, w, residual=r, codes=codes, static_scale=static)
    assert torch.equal(scale, static.expand(9))
    _check_codes(q, scale, _formula(h, w, 1e-6, 0), codes, float(static))


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_rows_of_zeros_nan_and_inf(gpu, codes):
    """A zero row has scale 1 and codes 0; one NaN or Inf makes its row's scale NaN and no other's."""
    from powershard_amd import ops
    x = heavy_rows(6, 512, 8).to(gpu)
    w = torch.ones(512, device=gpu)
    x[1] = 0
    x[2, 77] = float("nan")
    x[4, 500] = float("-inf")
    x[5] = 1e-38
    q, scale, _ = ops.add_rms_norm(x, w, codes=codes)
    assert scale[1] == 1 and (q[1].float() == 0).all() and scale[5] == 1 and (q[5].float() == 0).all()
    assert scale.isnan().tolist() == [False, False, True, False, True, False]
    same, s, _ = ops.add_rms_norm(x[3:4], w, codes=codes)
    assert torch.equal(q[3:4].view(torch.uint8), same.view(torch.uint8)) and scale[3] == s[0]


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("rot", [0, 16])
def test_rows_at_the_edge_of_zero(gpu, codes, rot):
    """Rows whose 127 / max or 448 / max is at the end of fp32: zero rows below the limit, the nearest codes from
    there on.  (One element per group of 16: its transform has the element's size everywhere.)"""
    from powershard_amd import ops
    tops = [2.0 ** -121, 2.0 ** -120, 1.5 * 2.0 ** -120, 1.75 * 2.0 ** -120, 2.0 ** -119, 1.5 * 2.0 ** -119, 2.0 ** -110]
    x = torch.zeros(len(tops), 64)
    x[:, 16] = torch.tensor(tops)
    x[:, 37] = -0.25 * torch.tensor(tops)
    x = x.to(torch.bfloat16).to(gpu)
    w = torch.ones(64, device=gpu)
    q, scale, _ = ops.add_rms_norm(x, w, eps=1.0, codes=codes, rot_group=0 if codes == "fp8" else rot)
    limit = 2.0 ** -120 if codes == "int8" else 2.0 ** -119
    y = _formula(x, w, 1.0, rot if codes == "int8" else 0)
    for i, top in enumerate(tops):
        if top >= limit:
            _check_codes(q[i:i + 1], scale[i:i + 1], y[i:i + 1], codes)
        else:
            assert (q[i].float() == 0).all() and scale[i] == 1, top


def test_strided_offset_and_empty_rows(gpu):
    from powershard_amd import ops
    x, r, w = _inputs(5, 512, torch.bfloat16, 21, gpu)
    ref = ops.add_rms_norm(x, w, residual=r, codes="int8", rot_group=256)
    wide = torch.zeros(5, 1032, dtype=x.dtype, device=gpu)
    wide[:, 8:520] = x
    odd = torch.zeros(5 * 512 + 3, dtype=x.dtype, device=gpu)[3:].view(5, 512)
    odd.copy_(r)
    got = ops.add_rms_norm(wide[:, 8:520], w, residual=odd, codes="int8", rot_group=256)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    one = ops.add_rms_norm(x[:1].expand(5, 512), w, residual=r[:1].expand(5, 512), codes="int8", rot_group=256)
    assert all(torch.equal(a[:1].expand_as(b), b) for a, b in zip(ref, one))
    q, scale, h = ops.add_rms_norm(x[:0], w, residual=r[:0], codes="fp8")
    assert q.shape == (0, 512) and scale.shape == (0,) and h.shape == (0, 512)


@pytest.mark.parametrize("over", ["x", "residual"])
def test_sum_in_place(gpu, over):
    """The sum may be written over x or over the residual."""
    from powershard_amd import _native, ops
    x, r, w = _inputs(7, 1024, torch.bfloat16, 23, gpu)
    q, scale, h = ops.add_rms_norm(x, w, residual=r, codes="int8", rot_group=256)
    to = x if over == "x" else r
    q2, s2 = torch.empty_like(q), torch.empty_like(scale)
    _native.check(_native.lib().psq_add_rms_norm(
        _native.CODES_I8, x.data_ptr(), _native.BF16, 1024, r.data_ptr(), 1024, w.data_ptr(), _native.F32, 1e-6, to.data_ptr(), 1024,
        256, None, q2.data_ptr(), 1024, s2.data_ptr(), 7, 1024, torch.cuda.current_stream(gpu).cuda_stream), "add_rms_norm")
    assert torch.equal(to, h) and torch.equal(q, q2) and torch.equal(scale, s2)


def test_feeds_the_gemm(gpu):
    """norm -> int8 GEMM equals the GEMM of the dequantized rows."""
    from powershard_amd import ops
    x, r, w = _inputs(4, 512, torch.bfloat16, 31, gpu)
    q, scale, _ = ops.add_rms_norm(x, w, residual=r, codes="int8")
    wq = torch.randint(-127, 128, (96, 512), generator=seeded(4), dtype=torch.int8).to(gpu)
    ws = torch.rand(96, generator=seeded(5)).to(gpu)
    y = ops.gemm_i8(q, scale, wq, ws, out_dtype=torch.float32)
    want = (q.double() @ wq.double().T) * scale.double()[:, None] * ws.double()
    assert ((y.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()


def test_another_stream(gpu):
    from powershard_amd import ops
    x, r, w = _inputs(33, 2048, torch.bfloat16, 41, gpu)
    ref = ops.add_rms_norm(x, w, residual=r, codes="fp8")
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        got = ops.add_rms_norm(x, w, residual=r, codes="fp8")
    side.synchronize()
    assert torch.equal(ref[0].view(torch.uint8), got[0].view(torch.uint8)) and torch.equal(ref[1], got[1]) and torch.equal(ref[2], got[2])


def test_refusals(gpu):
    from powershard_amd import ops
    x, r, w = _inputs(2, 512, torch.bfloat16, 1, gpu)
    for error, call in [
            (ValueError, lambda: ops.add_rms_norm(x, w, codes="int4")),
            (ValueError, lambda: ops.add_rms_norm(x, w[:256], codes="int8")),
            (ValueError, lambda: ops.add_rms_norm(x, w, residual=r[:1])),
            (ValueError, lambda: ops.add_rms_norm(x, w, residual=r.half())),
            (ValueError, lambda: ops.add_rms_norm(x, w, static_scale=w[:1])),
            (TypeError, lambda: ops.add_rms_norm(x.float(), w, codes="int8")),
            (TypeError, lambda: ops.add_rms_norm(x, w.double(), codes="int8")),
            (RuntimeError, lambda: ops.add_rms_norm(x, w.cpu(), codes="int8")),
            (RuntimeError, lambda: ops.add_rms_norm(x[:, :504].contiguous(), w[:504].contiguous(), codes="int8")),
            (RuntimeError, lambda: ops.add_rms_norm(x, w, codes="int8", rot_group=128)),
            (RuntimeError, lambda: ops.add_rms_norm(x, w, eps=-1.0, codes="int8"))]:
        with pytest.raises(error):
            call()
