"""QuantLinear.forward_codes on the CPU: the rows that it refuses (no kernel runs here)."""
import pytest
import torch

from powershard_amd.quant_linear import QuantizedRows
from test_quant_linear_cpu import make_layer


def layer(weight_format, **kw):
    module = make_layer(weight_format, **kw)[0][0]
    module._ps_native = True
    return module


def rows(M=6, K=128, dtype=torch.int8, shape=None, scale=None, group=0):
    codes = torch.zeros(M, K, dtype=torch.uint8).view(dtype) if dtype.itemsize == 1 else torch.zeros(M, K, dtype=dtype)
    return QuantizedRows(codes, torch.ones(M) if scale is None else scale, group, shape or (2, 3, K), torch.bfloat16)


@pytest.mark.parametrize("bad", [
    rows(scale=torch.ones(5)), rows(scale=torch.ones(6, dtype=torch.float64)), rows(scale=torch.ones(6, 1)),
    rows(scale=torch.ones((), dtype=torch.float32)), rows(scale=torch.ones(6, device="meta")), rows(shape=(2, 2, 128)),
    rows(shape=(6, 64)), rows(shape=(7, 128)), rows(dtype=torch.uint8), rows(dtype=torch.float16),
    rows()._replace(codes=torch.zeros(6, 2, 128, dtype=torch.int8)),
], ids=lambda r: f"{r.codes.dtype}-{tuple(r.scale.shape)}-{r.shape}")
def test_rows_that_do_not_belong_together(bad):
    with pytest.raises(ValueError):
        layer("int8", opts={"convrot": False}).forward_codes(bad)


@pytest.mark.parametrize("dtype", [torch.float8_e5m2, torch.uint8, torch.int8])
def test_codes_of_another_kind(dtype):
    with pytest.raises(ValueError):
        layer("fp8").forward_codes(rows(dtype=dtype))


def test_which_rows_are_plain():
    """Only dense rows and scales go to the library by their addresses."""
    assert rows().plain()
    wide = torch.zeros(6, 256, dtype=torch.int8)
    for codes in (wide[:, :128], wide[:1, :128].expand(6, 128), torch.zeros(128, 6, dtype=torch.int8).t(),
                  torch.zeros(6 * 128 + 1, dtype=torch.int8)[1:].view(6, 128)):
        assert not rows()._replace(codes=codes).plain()
    assert not rows(scale=torch.ones(12)[::2]).plain() and not rows(scale=torch.ones(1).expand(6)).plain()
