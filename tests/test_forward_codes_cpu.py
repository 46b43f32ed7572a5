"""QuantLinear.forward_codes on the CPU, where no kernel runs: the rows that it refuses, and what it does when
the native call fails."""
import warnings

import pytest
import torch

from powershard_amd.quant_linear import QuantizedRows, pack, quantized_from_float
from powershard_amd.quant_tensor import regular_hadamard
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


@pytest.mark.parametrize("weight_format,opts", [("int8", {"convrot": True, "convrot_groupsize": 64}), ("int8", {"convrot": False}), ("fp8", {})])
@pytest.mark.parametrize("activation", [None, "gelu_tanh", "silu_gate"])
@pytest.mark.parametrize("follow", [False, True])
def test_a_failing_native_call_dequantizes(weight_format, opts, activation, follow):
    """Here every native call fails (no GPU): one warning, then the forward's values of the rows that the codes
    stand for, also for rows that were quantized before the module switched."""
    module = layer(weight_format, opts=opts, dtype=torch.bfloat16)
    module._ps_follow_input = follow
    weight = quantized_from_float(torch.randn(64, 128, generator=torch.Generator().manual_seed(1)), module._ps_qplan.fmt, **opts)
    module.qbytes = torch.nn.Parameter(pack(weight, module._ps_qplan, "cpu"), requires_grad=False)
    module.bias = torch.nn.Parameter(torch.linspace(-1, 1, 64).bfloat16(), requires_grad=False)
    x = torch.randn(2, 3, 128, generator=torch.Generator().manual_seed(2))
    kind, group = module.input_codes()
    flat = x.reshape(6, 128)
    if group:
        flat = (flat.reshape(-1, group) @ regular_hadamard(group, "cpu")).reshape(6, 128)
    lim = 127.0 if kind == "int8" else 448.0
    scale = flat.abs().amax(-1) / lim
    codes = (flat / scale[:, None]).clamp(-lim, lim)
    codes = codes.round().to(torch.int8) if kind == "int8" else codes.to(torch.float8_e4m3fn)
    r = QuantizedRows(codes, scale, group, (2, 3, 128), torch.float16)
    # the values that the codes stand for, in 64 bits
    value = codes.double() * scale.double()[:, None]
    if group:
        value = (value.reshape(-1, group) @ regular_hadamard(group, "cpu").double().T).reshape(6, 128)
    assert (r.dequantize().double() - value.reshape(2, 3, 128)).abs().max() <= 2.0 ** -11 * value.abs().max() + 2.0 ** -20
    with pytest.warns(UserWarning, match="switches to dequantize"):
        got = module.forward_codes(r, activation)
    assert not module._ps_native and module.input_codes() is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        again = module.forward_codes(r, activation)
        want = module(r.dequantize()) if activation is None else module.forward_act(r.dequantize(), activation)
    assert got.dtype is (torch.float16 if follow else torch.bfloat16) and got.shape == (2, 3, 32 if activation == "silu_gate" else 64)
    assert torch.equal(got, again) and torch.equal(got, want.to(got.dtype))


def test_out_of_memory_is_not_a_native_failure(monkeypatch):
    from powershard_amd import quant_linear
    module = layer("int8", opts={"convrot": False})
    module.qbytes = torch.nn.Parameter(torch.zeros(module._ps_qplan.total, dtype=torch.uint8), requires_grad=False)

    def full(*args):
        raise torch.cuda.OutOfMemoryError("full")
    monkeypatch.setattr(quant_linear, "gemm_codes", full)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        module.forward_codes(rows())
    assert module._ps_native


def test_the_module_call_takes_codes_and_runs_its_hooks():
    """norm.linear calls the module: hooks (a sharded layer's among them) run around forward_codes, and a replaced
    forward is given rows, not codes."""
    from powershard_amd.norm import linear, rows_for
    module = layer("int8", opts={"convrot": False})
    weight = quantized_from_float(torch.randn(64, 128), module._ps_qplan.fmt, convrot=False)
    module.qbytes = torch.nn.Parameter(pack(weight, module._ps_qplan, "cpu"), requires_grad=False)
    module.bias = None
    seen = []
    module.register_forward_pre_hook(lambda m, args: seen.append(type(args[0])))
    module.register_forward_hook(lambda m, args, out: seen.append(out.shape))
    with pytest.warns(UserWarning, match="switches to dequantize"):
        linear(module, rows())
    assert seen == [QuantizedRows, (2, 3, 64)]
    module._ps_native = True
    assert rows_for([module]) == ("int8", 0)
    module.forward = lambda x: x
    assert rows_for([module]) is None
