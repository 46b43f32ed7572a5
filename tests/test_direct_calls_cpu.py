"""The module of the decoder operators' direct calls (csrc/direct.cpp) on the CPU: it is the installed torch's,
and arguments that it does not take come back as None, without an error left behind."""
import pytest
import torch

from powershard_amd import _native


def test_belongs_to_this_torch():
    assert _native.direct().TORCH_VERSION == torch.__version__.split("+")[0]


@pytest.mark.parametrize("name,count", [("add_rms_norm", 7), ("kv_write", 8), ("kv_read", 7), ("paged_attention", 13)])
@pytest.mark.parametrize("value", [None, 0, "x", 1 << 70, torch.zeros(4, 32), torch.zeros(4, 32, dtype=torch.bfloat16),
                                   torch.zeros(4, 32, dtype=torch.bfloat16, device="meta")], ids=str)
def test_other_arguments_are_left_alone(name, count, value):
    call = getattr(_native.direct(), name)
    for n in (0, count - 1, count, count + 1):
        assert call(*[value] * n) is None


def test_a_foreign_module_is_not_used(monkeypatch, tmp_path):
    monkeypatch.setattr(_native, "_direct", None)
    monkeypatch.setattr(_native, "DIRECT_PATH", tmp_path / "psq_direct.so")
    with pytest.warns(UserWarning, match="is not used"):
        assert _native.direct() is False
    assert _native.direct() is False   # and is not looked for again


def test_bind_takes_a_dict():
    from powershard_amd._native import DIRECT_CALLS, SIGNATURES
    assert set(DIRECT_CALLS) <= set(SIGNATURES)


def test_belongs_to_this_python(monkeypatch):
    import sys
    assert _native.direct().PYTHON_VERSION == sys.hexversion >> 16
    monkeypatch.setattr(_native, "_direct", None)
    monkeypatch.setattr(_native.sys, "hexversion", sys.hexversion + (1 << 16))
    with pytest.warns(UserWarning, match="built for Python"):
        assert _native.direct() is False


@pytest.mark.parametrize("compiler", ["/no/such/compiler", "false"])
def test_the_library_builds_without_a_host_compiler(monkeypatch, tmp_path, compiler):
    """The module is optional: its build fails with a warning, and leaves none of an earlier build."""
    from powershard_amd import build_lib
    old = tmp_path / "psq_direct.so"
    old.write_bytes(b"of another build")
    monkeypatch.setattr(build_lib, "DIRECT", old)
    monkeypatch.setenv("CXX", compiler)
    with pytest.warns(UserWarning, match="was not built"):
        build_lib._build_direct()
    assert not old.exists()
