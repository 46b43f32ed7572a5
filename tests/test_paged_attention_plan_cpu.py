"""Which calls of paged_attention carry parts from one launch to a second, asked for without a device (the
plan then counts the 256 CUs of an MI355X)."""
import pytest

from powershard_amd import _native

I8, NONE = _native.CODES_I8, _native.CODES_NONE


@pytest.mark.parametrize("args,own", [
    ((I8, 1, 8, 1, 128, 30000), 1),        # one unit in 235 parts
    ((I8, 8, 16, 1, 256, 6000), 1),        # 47 parts of 16 x 256
    ((I8, 1, 40, 8, 128, 131071), 1),
    ((I8, 1, 40, 8, 128, 2000), 0),        # few parts: joined inside
    ((NONE, 128, 64, 8, 128, 8192), 0),    # many units
    ((I8, 1, 8, 1, 128, 100), 0),          # nothing to split
    ((I8, 1, 8, 1, 128, 0), 0), ((I8, 0, 8, 1, 128, 30000), 0), ((I8, 1, 8, 3, 128, 30000), 0), ((I8, 1, 8, 0, 128, 30000), 0),
])
def test_calls_of_two_launches(args, own):
    assert _native.lib().psq_paged_attention_own_workspace(*args) == own
    if own:
        assert _native.lib().psq_paged_attention_workspace_bytes(*args) > 0
