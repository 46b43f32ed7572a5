"""Which calls of paged_prompt_attention and paged_tree_attention split sequences over their length, asked for without a
device (the plan then counts the 256 CUs of an MI355X)."""
import pytest

from powershard_amd import _native


def workspace(codes, T, B, N=0, Hq=40, Hk=8, D=128, window=0, sinks=0, max_len=65537):
    return _native.lib().psq_paged_block_workspace_bytes(codes, T, B, N, Hq, Hk, D, window, sinks, max_len)


@pytest.mark.parametrize("codes", [_native.CODES_NONE, _native.CODES_I8, _native.CODES_E4M3])
@pytest.mark.parametrize("T,B", [(1, 1), (1, 2), (1, 16), (5, 16), (15, 16), (16, 16), (17, 16), (1, 128), (7, 128)])
def test_few_rows_on_long_texts_are_split(codes, T, B):
    """Also where fewer rows than sequences are new, so that some have none: down to one token in all."""
    assert workspace(codes, T, B) > 0
    assert T > B or workspace(codes, T, B) == workspace(codes, T, T)      # as those that have one by themselves
    assert workspace(codes, T, B, max_len=64) == 0                        # nothing to split
