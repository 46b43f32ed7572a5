"""Sizes at which the attention of prompts and trees would count past 32 bits, asked for without a device."""
import pytest

from test_more_decoder_ops_cpu import ARG, SHAPE, prompt, tree

MOST = (1 << 30) - 1


@pytest.mark.parametrize("T,cols", [(MOST, MOST // 16), (MOST - 300, MOST // 16), (MOST, MOST // 16 - 1)])
def test_tokens_and_table_in_31_bits(T, cols):
    """A length that is past the table counts as the table's tokens, the rows and 64: that and a tile more have to fit."""
    too_many = T + 16 * cols > 0x7FFFFF00
    # (sizes are looked at in front of the rows' own pointers, whose absence ends the calls that fit)
    assert prompt(T=T, Hq=1, Hk=1, cols=cols, stride=cols, starts=None) == (SHAPE if too_many else ARG)
    assert tree(B=65535, N=64, Hq=1, Hk=1, cols=cols, stride=cols, parents=None) == ARG
