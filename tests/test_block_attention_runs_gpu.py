"""paged_prompt_attention and paged_tree_attention where sequences are split over their length (the key tiles cut into runs, their
parts joined by a second kernel).  Each call's split is asked for, so that these cases stay what they are.  Tolerances as in
test_block_attention_gpu."""
import pytest

from powershard_amd import _native
from test_block_attention_gpu import check_prompts, prompts
from test_paged_attention_gpu import TYPES

pytestmark = pytest.mark.gpu

KIND = {"none": _native.CODES_NONE, "int8": _native.CODES_I8, "fp8": _native.CODES_E4M3}


def split(codes, T, B, N, Hq, Hk, D, window=0, sinks=0, max_len=0):
    return _native.lib().psq_paged_block_workspace_bytes(KIND[codes], T, B, N, Hq, Hk, D, window, sinks, max_len) > 0


def table_holds(pools):
    return pools[2].shape[1] * pools[0].shape[2]


@pytest.mark.parametrize("codes,dtype", TYPES)
@pytest.mark.parametrize("new", [[0, 0, 1, 0, 0], [1, 0, 0, 0, 0], [0, 2, 0, 0, 1, 0, 0]])
def test_fewer_rows_than_sequences(gpu, codes, dtype, new):
    shapes = [(n, 3000 + 171 * b) for b, n in enumerate(new)]
    q, pools, starts = prompts(shapes, 10, 2, 128, 64, codes, dtype, gpu, seed=12)
    assert split(codes, len(q), len(new), 0, 10, 2, 128, max_len=table_holds(pools))
    check_prompts(shapes, q, pools, starts)
