"""Edges of the rotary, cache-append and cache-attention calls, by the forms and bounds of test_attention_gpu.py."""
import pytest

from test_attention_gpu import BF16, FP16, Case, _check_append, _check_attention, _qkv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,page,dtype", [(128, 16, BF16), (64, 64, FP16), (256, 32, BF16)])
@pytest.mark.parametrize("lens,new,room", [([130], [4], 128), ([66, 20, 70], [3, 2, 1], 64), ([300, 90], [200, 9], 128), ([150], [149], 64),
                                           ([20_000, 9], [45, 3], 19_968)])
def test_lengths_past_the_block_table_keep_their_positions(cuda_device, lens, new, room, dim, page, dtype):
    """Several new tokens, some of them behind the end of the table, which has room for `room`: every row sees the tokens up to
    its own position that are in the table.  The last case goes by the list of units, the others by clusters; all but its last
    pages are not there, so that a few tokens weigh."""
    case = Case(lens, new, kv=2, group=3, dim=dim, page=page, dtype=dtype)
    case.block_table = case.block_table[:, : room // page]
    if room > 10_000:
        case.block_table[0, : room // page - 128 // page] = -1
    q, k, v = _qkv(case, extra=1)
    rotated = _check_append(case, q, k, v)
    _check_attention(case, rotated)
