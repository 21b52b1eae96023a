"""GPU: arguments and values at the ends of what the paged cache's entry points take, against the 64-bit oracle."""
import pytest
import torch

from tests.paged_util import make, to_gpu
from tests.test_paged_gpu import check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window", [None, 1, 40, 2**31 - 1])
@pytest.mark.parametrize("sinks", [2**31 - 1, 2**31 - 16, 2**40])
@pytest.mark.parametrize("lens", [[180], [900, 0, 31], [600 + 7 * i for i in range(20)], [3 * i for i in range(160)]])
def test_sinks_that_cover_everything(lens, sinks, window, e4m3):
    """Every slot is visible then: parts of rows, one list of all tiles (of more than 16 sequences, too), a part a row."""
    import flex_block_attn_b200 as fba

    pools, table = make(lens, 8, 16, e4m3, seed=len(lens))
    q, n = queries(len(lens), 8, 3), torch.tensor(lens, dtype=torch.int32).cuda()
    o, lse = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), n, window, sinks, need_lse=True)
    check(q, pools, table, lens, o, lse)
