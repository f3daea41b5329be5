"""Edges of the paged key / value cache's operators: what a row's company in the batch may change, numbers at the ends of
their formats, infinities and NaN in every place, long pieces, shared pages in odd places, tables of 2^31 entries."""
import math

import pytest
import torch

from tests import paged_reference as R
from tests.test_gpu_paged import DTYPES, check_attend, fill, make

pytestmark = pytest.mark.gpu
LN2 = 0.6931471824645996  # in fp32; times log2(e) in fp32 this is exactly 1, so scores are powers of two


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability(0)[0] != 10:
        pytest.fail("GPU tests need an sm_100 device")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 16, 40])
def test_scores_of_2_to_the_29(tokens, dtype):
    """Scores near the end of what 16-bit queries and keys give, where fp32 counts in steps of 32: the best key is further
    from the next than those steps, so it takes everything."""
    past, dim, heads = 300, 128, 4
    c, g = make(1, 1, dim, dtype, 32, [past + tokens], seed=11)
    keys, values = fill(c, [past + tokens], g)
    keys = (torch.rand(past + tokens, dim, generator=g) * 4096 - 2048).to(dtype)
    pos = torch.arange(past + tokens)
    c.data[0, 0][c.table.cpu()[0].long()[pos // 32].cuda(), 0, (pos % 32).cuda()] = keys.cuda()
    q = (torch.rand(1, tokens, heads, dim, generator=g) * 4096 - 2048).to(dtype)
    s = torch.einsum("thd,jd->thj", q[0].double(), keys.double()) * 8
    s = s.masked_fill(pos[None, None] > past + torch.arange(tokens)[:, None, None], -math.inf)
    top = s.topk(2, dim=-1)
    out = c.attend(0, q.cuda(), torch.tensor([past], device="cuda"), scale=8.0)[0].cpu()
    # a product's 128 terms of up to 2^25 are summed with steps of at most 2^9 each (2^32 in fp32, cut off): 2^16 in all
    clear = top.values[..., 0] - top.values[..., 1] > 2.0 ** 17
    assert clear.double().mean() > 0.9
    assert torch.equal(out[clear], values[0][0][top.indices[..., 0]][clear])
    assert c.status() == 0
