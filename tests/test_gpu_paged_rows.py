"""Rows of paged attention that see no key, and values that are not finite, at every head size and in every form of the work:
one part, parts joined by a second launch, parts joined by the wave that arrives last."""
import pytest
import torch

from common import TINY, QWEN3_NEXT, D128
from test_gpu_paged import BF16, F32, NAN, Batch, attend, contexts  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n,pos", [(TINY, 1, 40), (QWEN3_NEXT, 1, 3000), (D128, 4, 3000), (QWEN3_NEXT, 60, 40), (TINY, 60, 3000),
                                     (QWEN3_NEXT, 600, 900), (D128, 700, 300)], ids=str)
def test_rows_that_see_nothing_are_zero_whatever_their_gate(contexts, s, n, pos, dtype):  # noqa: F811
    """A sequence without pages and the tokens of others outside their table's positions, with gates of NaN and infinities as an
    idle place's rows may hold them: zero, and the other rows as the formula has them."""
    b = Batch(n, s, [pos, pos, pos, 5], n, 32, dtype)
    top = b.table.shape[1] * 32
    b.pos = [pos, pos, top, 5]
    b.table[1] = -1
    junk = torch.tensor([NAN, float("inf"), -float("inf"), NAN]).repeat(s.D // 4)
    b.qg[1:3, :, :, s.D:] = junk
    out = attend(contexts(s), b)
    assert (out[1:3] == 0).all()
    b.new[0] = b.new[3] = min(n, 50)  # (of the others, the first tokens)
    b.check(out)
    # before position 0: the first token of two, or none of one
    if 2 <= n <= 60:
        c = Batch(n, s, [0], n, 32, dtype)
        c.pos = [-1]
        c.qg[:, 0, :, s.D:] = junk
        out = attend(contexts(s), c)
        assert (out[0, 0] == 0).all()
        c.check(out)
