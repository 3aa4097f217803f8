"""What the accuracy limits of the chunked delta rule and of the grouped experts can see, without a GPU: 64-bit restatements
with operands cut to fewer parts than the kernels use are beyond them."""
import pytest
import torch

import layer_oracle as lo

PRODUCTS = ("kk", "qk", "k", "s", "t", "x", "q", "qs", "p", "u", "kt", "w")


def normal(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(shape, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_chunk_limit_sees_any_operand_short_of_a_part(dtype):
    d = lo.remembering(normal(1), 1, 333, 1, 2, 64, 64, dtype)
    out, _, state, _, _ = lo.delta(**d)

    def worst(parts):
        o, s = lo.delta_chunks(**d, parts=parts)
        return max(lo.apart(o, out), lo.apart(s, state))

    assert worst({}) < lo.CHUNK_LIMIT / 20
    assert worst({name: 2 for name in PRODUCTS}) > 5 * lo.CHUNK_LIMIT
    assert worst({name: 1 for name in PRODUCTS}) > 1000 * lo.CHUNK_LIMIT
    # a bf16 q or k is one exact part
    for name in PRODUCTS if dtype is torch.float32 else [p for p in PRODUCTS if p not in ("kk", "qk", "k", "q", "kt")]:
        assert worst({name: 2}) > 1.2 * lo.CHUNK_LIMIT, name


def test_the_expert_limit_sees_a_missing_part():
    r = normal(2)
    x, e, hidden, ffn = r(40, 1056), 3, 1056, 352
    q = [(torch.randint(-128, 128, (e, rows, cols), dtype=torch.int8, generator=torch.Generator().manual_seed(rows)),
          (0.5 + r(e, rows, cols // 32).abs()) / (73 * cols ** 0.5)) for rows, cols in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    ids, w = torch.arange(80, dtype=torch.int32).view(40, 2) % e, r(40, 2)
    want = lo.moe(x, ids, w, *q)[0]
    assert lo.apart(lo.moe(x.half().float(), ids, w, *q)[0], want) > 30 * lo.moe_limit(hidden, ffn)
