"""GPU tests of attention over a paged cache at the ends of its range of values."""
import pytest
import torch

from tests.paged_cases import BF16_STEP

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["attention", "prefix"])
def test_large_values_in_every_part(kernels, form):
    """Keys that several CTAs share, a part of 10 blocks of 128 to each: nine of score 0 and a last one whose weights add up to
    some 2^24 times a block's of those, which is under what makes a part take another reference.  Values of 1.5 * 2^99, all alike:
    the result is that value, however many parts are added up.

    The weights are rounded to bf16 and divided by the sum of the unrounded ones: with all values alike that is off by half a step
    at most, and the result's rounding by none, since the value is a bf16 number and half a step down from it the next one is
    nearer by no more than that: two halves of a step, with 2^-16 for the sums' 32 bits."""
    Hq, Hk, D, page, parts = 2, 1, 64, 128, 60
    value = 1.5 * 2.0 ** 99
    keys = torch.zeros(2, Hk, page, D, dtype=torch.bfloat16, device="cuda")
    keys[1, ..., 0] = 17.75  # 64 of them: 2^23.75 in half a block
    values = torch.full_like(keys, value)
    table = torch.tensor(([0] * 9 + [1]) * parts, dtype=torch.int32, device="cuda")
    n = torch.tensor([parts * 10 * page], dtype=torch.int32, device="cuda")
    T = 40
    q = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    q, scale = q.view(T, -1), 0.6931471805599453  # scores count powers of two
    if form == "attention":
        cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
        out = kernels.paged_attention(q, keys, values, table[None], n, Hq, Hk, D, cu_tokens=cu, scale=scale)
    else:
        own, none = torch.zeros(T, 1, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
        out = kernels.shared_prefix_attention(q, keys, values, table, n, own, none, Hq, Hk, D, scale=scale)
    assert ((out.double() / value - 1).abs() <= 2 * BF16_STEP + 2.0 ** -16).all(), (out.float().min(), out.float().max())
