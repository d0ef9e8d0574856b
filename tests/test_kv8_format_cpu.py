"""What include/dg_attn.h says of the 8-bit format and of sums of codes, at the block maxima where it is nearest to false."""
import pytest
import torch

import kv8_ref as ref


def block(top, rest):
    """One block of one head: its largest magnitude and other numbers."""
    x = torch.zeros(128, 1, 256, dtype=torch.float64)
    x.view(-1)[0] = top
    x.view(-1)[1:1 + len(rest)] = rest
    return x.clone()


# from just above half of 448 (the smallest largest code) to 448 itself, and the same at other scales
@pytest.mark.parametrize("top", [224.0001, 225.0, 240.0, 255.0, 300.0, 448.0])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -20, 2.0 ** 30])
def test_bits_and_error_of_a_held_value(top, scale):
    g = torch.Generator().manual_seed(3)
    rest = top * scale * torch.exp2(-20 * torch.rand(32000, generator=g, dtype=torch.float64))
    x = block(top * scale, rest)
    off = (ref.code(x) - x).abs()
    large = x >= 2.0 ** -13.8 * top * scale
    assert (off[large] <= 2.0 ** -4 * x[large]).all()
    assert (off[~large] <= 2.0 ** -17.8 * top * scale).all()


def test_the_limits_are_near():
    """A block maximum of 225: neither four bits down to 2^-14 of it nor an error of 2^-19 of it below would be true."""
    x = block(225.0, torch.tensor([2.0 ** -6 * 0.94, 2.0 ** -9 * 1.49], dtype=torch.float64))
    off = (ref.code(x) - x).abs().view(-1)
    x = x.view(-1)
    assert x[1] > 2.0 ** -14 * 225 and off[1] > 2.0 ** -4 * x[1]
    assert off[2] > 2.0 ** -19 * 225


def test_a_query_element_is_two_codes():
    """bf16 numbers within 2^9.8 of the largest of their row are the sum of two codes at its scale; just outside, one is not."""
    def two(x):
        return ref.code(x) + ref_code_at(x - ref.code(x), x)

    def ref_code_at(r, x):
        # codes of what is left, at the first one's scale
        e = 2.0 ** ref.scale_exp(float(x.abs().max()))
        y = r / e
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step * e

    bits = torch.arange(128, dtype=torch.float64) / 128 + 1
    for top in (224.0 + 1, 255.0, 256.0, 448.0):
        rest = torch.cat([bits * 2.0 ** -x for x in range(-8, 12)])
        rest = rest[rest <= top]
        x = block(top, rest)
        near = x * 2.0 ** 9.8 >= top
        assert torch.equal(two(x)[near], x[near])
    x = block(225.0, 0.25 * bits * (1 - 2.0 ** -1))       # below a quarter: 2^-9.8 to 2^-10.8 of 225
    assert not torch.equal(two(x), x)
