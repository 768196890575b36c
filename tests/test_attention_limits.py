"""Limits of the attention entry points, checked where the value is used: nothing is queued for what is refused."""
import pytest

from test_attention_api import FIELDS, refused


def with_field(name, at, value):
    packed, fields = FIELDS[name]
    fields = list(fields)
    fields[at] = value
    return refused(f"vesper_{name}_device", packed.pack(packed.size, *fields))


@pytest.mark.parametrize("name,at", [("prompt_attention", 8), ("shared_prefix_attention", 5)])
@pytest.mark.parametrize("scale", [1e39, 1e300, 3e38])
def test_scale_is_finite_in_the_kernels_32_bits(name, at, scale):
    """The kernels use scale * log2(e) in 32 bits: infinite there, a score of zero would become NaN."""
    assert "scale" in with_field(name, at, scale)


@pytest.mark.parametrize("eps", [1e39, 1e300])
def test_eps_is_finite_in_32_bits(eps):
    assert "eps" in with_field("norm_rotate", 7, eps)


@pytest.mark.parametrize("at", [1, 2, 3])
def test_counts_leave_room_for_a_tile_below_2_to_the_31(at):
    """Rows, keys and requests are numbered in 32 bits and counted in whole tiles of 128 (two of them a block)."""
    for n in ((1 << 31) - 1, (1 << 31) - 256):
        assert "2^31" in with_field("prompt_attention", at, n)
