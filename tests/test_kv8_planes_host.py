"""What the tests of f32 attention over the 8-bit cache can tell apart, without a GPU."""
import numpy as np
import pytest

from kv8_planes import plane_case, plane_reference, plane_tolerance


@pytest.mark.parametrize("which", ["query", "weight"])
@pytest.mark.parametrize("dim", [24, 64, 96, 128, 256])
def test_one_plane_is_told_from_two(which, dim):
    q, codes, k_scale, v_scale = plane_case(which, dim, 40, 3, 4, 2)
    pos = np.array([17, 38, 39])
    want, weighed = plane_reference(q, codes, k_scale, v_scale, pos)
    tolerance = plane_tolerance(want, weighed)
    two, one = (np.abs(plane_reference(q, codes, k_scale, v_scale, pos, planes)[0] - want) for planes in (2, 1))
    assert (two <= tolerance).all() and (one > 3 * tolerance).all()
