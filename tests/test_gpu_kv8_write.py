"""The write of the 8-bit cache where quotients by reciprocal and remainder could go wrong."""
import numpy as np
import pytest
import torch

from paged_infer_b200 import api
from test_gpu_kv8 import check_write, new_cache, rows_plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = api.Context(0, stream=1)
    yield c
    c.close()


def pairs(exponent):
    """(value, scale) whose quotient lies next to 2^-10 (1 + 2^-24), halfway between two f32, and 2^-10 is halfway between two e4m3 codes: S of 24 bits and X
    with X 2^25 - S (2^24 + 1) = k, a small number."""
    m = 2 ** 24 + 1
    inverse = pow(m, -1, 2 ** 25)
    for k in [*range(-200, 0), *range(1, 200)]:
        s = -k * inverse % 2 ** 25
        if 2 ** 23 <= s < 2 ** 24:
            yield np.ldexp(np.float32((s * m + k) >> 25), exponent - 32), np.ldexp(np.float32(s), exponent - 23)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("exponent", [-99, -98, -97, -95, -80, -66, -60, 0, 90])
def test_codes_of_quotients_next_to_a_border(ctx, kind, exponent):
    """Appended to a block that has the scale already; the codes are those of the rounded quotient."""
    x, s = (np.array(v, np.float32) for v in zip(*pairs(exponent)))
    n, block, dim = len(x), 16, 64
    cache = new_cache(ctx, kind, 1, n, 1, block, dim)
    cache.scales[0, :, 0] = torch.tensor(s, device="cuda")[:, None]
    k = torch.zeros(n, 1, dim, device="cuda")
    k[:, 0, 3], k[:, 0, 7] = torch.tensor(x, device="cuda"), torch.tensor(-x, device="cuda")
    slots = [b * block + 1 for b in range(n)]
    assert n > 20
    check_write(ctx, cache, kind, rows_plan(ctx, block, slots), k, -k, 0, slots, block)
