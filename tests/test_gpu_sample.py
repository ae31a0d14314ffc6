"""Sampling where the tokens that can be drawn span less or more than a float's range divides, and under flat weights."""
import numpy as np
import pytest
import torch

from paged_infer_b200 import api
from test_gpu_kv8 import check_sample

pytestmark = pytest.mark.gpu

KINDS = [(0, 0.9, 0), (0, 0.3, 0), (5, 1, 0), (700, 1, 0), (700, 0.8, 0), (0, 1, 0.2), (0, 0.9, 0.01), (1, 0.5, 0), (0, 1, 0)]   # top_k, top_p, min_p


@pytest.fixture(scope="module")
def ctx():
    c = api.Context(0, stream=1)
    yield c
    c.close()


@pytest.mark.parametrize("t", [np.finfo(np.float32).tiny, 5e-38, 9e-38, 1e-37, 1e-36, 1e-40, 1e-42, 1.4e-45])
def test_sample_at_temperatures_near_zero(ctx, t):
    """Rows whose largest logit is 0: one or many of it, the others a few temperatures below (subnormal numbers among them), far below, not there."""
    rng = np.random.default_rng(1)
    n, t = 3000, np.float32(t)
    x = np.zeros((6, n), np.float32)
    x[1:4] = -np.abs(rng.standard_normal((3, n))) * 8 * np.float64(t)
    x[1, 17] = x[2, [40, 1500, 2999]] = 0.0
    x[3] -= np.float32(3e-37)
    x[3, 1000] = -0.0
    x[4, 1:] = -rng.uniform(1, 9, n - 1)
    x[5, 3:] = -np.inf
    for k, p, m in KINDS:
        check_sample(ctx, torch.tensor(x, device="cuda"), t, k, p, m, rng.random(6).astype(np.float32))


@pytest.mark.parametrize("t", [1e37, 1e38, 3e38, np.inf])
def test_sample_of_logits_across_the_whole_range(ctx, t):
    """The interval of the logits is wider than the largest float."""
    rng = np.random.default_rng(2)
    x = rng.uniform(-3.4e38, 3.4e38, (3, 4000)).astype(np.float32)
    x[1, :1000] = np.finfo(np.float32).min
    x[2] = np.round(x[2] / 4e37) * np.float32(4e37)      # many equal ones
    for k, p, m in KINDS + [(2600, 1, 0), (3500, 0.999, 0)]:
        check_sample(ctx, torch.tensor(x, device="cuda"), t, k, p, m, rng.random(3).astype(np.float32))


@pytest.mark.parametrize("t", [1e6, np.inf])
def test_top_k_of_flat_weights(ctx, t):
    """Counting does not look at weights."""
    rng = np.random.default_rng(3)
    x = torch.tensor(rng.standard_normal((8, 5000)), dtype=torch.float32, device="cuda")
    x[1] = x[1].round()
    x[2, 100:] = -float("inf")
    x[3] = 0.25
    for k in (1, 2, 7, 40, 1000, 4999):
        check_sample(ctx, x, t, k, 1, 0, rng.random(8).astype(np.float32))
