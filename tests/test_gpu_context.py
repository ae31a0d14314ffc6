"""Contexts as a program makes and drops them beside running work."""
import pytest
import torch

from paged_infer_b200 import api

pytestmark = pytest.mark.gpu


def draw(ctx, x):
    f, i = torch.ones(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.full_like(i, -9)
    return lambda: api.sample(ctx, x, f, i, f, f, f * 0, ids), ids


def test_contexts_come_and_go_beside_running_work():
    """Neither creating nor destroying a context on a caller's stream waits for what runs on other streams."""
    x = torch.tensor([[0.0, 2.0, 1.0]], device="cuda")
    side, mine = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(mine):
        warm = api.Context(0, stream=mine.cuda_stream)
        run, ids = draw(warm, x)
        run()                                            # kernels are loaded at their first launch
        torch.cuda.synchronize()
        done = torch.cuda.Event()
        with torch.cuda.stream(side):
            torch.cuda._sleep(600_000_000)               # about 0.3 s
            done.record()
        for _ in range(3):
            c = api.Context(0, stream=mine.cuda_stream)
            run, ids = draw(c, x)
            run()
            c.close()
        assert not done.query()
        done.synchronize()
    assert ids.item() == 1                               # min_p = 1 keeps the largest alone


def test_many_contexts_at_once():
    """More contexts than error records that a device's contexts share, twice; each of them works and reports no error."""
    x = torch.tensor([[0.0, 2.0, 1.0]], device="cuda")
    for _ in range(2):
        contexts = [api.Context(0, stream=1) for _ in range(300)]
        for c in contexts[::7]:
            run, ids = draw(c, x)
            run()
            c.synchronize()
            assert ids.item() == 1
        for c in contexts:
            c.close()
