"""Attention over the 8-bit cache where its parts meet: waits that run out, dispatch of large batches, scales far apart, both planes."""
import numpy as np
import pytest
import torch

from paged_infer_b200 import _lib, api
from test_gpu_kv8 import attention_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = api.Context(0, stream=1)
    yield c
    c.close()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,contexts,news", [("bf16", 8, 2, 64, [300, 200], [130, 1]), ("f32", 4, 2, 128, [400], [300]), ("bf16", 8, 1, 128, [3000], [20])])
def test_a_wait_that_runs_out_is_reported_and_leaves_nan(ctx, dtype, heads, kv_heads, dim, contexts, news):
    """With a limit of one clock no warp waits for another: portions give up, say so, and the context works on; single tokens beside
    them have nothing to wait for.  The last case: a cluster shares the positions."""
    q, out, cache, plan, _ = attention_case(ctx, "int8", dtype, 16, heads, kv_heads, dim, contexts, news, seed=3, pad=2)
    a, again = api.PagedAttention8(cache.layout, heads), torch.full_like(out, 7.0)
    ctx.synchronize()
    ctx.set_option(_lib.PI_OPT_KV8_WAIT_LIMIT, 1)
    a.run_device(q, again, cache, plan, layer=1, max_seq_rows=max(news), max_context=max(contexts))
    ctx.set_option(_lib.PI_OPT_KV8_WAIT_LIMIT, 0)
    with pytest.raises(api.PiError) as err:
        ctx.synchronize()
    assert err.value.status == _lib.PI_ERR_TIMEOUT
    rows = sum(news)
    assert torch.isnan(again[: news[0]]).all() and torch.equal(again[news[0]: rows], out[news[0]: rows]) and (again[rows:] == 7.0).all()
    ctx.synchronize()                                    # reported once
    a.run_device(q, again, cache, plan, layer=1, max_seq_rows=max(news), max_context=max(contexts))
    ctx.synchronize()
    assert torch.equal(again, out)
    with pytest.raises(api.PiError):
        ctx.set_option(_lib.PI_OPT_KV8_WAIT_LIMIT, -1)
