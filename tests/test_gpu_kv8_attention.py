"""Attention over the 8-bit cache where its parts meet: waits that run out, dispatch of large batches, scales far apart, both planes."""
import math

import numpy as np
import pytest
import torch

from kv8_helpers import TORCH, TYPES, attention_reference, attention_tolerance, pitch_of
from kv8_planes import plane_case, plane_reference, plane_tolerance
from paged_infer_b200 import _lib, api
from test_gpu_kv8 import attention_case, i32, new_cache

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


@pytest.mark.parametrize("heads,kv_heads,dim,news", [(128, 1, 64, [40000, 30000]), (64, 1, 64, [100000, 1, 39999]), (200, 1, 24, [6000])])
def test_attention_of_more_tiles_than_a_grid_has_rows(ctx, heads, kv_heads, dim, news):
    """Groups so wide that a tile holds one or two rows, in batches of more than 65535 tiles; and more tiles of columns than that in one
    sequence.  Rows here and there against the reference, all of them against the call that is told to expect few."""
    block, window = 16, 20
    contexts = np.array(news)
    rng = np.random.default_rng(heads)
    after = -(-contexts // block)
    wide, blocks = int(after.max()), int(after.sum())
    tables, at = np.full((len(news), wide), -1, np.int32), 0
    for b, n in enumerate(after):
        tables[b, :n] = np.arange(at, at + n)
        at += n
    cu = np.concatenate([[0], np.cumsum(news)])
    rows, pos = int(cu[-1]), np.concatenate([np.arange(n) for n in news])
    cache = new_cache(ctx, "int8", 1, blocks, kv_heads, block, dim, seed=1)
    g = torch.Generator(device="cuda").manual_seed(heads)
    q = torch.randn(rows, heads, dim, generator=g, device="cuda", dtype=torch.bfloat16)
    plan = api.StepPlan(ctx, block, i32(tables), lens=i32(after), cu_rows=i32(cu), row_pos=i32(pos))
    a, out, again = api.PagedAttention8(cache.layout, heads), torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    a.run_device(q, out, cache, plan, window=window)
    ctx.synchronize()
    a.run_device(q, again, cache, plan, window=window, max_seq_rows=1)
    some = np.unique(np.concatenate([cu[:-1], cu[1:] - 1, rng.integers(0, rows, 40), [65535, 65536, rows - 2] if rows > 65536 else []]).astype(int))
    seq = np.searchsorted(cu, some, side="right") - 1
    codes, scales = cache.codes[0].view(torch.uint8).cpu().numpy(), cache.scales[0].cpu().numpy()
    sub = np.concatenate([[0], np.cumsum([(seq == b).sum() for b in range(len(news))])])
    want, most, mass = attention_reference(q[some].float().cpu().numpy(), codes, scales, tables=tables, lens=after, cu=sub, pos=pos[some], block=block, kind="int8", window=window)
    tolerance = attention_tolerance(want, most, mass, dim, "bf16")
    for o in (out, again):
        assert (np.abs(o[some].float().cpu().numpy() - want) <= tolerance).all()
    # a rounding of the result each, and 2^-9 of the largest value: 2^-10 of the weights and, scores being products of 64 channels at most
    # (the sum of their magnitudes below 25), 4 x 25 x 78 x 2^-23 from those
    off = (out.float() - again.float()).abs() - 2.0 ** -7 * torch.maximum(out.float().abs(), again.float().abs())
    assert off.max() <= 2 * 2.0 ** -9 * 100 * 0.025      # largest |code| x largest scale of the cache


def test_a_refused_call_leaves_the_results_alone(ctx):
    q, out, cache, plan, given = attention_case(ctx, "int8", "bf16", 16, 8, 2, 64, [300, 40], [130, 1], seed=3)
    n = 65536
    many = api.StepPlan(ctx, 16, i32(np.full((n, 1), -1)), lens=i32(np.zeros(n)), cu_rows=i32(np.minimum(np.arange(n + 1), 131)), row_pos=plan.row_pos)
    before = out.clone()
    with pytest.raises(api.PiError, match="65535"):
        api.PagedAttention8(cache.layout, 8).run_device(q, out, cache, many, layer=1)
    ctx.synchronize()
    assert torch.equal(out, before)


def weighted_reference(q, codes, scales, table, pos, block, kind, window=0):
    """(out, sum of weight x largest |v| of the token, largest sum of |q||k| scale) of one sequence in 64 bits; codes as values of one layer."""
    rows, heads, dim = q.shape
    group = heads // codes.shape[1]
    n = int(pos.max()) + 1
    t = np.arange(n)
    value = codes[table[t // block], :, :, t % block, :dim].astype(np.float64) * scales[table[t // block]].astype(np.float64)[..., None]   # [n][kv_heads][2][dim]
    out, weighed, mass = np.zeros((rows, heads, dim)), np.zeros((rows, heads)), np.zeros((rows, heads))
    for h in range(heads):
        k, v = value[:, h // group, 0], value[:, h // group, 1]
        s = q[:, h].astype(np.float64) @ k.T * dim ** -0.5
        unseen = (t[None] > pos[:, None]) | ((t[None] <= pos[:, None] - window) if window else False)
        s[unseen] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h], weighed[:, h] = w @ v, w @ np.abs(v).max(1)
        mass[:, h] = np.where(unseen, 0, np.abs(q[:, h]).astype(np.float64) @ np.abs(k).T * dim ** -0.5).max(1)
    return out, weighed, mass


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,news,context", [(64, 200, 300), (128, 200, 300), (64, 1, 300), (128, 40, 2500)])
@pytest.mark.parametrize("ratio", [24, 40, -30])
def test_a_large_scale_of_next_to_no_weight(ctx, kind, dtype, dim, news, context, ratio):
    """Blocks whose V scale is 2^ratio of their neighbours', seen with a weight so small that they add little: every result keeps its
    precision relative to what it is made of, sum of weight x |v|, not to the largest |v| in sight.  The last case but one: single
    tokens; the last: a cluster shares the positions."""
    rng = np.random.default_rng(ratio + 50 + dim)
    block, heads, kv_heads = 16, 4, 2
    blocks = -(-context // block)
    shape = (2, blocks, kv_heads, 2, block, dim)
    values = np.clip(np.round(rng.standard_normal(shape) * 30), -60, 60).astype(np.float32)
    if kind == "e4m3":
        values = torch.tensor(values).to(torch.float8_e4m3fn).float().numpy()
    scales = (np.exp(rng.standard_normal(shape[:4]) * 0.2) / 40).astype(np.float32)
    q = rng.standard_normal((news, heads, dim)).astype(np.float32)
    q[..., 0] = 8.0
    values[..., 0, :, 0] = 0                              # K's first channel: nothing, but in the blocks in question
    odd = np.arange(2, blocks, 5)
    far = 2.0 ** abs(ratio)
    # weights of about exp(-ratio ln 2 - 10) at 2^ratio, of 1 at 2^-ratio (the others then lie that far below)
    low = (max(ratio, 0) * math.log(2) + 10) * dim ** 0.5 / 8.0 / 60 if ratio > 0 else 0.0
    if ratio > 0:
        values[1][odd, :, 0] = 0
        values[1][odd, :, 0, :, 0] = -60
        scales[1][odd, :, 0] = low
        scales[1][odd, :, 1] *= far
    else:
        values[1][odd, :, 0] = 0
        values[1][odd, :, 0, :, 0] = 60
        scales[1][odd, :, 0] = (abs(ratio) * math.log(2) + 10) * dim ** 0.5 / 8.0 / 60
        scales[1][odd, :, 1] /= far
    table = rng.permutation(blocks)
    codes = torch.tensor(values, device="cuda").to(TORCH[kind])
    layout = api.KvLayout(2, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=codes, scales=torch.tensor(scales, device="cuda"))
    qt = torch.tensor(q, device="cuda").to(TYPES[dtype])
    out = torch.full_like(qt, 7.0)
    pos = np.arange(context - news, context)
    plan = api.StepPlan(ctx, block, i32(table[None]), lens=i32([blocks]), cu_rows=i32([0, news]), row_pos=i32(pos))
    api.PagedAttention8(layout, heads).run_device(qt, out, cache, plan, layer=1)
    want, weighed, mass = weighted_reference(qt.float().cpu().numpy(), values[1], scales[1], table, pos, block, kind)
    tolerance = attention_tolerance(want, weighed, mass, dim, dtype) + (2.0 ** -25 if dtype == "f16" else 0)   # half of f16's smallest step
    off = np.abs(out.float().cpu().numpy() - want) - tolerance
    assert not (off > 0).any(), off.max()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,news", [(64, 1), (128, 1), (96, 3), (256, 2), (64, 60), (128, 60)])
def test_an_outlier_channel_of_keys_beside_small_codes(ctx, dtype, dim, news):
    """A K channel that sets the scale and in which the query is zero: a token's other codes are zero but for two of them, and scores keep
    their precision relative to those, however large the query is beside the others."""
    rng = np.random.default_rng(dim + news)
    block, heads, kv_heads, context = 16, 8, 2, 70
    blocks = -(-context // block)
    shape = (2, blocks, kv_heads, 2, block, pitch_of(dim))
    values = np.clip(np.round(rng.standard_normal(shape) * 35), -127, 127).astype(np.float32)
    values[..., dim:] = 0
    values[..., 0, :, :] = 0
    np.put_along_axis(values[..., 0, :, :], rng.integers(1, dim, shape[:3] + (block, 2)), 1.0, -1)
    values[..., 0, :, 0] = 127
    scales = np.full(shape[:4], 1 / 40, np.float32)
    scales[..., 0] = 3 * dim ** 0.5                       # scores of 1.5 to 6
    q = torch.tensor(rng.uniform(0.5, 1.0, (news, heads, dim)), device="cuda").to(TYPES[dtype])
    q[..., 0] = 0
    table, pos = rng.permutation(blocks), np.arange(context - news, context)
    layout = api.KvLayout(2, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=torch.tensor(values, device="cuda").to(torch.int8), scales=torch.tensor(scales, device="cuda"))
    plan = api.StepPlan(ctx, block, i32(table[None]), lens=i32([blocks]), cu_rows=i32([0, news]), row_pos=i32(pos))
    out = torch.full_like(q, 7.0)
    api.PagedAttention8(layout, heads).run_device(q, out, cache, plan, layer=1)
    want, weighed, mass = weighted_reference(q.float().cpu().numpy(), values[1], scales[1], table, pos, block, "int8")
    off = np.abs(out.float().cpu().numpy() - want) - attention_tolerance(want, weighed, mass, dim, dtype)
    assert not (off > 0).any(), (off.max(), (off > 0).sum())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("which", ["query", "weight"])
@pytest.mark.parametrize("dim,heads,kv_heads,context,news", [(64, 8, 2, 40, 1), (128, 8, 2, 41, 2), (96, 4, 2, 40, 1), (256, 16, 1, 40, 1), (24, 4, 2, 33, 3), (64, 8, 1, 3000, 1), (128, 4, 1, 3000, 1),
                                                               (64, 8, 2, 300, 200), (128, 8, 2, 300, 200), (64, 8, 1, 3000, 20), (128, 8, 1, 3000, 20), (96, 8, 2, 90, 40)])
def test_f32_rows_have_both_planes(ctx, kind, which, dim, heads, kv_heads, context, news):
    """Single tokens and portions, each alone and with the positions shared by a cluster."""
    block = 16
    q, values, k_scale, v_scale = plane_case(which, dim, context, news, heads, kv_heads)
    blocks = -(-context // block)
    codes = np.zeros((1, blocks * block, kv_heads, 2, pitch_of(dim)), np.float32)
    codes[0, :context, ..., :dim] = values
    codes = codes.reshape(1, blocks, block, kv_heads, 2, -1).transpose(0, 1, 3, 4, 2, 5)
    scales = np.empty((1, blocks, kv_heads, 2), np.float32)
    scales[..., 0], scales[..., 1] = k_scale, v_scale
    layout = api.KvLayout(1, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=torch.tensor(codes, device="cuda").to(TORCH[kind]).contiguous(), scales=torch.tensor(scales, device="cuda"))
    pos = np.arange(context - news, context)
    plan = api.StepPlan(ctx, block, i32(np.arange(blocks)[None]), lens=i32([blocks]), cu_rows=i32([0, news]), row_pos=i32(pos))
    qt = torch.tensor(q, device="cuda")
    out = torch.full_like(qt, 7.0)
    api.PagedAttention8(layout, heads).run_device(qt, out, cache, plan)
    want, weighed = plane_reference(q, values, k_scale, v_scale, pos)
    off = np.abs(out.cpu().numpy() - want) - plane_tolerance(want, weighed)
    assert not (off > 0).any(), off.max()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,dim,contexts,news", [(4, 1, 256, [2526, 5000, 7021], [1, 1, 1]), (2, 1, 256, [366, 400, 622], [1, 2, 1]), (4, 2, 128, [339, 429], [1, 1]), (8, 2, 64, [700], [90]), (4, 2, 128, [1500], [90])])
def test_f32_rows_against_64_bits_as_a_whole(ctx, kind, heads, kv_heads, dim, contexts, news):
    """Results are sums of values of random signs, so that their error over their norm is the root mean square of the weights' relative
    errors, below the sum of what those can be for scores of a few units: the exponential 2^-22, its argument (below 8) 2^-22 ln 2, the score's
    factor and the queries' planes 2^-23 each; sums of products add nothing to speak of.  Together 2^-20.5."""
    rng = np.random.default_rng(dim + len(news))
    block, B = 16, len(news)
    after = [-(-c // block) for c in contexts]
    blocks, wide = sum(after), max(after)
    shape = (1, blocks, kv_heads, 2, block, dim)
    values = torch.tensor(np.clip(np.round(rng.standard_normal(shape) * 35), -127, 127), device="cuda", dtype=torch.float32)
    codes = values.to(torch.int8) if kind == "int8" else (values * 3).to(torch.float8_e4m3fn)
    scales = torch.tensor(np.exp(rng.standard_normal(shape[:4]) * 0.2) / (35 if kind == "int8" else 105), device="cuda", dtype=torch.float32)
    tables, at = np.full((B, wide), -1), 0
    for b, n in enumerate(after):
        tables[b, :n] = np.arange(at, at + n)
        at += n
    layout = api.KvLayout(1, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=codes, scales=scales)
    cu = np.concatenate([[0], np.cumsum(news)])
    pos = np.concatenate([np.arange(c - n, c) for c, n in zip(contexts, news)])
    q = torch.tensor(rng.standard_normal((int(cu[-1]), heads, dim)), dtype=torch.float32, device="cuda")
    plan = api.StepPlan(ctx, block, i32(tables), lens=i32(after), cu_rows=i32(cu), row_pos=i32(pos))
    out = torch.full_like(q, 7.0)
    api.PagedAttention8(layout, heads).run_device(q, out, cache, plan, max_seq_rows=max(news), max_context=max(contexts))
    values, sc, want = codes.float().cpu().numpy()[0], scales.cpu().numpy()[0], np.zeros(q.shape)
    for b in range(B):
        r = slice(cu[b], cu[b + 1])
        want[r] = weighted_reference(q[r].cpu().numpy(), values, sc, tables[b], pos[r], block, kind)[0]
    error = np.linalg.norm(out.cpu().numpy() - want) / np.linalg.norm(want)
    assert error <= 2.0 ** -20.5, error


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,news", [(64, 1), (128, 2), (96, 1), (64, 60), (128, 60)])
def test_an_outlier_channel_of_the_query(ctx, kind, dtype, dim, news):
    """A query channel 2^20 times the others, where the keys are zero: scores are made of the others alone and keep their precision."""
    rng = np.random.default_rng(dim + news)
    block, heads, kv_heads, context = 16, 8, 2, 90
    blocks = -(-context // block)
    shape = (1, blocks, kv_heads, 2, block, pitch_of(dim))
    values = np.clip(np.round(rng.standard_normal(shape) * 35), -120, 120).astype(np.float32)
    if kind == "e4m3":
        values = torch.tensor(values).to(torch.float8_e4m3fn).float().numpy()
    values[..., dim:] = 0
    values[..., 0, :, 5] = 0
    q = rng.uniform(0.5, 1.0, (news, heads, dim)) * rng.choice([-1, 1], (news, heads, dim)) * 2.0 ** -5
    q[..., 5] = 2.0 ** 15
    q = torch.tensor(q, device="cuda").to(TYPES[dtype])
    scales = np.full(shape[:4], 1 / 40, np.float32)
    scales[..., 0] = 2.0 ** 5 / 30                       # scores of a few units
    table, pos = rng.permutation(blocks), np.arange(context - news, context)
    layout = api.KvLayout(1, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=torch.tensor(values, device="cuda").to(TORCH[kind]), scales=torch.tensor(scales, device="cuda"))
    plan = api.StepPlan(ctx, block, i32(table[None]), lens=i32([blocks]), cu_rows=i32([0, news]), row_pos=i32(pos))
    out = torch.full_like(q, 7.0)
    api.PagedAttention8(layout, heads).run_device(q, out, cache, plan)
    want, weighed, mass = weighted_reference(q.float().cpu().numpy(), values[0], scales[0], table, pos, block, kind)
    off = np.abs(out.float().cpu().numpy() - want) - attention_tolerance(want, weighed, mass, dim, dtype)
    assert not (off > 0).any(), (off.max(), (off > 0).sum())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,nats", [("f32", 10), ("bf16", 10), ("f16", 10), ("f32", 17), ("bf16", 20), ("f16", 20)])
@pytest.mark.parametrize("dim,news,context", [(64, 1, 65), (128, 2, 80), (96, 1, 70), (64, 60, 120), (128, 60, 120)])
def test_a_token_of_nearly_all_the_weight_and_no_value(ctx, kind, dtype, nats, dim, news, context):
    """A first token `nats` above the others whose values are zero: results are made of the others, whose weights keep their precision.  One
    channel makes the scores, whose sums are exact."""
    rng = np.random.default_rng(dim + news)
    block, heads, kv_heads = 16, 4, 2
    blocks = -(-context // block)
    values = np.zeros((1, blocks, kv_heads, 2, block, pitch_of(dim)), np.float32)
    values[..., 1, :, :dim] = np.clip(np.round(rng.standard_normal(values[..., 1, :, :dim].shape) * 35), -120, 120)
    values[..., 0, :, 0] = rng.integers(-7, 8, values[..., 0, :, 0].shape)
    values[0, 0, :, 0, 0, 0], values[0, 0, :, 1, 0] = 120, 0
    if kind == "e4m3":
        values = torch.tensor(values).to(torch.float8_e4m3fn).float().numpy()
    scales = np.full(values.shape[:4], 1 / 40, np.float32)
    scales[..., 0] = nats / 120 * dim ** 0.5
    q = np.zeros((news, heads, dim), np.float32)
    q[..., 0] = 1.0
    q = torch.tensor(q, device="cuda").to(TYPES[dtype])
    table = np.arange(blocks)
    pos = np.arange(context - news, context)
    layout = api.KvLayout(1, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=torch.tensor(values, device="cuda").to(TORCH[kind]), scales=torch.tensor(scales, device="cuda"))
    plan = api.StepPlan(ctx, block, i32(table[None]), lens=i32([blocks]), cu_rows=i32([0, news]), row_pos=i32(pos))
    out = torch.full_like(q, 7.0)
    api.PagedAttention8(layout, heads).run_device(q, out, cache, plan)
    want, weighed, mass = weighted_reference(q.float().cpu().numpy(), values[0], scales[0], table, pos, block, kind)
    tolerance = attention_tolerance(want, weighed, mass, 2, dtype) + (2.0 ** -25 if dtype == "f16" else 0)   # half of f16's smallest step
    off = np.abs(out.float().cpu().numpy() - want) - tolerance
    assert not (off > 0).any(), (off.max(), (off > 0).sum())
