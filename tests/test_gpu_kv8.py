"""The device-side step over an 8-bit KV cache on the GPU, each operator against a plain form in whole numbers or 64 bits, and the
four of them together, eager and replayed."""
import numpy as np
import pytest
import torch

from kv8_helpers import (TORCH, TYPES, attention_reference, attention_tolerance, pitch_of, plan_reference, sample_reference, write_reference)
from paged_infer_b200 import _lib, api

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = api.Context(0, stream=1)   # the legacy default stream, torch's own
    yield c
    c.close()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def refused(status=_lib.PI_ERR_INVALID_ARG):
    return pytest.raises(api.PiError, match=f"error {status}")


# ---- plan -------------------------------------------------------------------------------------------------------------------
def new_plan(ctx, tables, block, rows):
    n = tables.shape[0]
    full = lambda k, t=torch.int32: torch.full((k,), -77, dtype=t, device="cuda")  # noqa: E731
    return api.StepPlan(ctx, block, i32(tables), lens=full(n), cu_rows=full(n + 1), row_seq=full(rows), row_pos=full(rows), slots=full(rows, torch.int64), counts=full(3))


def check_plan(plan, want, seqs):
    got = [t.cpu().numpy() for t in (plan.tables, plan.lens, plan.cu_rows, plan.row_seq, plan.row_pos, plan.slots, plan.counts)]
    for g, w, name in zip(got, want, ("tables", "lens", "cu_rows", "row_seq", "row_pos", "slots", "counts")):
        assert np.array_equal(g[: len(w)] if name in ("lens", "cu_rows") else g, w), name
        if name in ("lens", "cu_rows"):
            assert (g[len(w):] == -77).all(), name       # sequences that the step does not have


@pytest.mark.parametrize("seqs,block,lo,hi,new,rows,short", [
    (1, 16, 0, 0, 1, 1, 0), (1, 1, 7, 7, 5, 5, 0), (3, 16, 0, 40, 20, 64, 0), (8, 24, 100, 300, 1, 8, 0), (33, 16, 0, 500, 70, 1500, 0),
    (40, 128, 0, 1000, 300, 12000, 5), (1025, 16, 0, 300, 3, 4096, 0), (5000, 8, 0, 30, 4, 9000, 40), (16384, 16, 0, 10, 1, 16384, 0)])
def test_plan(ctx, seqs, block, lo, hi, new, rows, short):
    rng = np.random.default_rng(seqs + block)
    start, n = rng.integers(lo, hi + 1, seqs), rng.integers(0, new + 1, seqs)
    n[rng.random(seqs) < 0.1] = -3                       # counts as none
    held = -(-start // block)
    wide = int(max(1, (-(-(start + np.maximum(n, 0)) // block)).max() - (1 if short else 0)))   # the longest sequence may find its row full
    ids = rng.permutation(int(held.sum()) + seqs * (new // block + 2))
    tables = np.full((seqs + 2, wide), -1, np.int32)     # room for two sequences more
    at = 0
    for b in range(seqs):
        h = min(held[b], wide)
        tables[b, :h] = ids[at: at + h]
        at += h
    need = int((-(-(start + np.maximum(n, 0)) // block) - held).sum())
    free = ids[at: at + max(0, need + (3 if not short else -short))]
    plan = new_plan(ctx, tables, block, rows)
    for _ in range(2):                                   # a second call finds the same
        plan.build(i32(start), i32(n), i32(free))
    want = plan_reference(start, n, free, tables, block, rows)
    assert plan.n_seqs == seqs
    check_plan(plan, want, seqs)


def test_plan_refusals(ctx):
    plan = new_plan(ctx, np.full((4, 8), -1, np.int32), 16, 8)
    one = i32([1])
    for args in ((i32([1] * 5), i32([1] * 5), one), (i32([1, 2]), one, one), (one.float(), one, one), (one, one, torch.zeros(1, dtype=torch.int32)), (one[:0], one[:0], one)):
        with refused():
            plan.build(*args)
    with refused():
        api.StepPlan(ctx, 16, plan.tables).build(one, one, one)                          # no arrays to fill
    with refused():
        api.StepPlan(ctx, 0, plan.tables, plan.lens, plan.cu_rows, plan.row_seq, plan.row_pos, plan.slots, plan.counts).build(one, one, one)
    with refused():
        api.StepPlan(ctx, 16, plan.tables, lens=plan.lens[:2])


# ---- write ------------------------------------------------------------------------------------------------------------------
def new_cache(ctx, kind, layers, blocks, heads, block, dim, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, blocks, heads, 2, block, pitch_of(dim))
    codes = torch.randint(-100, 100, shape, generator=g, device="cuda", dtype=torch.int8)
    codes[..., dim:] = 0
    if kind == "e4m3":
        codes = torch.where(codes.bitwise_and(127) == 127, 0, codes).to(torch.int8).view(torch.float8_e4m3fn)   # no NaN among them
    scales = torch.rand(shape[:4], generator=g, device="cuda") * 0.02 + 0.005
    layout = api.KvLayout(layers, blocks, block, heads, dim)
    return api.KvCache8(ctx, layout, codes=codes, scales=scales)


def rows_plan(ctx, block, slots, tables=None):
    return api.StepPlan(ctx, block, i32(np.zeros((1, 1)) if tables is None else tables), slots=torch.tensor(slots, dtype=torch.int64, device="cuda"))


def check_write(ctx, cache, kind, plan, k, v, layer, slots, block):
    codes, scales = cache.codes.view(torch.int8).view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy()
    cache.write(plan, k, v, layer=layer)
    want_c, want_s = codes.copy(), scales.copy()
    want_c[layer], want_s[layer] = write_reference(codes[layer], scales[layer], k.float().cpu().numpy(), v.float().cpu().numpy(), slots, kind, block)
    got_c, got_s = cache.codes.view(torch.int8).view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy()
    assert np.array_equal(got_s, want_s, equal_nan=True)
    assert np.array_equal(got_c, want_c)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,block,heads,dim", [("f32", 16, 2, 64), ("bf16", 16, 3, 128), ("f16", 8, 1, 80), ("f32", 1, 2, 24), ("bf16", 24, 2, 7), ("f16", 128, 1, 256), ("f32", 40, 1, 97)])
def test_write(ctx, kind, dtype, block, heads, dim):
    rng = np.random.default_rng(block * dim)
    blocks = 12
    cache = new_cache(ctx, kind, 2, blocks, heads, block, dim, seed=dim)
    # runs: a whole block and the beginning of the next, a token behind old ones, some in the middle of a block up to its end
    order = rng.permutation(blocks)
    slots = [order[0] * block + i for i in range(block)] + [order[1] * block + i for i in range((block + 1) // 2)]
    for b, first in ((order[2], block // 2), (order[3], block - 1), (order[4], 0)):
        slots += [b * block + i for i in range(first, min(block, first + 3))]
    slots += [-1, -5, blocks * block, (1 << 40), order[5] * block]         # skipped, and one more
    n = len(slots)
    for scale in (0.001, 1.0, 30.0):                                       # scales that stay, and that grow
        k, v = (torch.tensor(rng.standard_normal((n, heads, dim)) * scale, dtype=TYPES[dtype], device="cuda") for _ in range(2))
        check_write(ctx, cache, kind, rows_plan(ctx, block, slots), k, v, 1, slots, block)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_write_long_run_of_rows(ctx, kind):
    """Prompts of which a warp looks through several rows: units that begin in one warp's rows and end in another's."""
    rng = np.random.default_rng(5)
    block, heads, dim, blocks = 24, 8, 64, 200
    cache = new_cache(ctx, kind, 1, blocks, heads, block, dim)
    order, slots = rng.permutation(blocks), []
    for i in range(0, 180, 3):
        first, last = rng.integers(0, block), rng.integers(1, 3 * block)
        slots += [order[i + t // block] * block + t % block for t in range(first, max(first + 1, last))]
    k, v = (torch.tensor(rng.standard_normal((len(slots), heads, dim)) * 5, dtype=torch.float32, device="cuda") for _ in range(2))
    assert len(slots) * heads * 2 > 2 * 148 * 32         # more than one row a warp
    check_write(ctx, cache, kind, rows_plan(ctx, block, slots), k, v, 0, slots, block)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_write_of_values_at_the_edges(ctx, kind):
    block, dim = 4, 64
    cache = new_cache(ctx, kind, 1, 8, 1, block, dim)
    lines = np.zeros((8, 1, dim), np.float32)
    lines[1, 0, :3] = [1e-45, -3e-44, 2e-42]          # a scale among the subnormals
    lines[2, 0, :2] = [3e38, -1e-3]
    lines[3, 0, 5] = np.inf
    lines[4, 0, 6] = np.nan
    lines[5, 0] = np.linspace(-127, 127, dim)         # halves
    lines[5, 0, :4] = [127, 0.5, -0.5, 1.5]
    lines[6, 0] = 1.0
    k = torch.tensor(lines, device="cuda")
    check_write(ctx, cache, kind, rows_plan(ctx, block, [i * block for i in range(8)]), k, -k, 0, [i * block for i in range(8)], block)
    slots = [i * block + 1 for i in range(8)]         # behind them: an empty block, one that is not a number
    k2 = torch.full((8, 1, dim), 0.25, device="cuda")
    check_write(ctx, cache, kind, rows_plan(ctx, block, slots), k2, k2, 0, slots, block)
    assert torch.isnan(cache.scales[0, 3]).all() and torch.isnan(cache.scales[0, 4]).all()
    check_write(ctx, cache, kind, rows_plan(ctx, block, [12]), k2[:1], k2[:1], 0, [12], block)   # written anew
    assert torch.isfinite(cache.scales[0, 3]).all()


def test_write_of_rows_cut_from_a_projection(ctx):
    """k and v as columns of one [q; k; v] row, at addresses that allow no wide loads."""
    rng = np.random.default_rng(8)
    for dtype, lead in (("f32", 3), ("f32", 4), ("bf16", 5), ("f16", 8)):
        heads, dim, block, n = 2, 64, 16, 20
        qkv = torch.tensor(rng.standard_normal((n, lead + 2 * heads * dim + 1)), dtype=TYPES[dtype], device="cuda")
        k, v = (qkv[:, lead + i * heads * dim: lead + (i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in range(2))
        cache = new_cache(ctx, "int8", 1, 4, heads, block, dim)
        slots = list(range(16, 16 + n))
        check_write(ctx, cache, "int8", rows_plan(ctx, block, slots), k, v, 0, slots, block)


def test_write_refusals_and_pool_calls(ctx):
    cache = new_cache(ctx, "int8", 2, 6, 2, 16, 64)
    plan = rows_plan(ctx, 16, [0, 1])
    k = torch.zeros(2, 2, 64, device="cuda")
    for a, b, p, layer in ((k, k, plan, 2), (k, k, plan, -1), (k.double(), k, plan, 0), (k, k.half(), plan, 0), (k[:1], k, plan, 0), (k.transpose(1, 2), k, plan, 0),
                           (k.cpu(), k, plan, 0), (k[..., ::2], k, plan, 0), (torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), plan, 0),
                           (k, k, rows_plan(ctx, 8, [0, 1]), 0), (k[:1].expand(2, 2, 64), k, plan, 0)):
        with refused():
            cache.write(p, a, b, layer=layer)
    cache.write(plan, k[:0], k[:0])                                       # nothing to do
    before = cache.codes.clone(), cache.scales.clone()
    cache.copy_block(1, 4)
    cache.ctx.synchronize()
    assert torch.equal(cache.codes[:, 4], before[0][:, 1]) and torch.equal(cache.scales[:, 4], before[1][:, 1]) and torch.equal(cache.codes[:, :4], before[0][:, :4])
    for src, dst in ((1, 1), (0, 6), (-1, 0)):
        with refused():
            cache.copy_block(src, dst)
    got = cache.read_token(1, 4, 3)
    for side in (0, 1):
        want = cache.codes[1, 4, :, side, 3].float() * cache.scales[1, 4, :, side, None]
        assert np.array_equal(got[side].reshape(2, 64), want.cpu().numpy())
    with refused():
        cache.read_token(0, 0, 16)
    own = api.KvCache8(ctx, api.KvLayout(1, 3, 16, 2, 80), kind=_lib.PI_E4M3)
    assert own.bytes() == 3 * 2 * 2 * (16 * 96 + 4)
    own.write(rows_plan(ctx, 16, [17, 18]), torch.ones(2, 2, 80, device="cuda"), torch.full((2, 2, 80), -2.0, device="cuda"))
    own.write(rows_plan(ctx, 16, [16]), torch.ones(1, 2, 80, device="cuda"), torch.full((1, 2, 80), -2.0, device="cuda"))
    k1, v1 = own.read_token(0, 1, 0)
    assert np.abs(k1 - 1).max() < 1e-6 and np.abs(v1 + 2).max() < 1e-6
    huge = 2**31 - 1
    for layout in (api.KvLayout(1, 3, 16, 2, 257), api.KvLayout(1, 3, 5000, 2, 64), api.KvLayout(0, 3, 16, 2, 64), api.KvLayout(huge, huge, 4096, 1024, 256)):
        with refused():
            api.KvCache8(ctx, layout)
    with refused():
        api.KvCache8(ctx, api.KvLayout(1, 3, 16, 2, 64), kind=_lib.PI_F32)


# ---- attention --------------------------------------------------------------------------------------------------------------
def attention_case(ctx, kind, dtype, block, heads, kv_heads, dim, contexts, news, window=0, seed=0, holes=False, spread=0.3, q_scale=1.0, pad=0, hints=True, scale=None):
    """One call against the reference; returns (q, out, cache, plan, everything that the reference was given)."""
    rng = np.random.default_rng(seed)
    contexts, news = np.asarray(contexts), np.asarray(news)
    B = len(contexts)
    after = -(-contexts // block)
    wide, blocks = int(max(1, after.max())), int(after.sum()) + 2
    ids = rng.permutation(blocks)
    tables, at = np.full((B, wide), -1, np.int32), 0
    for b in range(B):
        tables[b, : after[b]] = ids[at: at + after[b]]
        at += after[b]
    if holes:                                            # blocks that are not mapped, and ids that the pool does not have
        for b in range(B):
            for j in range(after[b]):
                if rng.random() < 0.3:
                    tables[b, j] = rng.choice([-1, blocks, 1 << 30])
        after = np.where(rng.random(B) < 0.3, after // 2, after)
    cu = np.concatenate([[0], np.cumsum(news)])
    rows = int(cu[-1])
    pos = np.concatenate([np.arange(c - n, c) for c, n in zip(contexts, news)] + [np.zeros(0, np.int64)]).astype(np.int64)
    shape = (2, blocks, kv_heads, 2, block, pitch_of(dim))
    codes = torch.tensor(np.clip(np.round(rng.standard_normal(shape) * 35), -127, 127), device="cuda", dtype=torch.float32)
    codes = codes.to(torch.int8) if kind == "int8" else (codes * 3).to(torch.float8_e4m3fn)
    scales = torch.tensor(np.exp(rng.standard_normal(shape[:4]) * spread) / (35 if kind == "int8" else 105), device="cuda", dtype=torch.float32)
    layout = api.KvLayout(2, blocks, block, kv_heads, dim)
    cache = api.KvCache8(ctx, layout, codes=codes, scales=scales)
    q = torch.tensor(rng.standard_normal((rows + pad, heads, dim)) * q_scale, dtype=TYPES[dtype], device="cuda")
    out = torch.full_like(q, 7.0)
    plan = api.StepPlan(ctx, block, i32(tables), lens=i32(after), cu_rows=i32(cu), row_pos=i32(np.concatenate([pos, np.full(pad, -1)])))
    given = dict(tables=tables, lens=after, cu=cu, pos=pos, block=block, kind=kind, window=window, scale=scale)
    kw = dict(max_seq_rows=int(max(1, news.max())), max_context=int(max(1, contexts.max()))) if hints else {}
    api.PagedAttention8(layout, heads).run_device(q, out, cache, plan, layer=1, window=window or None, scale=scale, **kw)
    check_attention(q, out, cache, given, rows, dtype)
    return q, out, cache, plan, given


def check_attention(q, out, cache, given, rows, dtype):
    codes, scales = cache.codes[1].view(torch.int8).view(torch.uint8).cpu().numpy(), cache.scales[1].cpu().numpy()
    want, most, mass = attention_reference(q[:rows].float().cpu().numpy(), codes, scales, **given)
    got = out.float().cpu().numpy().astype(np.float64)
    assert (got[rows:] == 7.0).all()                     # rows behind the last sequence
    off = np.abs(got[:rows] - want) - attention_tolerance(want, most, mass, want.shape[-1], dtype)
    assert not (off > 0).any(), f"{off.max()} beyond the tolerance at {np.unravel_index(off.argmax(), off.shape)}"
    assert (got[:rows][most == 0] == 0).all()            # rows that see nothing


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block,heads,kv_heads,dim", [(16, 8, 2, 64), (16, 8, 8, 128), (8, 12, 1, 80), (24, 10, 2, 24), (1, 4, 2, 32), (64, 7, 1, 96), (40, 16, 1, 256), (128, 5, 1, 129)])
def test_attention_of_single_tokens(ctx, kind, dtype, block, heads, kv_heads, dim):
    attention_case(ctx, kind, dtype, block, heads, kv_heads, dim, [1, 2, 15, 16, 17, 100, 333], [1] * 7, seed=dim)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block,heads,kv_heads,dim,window", [(16, 8, 2, 64, 0), (16, 4, 4, 128, 50), (24, 6, 2, 64, 17), (16, 32, 2, 64, 1), (8, 5, 1, 40, 0), (32, 4, 1, 192, 33), (16, 12, 4, 128, 0)])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attention_of_portions(ctx, kind, dtype, block, heads, kv_heads, dim, window):
    """Portions beside single tokens, a sequence without rows among them, rows behind the last."""
    attention_case(ctx, kind, dtype, block, heads, kv_heads, dim, [1, 90, 70, 200, 37], [1, 33, 0, 1, 37], window=window, seed=window + dim, pad=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_long_portions(ctx, dtype, dim):
    attention_case(ctx, "int8", dtype, 16, 4, 1, dim, [400, 300, 129], [300, 1, 129], seed=4)
    attention_case(ctx, "e4m3", dtype, 32, 2, 2, dim, [500], [257], window=200, seed=5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("contexts,window", [([3000], 0), ([2500, 10, 1300], 0), ([4000], 700)])
def test_attention_of_long_contexts(ctx, dtype, contexts, window):
    """Contexts that the CTAs of a cluster share."""
    attention_case(ctx, "int8", dtype, 16, 8, 2, 64, contexts, [1] * len(contexts), window=window, seed=9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,contexts,news,window", [(8, 1, 64, [3000], [20], 0), (8, 2, 128, [2500, 40], [33, 40], 0), (16, 1, 128, [2100], [9], 1500), (4, 1, 128, [5000], [40], 0),
                                                                       (96, 1, 64, [300, 1700], [1, 3], 0), (200, 2, 64, [700], [2], 0), (150, 1, 128, [90], [3], 0)])
def test_attention_of_portions_behind_long_contexts(ctx, dtype, heads, kv_heads, dim, contexts, news, window):
    """Few tiles of rows, whose positions a cluster shares; groups wider than a product, and than a tile."""
    attention_case(ctx, "e4m3" if dim == 64 else "int8", dtype, 16, heads, kv_heads, dim, contexts, news, window=window, seed=heads)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_many_sequences(ctx, dtype):
    """More sequences than a warp looks at once, portions, single tokens and nothing among them."""
    rng = np.random.default_rng(4)
    news = rng.choice([0, 1, 1, 2, 40, 70], 75)
    attention_case(ctx, "int8", dtype, 16, 2, 1, 64, news + rng.integers(0, 60, 75), news, seed=4, pad=5)


@pytest.mark.parametrize("news", [[1, 1, 1, 1, 1, 1], [20, 1, 3, 40, 1, 1], [90, 16, 3, 100, 31, 64]])
def test_attention_over_tables_with_holes(ctx, news):
    for dtype in ("f32", "bf16"):
        attention_case(ctx, "int8", dtype, 16, 8, 2, 64, [200, 16, 3, 150, 31, 64], news, seed=11, holes=True)


def test_attention_without_hints_and_with_wrong_ones(ctx):
    q, out, cache, plan, given = attention_case(ctx, "int8", "f32", 16, 8, 2, 64, [300, 40], [70, 40], seed=3, hints=False)
    for hints in (dict(max_seq_rows=1, max_context=1), dict(max_seq_rows=3), dict(max_context=100000)):
        again = torch.full_like(out, 7.0)
        api.PagedAttention8(cache.layout, 8).run_device(q, again, cache, plan, layer=1, **hints)
        check_attention(q, again, cache, given, q.shape[0], "f32")


def test_attention_scores_far_apart_and_scales_far_apart(ctx):
    """Sharp weights, and blocks whose scales differ by orders of magnitude."""
    for dtype in ("f32", "bf16"):
        for news in ([1, 20], [1, 130]):
            attention_case(ctx, "int8", dtype, 16, 4, 2, 64, [150, 300], news, seed=2, scale=3.0)
            attention_case(ctx, "int8", dtype, 16, 4, 2, 64, [150, 300], news, seed=2, spread=3.0, q_scale=0.05)
    for news in ([1, 10], [1, 80]):
        attention_case(ctx, "int8", "f32", 16, 4, 2, 64, [60, 90], news, seed=6, q_scale=1e30, scale=1e-31)
        attention_case(ctx, "e4m3", "f32", 16, 4, 2, 64, [60, 90], news, seed=6, q_scale=1e-30, scale=1e29)


@pytest.mark.parametrize("news", [[1], [30], [90]])
def test_attention_with_values_that_are_not_finite(ctx, news):
    """A block whose scales are NaN reaches the rows that see one of its tokens and no others."""
    q, out, cache, plan, given = attention_case(ctx, "int8", "f32", 16, 4, 2, 64, [100], news, seed=1, window=40, hints=False)
    tables, pos = given["tables"], given["pos"]
    for b, side in ((2, 0), (3, 1), (4, 1), (4, 0)):
        keep = cache.scales.clone()
        cache.scales[1, tables[0, b], :, side] = float("nan")
        again = torch.full_like(out, 7.0)
        api.PagedAttention8(cache.layout, 4).run_device(q, again, cache, plan, layer=1, window=40)
        sees = (pos >= b * 16) & (np.maximum(0, pos - 39) < b * 16 + 16)
        got = again.cpu().numpy()
        assert np.isnan(got[sees]).all() and np.array_equal(got[~sees], out.cpu().numpy()[~sees])
        cache.scales.copy_(keep)
    q[0, 1, 3] = float("inf")
    again = torch.full_like(out, 7.0)
    api.PagedAttention8(cache.layout, 4).run_device(q, again, cache, plan, layer=1, window=40)
    assert np.isnan(again[0, 1].cpu().numpy()).all()
    others = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    others[0, 1] = False
    assert torch.equal(again[others], out[others])


def test_attention_over_strided_rows(ctx):
    q, out, cache, plan, given = attention_case(ctx, "int8", "bf16", 16, 4, 2, 64, [100, 30], [5, 1], seed=1)
    wide = torch.zeros(6, 3 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    q2, out2 = (wide[:, o: o + 256].unflatten(1, (4, 64)) for o in (3, 301))
    q2.copy_(q)
    api.PagedAttention8(cache.layout, 4).run_device(q2, out2, cache, plan, layer=1, max_seq_rows=5, max_context=100)
    assert torch.equal(out2, out) and (wide[:, 557:] == 0).all() and (wide[:, :3] == 0).all()


@pytest.mark.parametrize("news", [[1, 1], [40, 1]])
def test_a_cache_beyond_32_bits(ctx, news):
    """The same blocks at the front of a small pool and at the end of one of 4.9 GB: the same codes, scales and results."""
    heads, dim, block, far = 8, 128, 16, 150000
    rng = np.random.default_rng(2)
    contexts = np.array([90, 33])
    after = -(-contexts // block)
    rows = int(sum(news))
    q, k, v = (torch.tensor(rng.standard_normal((rows, n, dim)), dtype=torch.bfloat16, device="cuda") for n in (16, heads, heads))
    small = new_cache(ctx, "int8", 1, 12, heads, block, dim, seed=3)
    codes = torch.zeros((1, far, heads, 2, block, dim), dtype=torch.int8, device="cuda")
    scales = torch.ones((1, far, heads, 2), device="cuda")
    codes[:, far - 12:], scales[:, far - 12:] = small.codes, small.scales
    large = api.KvCache8(ctx, api.KvLayout(1, far, block, heads, dim), codes=codes, scales=scales)
    outs = []
    for cache, shift in ((small, 0), (large, far - 12)):
        ids = rng.permutation(12)[: after.sum()] if not outs else ids
        tables = np.full((2, 6), -1)
        tables[0, : after[0]], tables[1, : after[1]] = ids[: after[0]] + shift, ids[after[0]:] + shift
        pos = np.concatenate([np.arange(c - n, c) for c, n in zip(contexts, news)])
        seq = np.repeat([0, 1], news)
        slots = torch.tensor(tables[seq, pos // block] * block + pos % block, dtype=torch.int64, device="cuda")
        plan = api.StepPlan(ctx, block, i32(tables), lens=i32(after), cu_rows=i32([0, news[0], rows]), row_pos=i32(pos), slots=slots)
        cache.write(plan, k, v)
        out = torch.zeros_like(q)
        api.PagedAttention8(cache.layout, 16).run_device(q, out, cache, plan)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(large.codes[:, far - 12:], small.codes) and torch.equal(large.scales[:, far - 12:], small.scales)
    assert (large.codes[:, : far - 12] == 0).all()


def test_attention_in_place(ctx):
    """Results may replace the queries."""
    for contexts, news in (([300, 40], [1, 1]), ([2000], [40]), ([400], [200])):
        q, out, cache, plan, given = attention_case(ctx, "int8", "bf16", 16, 8, 2, 64, contexts, news, seed=8)
        same = q.clone()
        api.PagedAttention8(cache.layout, 8).run_device(same, same, cache, plan, layer=1, max_seq_rows=int(max(news)), max_context=int(max(contexts)))
        assert torch.equal(same, out)


def test_attention_of_windows_and_lengths_out_of_any_range(ctx):
    """A window beyond 32 bits is none; tables of a negative length hold nothing; positions up to 2^31 - 1 see what is mapped of their window."""
    for news in ([1, 1, 1], [3, 40, 20]):
        q, out, cache, plan, given = attention_case(ctx, "int8", "bf16", 16, 8, 2, 64, [300, 40, 90], news, seed=9)
        a, cut = api.PagedAttention8(cache.layout, 8), dict(max_seq_rows=max(news), max_context=300)
        for window in (2**31 - 1, 2**32 + 1):
            same = torch.full_like(out, 7.0)
            a.run_device(q, same, cache, plan, layer=1, window=window, **cut)
            assert torch.equal(same, out)
        given.update(lens=np.array([given["lens"][0], 0, 0]), window=2**31 - 200)
        given["pos"] = np.where(np.arange(sum(news)) < news[0], 2**31 - 1, given["pos"])
        plan = api.StepPlan(ctx, 16, plan.tables, lens=i32([given["lens"][0], -1, -(2**27) - 1]), cu_rows=plan.cu_rows, row_pos=i32(given["pos"]))
        again = torch.full_like(out, 7.0)
        a.run_device(q, again, cache, plan, layer=1, window=given["window"], **cut)
        given["window"], given["pos"] = 304 - 200, np.where(given["pos"] == 2**31 - 1, 303, given["pos"])   # positions 200 to 303, as before
        check_attention(q, again, cache, given, q.shape[0], "bf16")


def test_attention_refusals(ctx):
    q, out, cache, plan, _ = attention_case(ctx, "int8", "f32", 16, 4, 2, 64, [20], [2], seed=1)
    a = api.PagedAttention8(cache.layout, 4)
    for kw in (dict(layer=2), dict(window=0), dict(window=-3), dict(scale=0.0), dict(scale=float("nan")), dict(scale=3e38), dict(max_seq_rows=0), dict(max_context=0)):
        with refused():
            a.run_device(q, out, cache, plan, **kw)
    for x, y, p in ((q.bfloat16(), out, plan), (q[:1], out, plan), (q.cpu(), out, plan), (q[:, :3], out[:, :3], plan), (q, out, api.StepPlan(ctx, 16, plan.tables)),
                    (q, out, api.StepPlan(ctx, 8, plan.tables, plan.lens, plan.cu_rows, row_pos=plan.row_pos)),
                    (q, out, api.StepPlan(ctx, 16, plan.tables, plan.lens, plan.cu_rows, row_pos=plan.row_pos[:1]))):
        with refused():
            a.run_device(x, y, cache, p)
    with refused():
        api.PagedAttention8(cache.layout, 3).run_device(q[:, :3].contiguous(), out[:, :3].contiguous(), cache, plan)
    a.run_device(q[:0], out[:0], cache, plan)


# ---- sampling ---------------------------------------------------------------------------------------------------------------
def check_sample(ctx, x, t, k, p, m, u):
    """Rows of x under parameters per row, against the reference; probabilities to a few roundings of f32."""
    rows = x.shape[0]
    f = lambda v: torch.tensor(np.broadcast_to(np.asarray(v, np.float32), rows).copy(), device="cuda")  # noqa: E731
    t, p, m, u = f(t), f(p), f(m), f(u)
    k = i32(np.broadcast_to(np.asarray(k), rows).copy())
    ids, probs = torch.full((rows,), -9, dtype=torch.int32, device="cuda"), torch.full((rows,), -9.0, device="cuda")
    api.sample(ctx, x, t, k, p, m, u, ids, probs)
    alone = torch.full_like(ids, -9)
    api.sample(ctx, x, t, k, p, m, u, alone)
    assert torch.equal(ids, alone)
    xs = x.float().cpu().numpy()
    got = ids.tolist(), probs.tolist()
    for r in range(rows):
        want = sample_reference(xs[r], *(v[r].item() for v in (t, k, p, m, u)))
        assert got[0][r] == want[0], (r, got[0][r], want)
        assert abs(got[1][r] - want[1]) <= 2.0 ** -22 * want[1], (r, got[1][r], want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 16384, 16385, 50257, 128256])
def test_sample(ctx, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 24
    x = torch.tensor(rng.standard_normal((rows, vocab)) * 3, dtype=TYPES[dtype], device="cuda")
    x[3] = 0.5                                           # all equal
    x[4, rng.random(vocab) < 0.9] = -float("inf")
    x[4, 0] = 1.0
    x[5] = x[5].round()                                  # many equal ones
    x[6, : vocab // 2] = torch.finfo(x.dtype).min        # masked with the type's lowest value
    t = rng.choice([0.3, 0.7, 1.0, 1.6], rows)
    k = rng.choice([0, 1, 2, 40, 1000, 200000], rows)
    p = rng.choice([1.0, 0.95, 0.5, 0.05], rows)
    m = rng.choice([0.0, 0.0, 0.02, 0.3], rows)
    u = rng.random(rows).astype(np.float32)
    u[:3] = [0.0, 0.99999994, 0.5]
    t[7], t[8] = 0.0, 0.0
    check_sample(ctx, x, t, k, p, m, u)
    check_sample(ctx, x, t, 0, p, 0, u)                  # the nucleus alone
    check_sample(ctx, x, t, k, 1, 0, u)
    check_sample(ctx, x, t, 0, 1, 0, u)


def test_sample_at_the_edges(ctx):
    rng = np.random.default_rng(3)
    x = torch.tensor(rng.standard_normal((16, 5000)), dtype=torch.float32, device="cuda")
    inf = float("inf")
    x[0] = -inf
    x[1] = float("nan")
    x[2, 100:] = float("nan")
    x[3, [7, 4000]] = inf
    x[4] = torch.finfo(torch.float32).min
    x[5, 10:] = -inf
    x[6, :] = -0.0
    x[6, 4000] = 0.0                                     # equal to the others
    x[7] *= 1e30
    for t in (1.0, 1e-30, 1e-6, 1e6, inf, 0.0, -1.0, float("nan")):
        for k, p, m in ((0, 1, 0), (1, 1, 0), (7, 0.5, 0), (0, 0.3, 0.5), (0, 0.0, 0), (0, -1, 0), (0, 1, 1.0), (0, 1, 5.0), (-4, 2.0, -1)):
            if not t > 1e5 or (k, p) == (0, 1):          # flat weights meet borders exactly: counts alone, without a nucleus
                check_sample(ctx, x, t, k, p, m, rng.random(16).astype(np.float32))
    ids = torch.empty(16, dtype=torch.int32, device="cuda")
    one, zero = torch.ones(16, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    for u in (-1.0, float("nan"), 1.0, 7.0):             # outside [0, 1): still one of the kept
        api.sample(ctx, x, one, zero + 3, one, one * 0, one * u, ids)
        for r in (5, 8, 12):
            assert ids[r].item() in x[r].topk(3).indices.tolist()
    assert ids[0] == -1 and ids[1] == -1


def test_sample_of_the_longest_rows_and_strided_ones(ctx):
    rng = np.random.default_rng(4)
    g = torch.Generator(device="cuda").manual_seed(1)
    for vocab in (200001, 393216):
        x = torch.randn(3, vocab, generator=g, device="cuda") * 2
        x[2] = 1.0
        check_sample(ctx, x, 1.0, [0, 50000, 0], [0.99, 0.9, 1.0], 0, [0.3, 0.999, 0.7])
    wide = torch.randn(9, 1003, generator=g, device="cuda").half()
    check_sample(ctx, wide[:, 2:1000], rng.uniform(0.5, 1.5, 9), 0, 0.9, 0, rng.random(9))
    check_sample(ctx, wide[:1], 1.0, 0, 0.9, 0, 0.3)


def test_sample_in_proportion(ctx):
    """Random numbers that cover [0, 1) evenly bring every kept token as often as its probability says, up to one draw at each border."""
    n = 4096
    x = torch.tensor([[1.0, 0.0, 2.0, -1.0, 1.5]], device="cuda").expand(n, 5).contiguous()
    full = lambda v: torch.full((n,), v, device="cuda")  # noqa: E731
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    api.sample(ctx, x, full(0.8), torch.full((n,), 4, dtype=torch.int32, device="cuda"), full(1.0), full(0.0), (torch.arange(n, device="cuda") + 0.5) / n, ids)
    w = torch.exp(x[0].double() / 0.8)
    w[3] = 0
    assert (ids.long().bincount(minlength=5) - w / w.sum() * n).abs().max() <= 1


def test_sample_refusals(ctx):
    x, f, i = torch.zeros(2, 8, device="cuda"), torch.ones(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for args in ((x.double(), f, i, f, f, f, i), (x[0], f, i, f, f, f, i), (x.T, f, i, f, f, f, i), (x, f[:1], i, f, f, f, i), (x, f, f, f, f, f, i), (x, f, i, f, f, f, i.long()),
                 (x.cpu(), f, i, f, f, f, i), (x, f, i, f.double(), f, f, i), (x[:1].expand(2, 8), f, i, f, f, f, i), (x[:, :0], f, i, f, f, f, i)):
        with refused():
            api.sample(ctx, *args)
    with refused():
        api.sample(ctx, torch.zeros(1, 393217, device="cuda"), f[:1], i[:1], f[:1], f[:1], f[:1], i[:1])
    api.sample(ctx, x[:0], f[:0], i[:0], f[:0], f[:0], f[:0], i[:0])


# ---- the four together ------------------------------------------------------------------------------------------------------
class Step:
    """A step of a toy model: q, k, v and logits are given, everything between lengths and tokens happens on the device."""

    def __init__(self, ctx, seed, seqs=6, rows=40, block=16, heads=8, kv_heads=2, dim=64, vocab=500):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.block, self.blocks = ctx, block, 80
        self.cache = new_cache(ctx, "int8", 2, self.blocks, kv_heads, block, dim, seed)
        self.plan = new_plan(ctx, np.full((seqs, 10), -1, np.int32), block, rows)
        self.start, self.n = i32([0] * seqs), i32([0] * seqs)
        self.free = i32(np.random.default_rng(seed).permutation(self.blocks))
        new = lambda *s: torch.empty(*s, device="cuda").normal_(generator=g)  # noqa: E731
        self.q, self.k, self.v = new(rows, heads, dim), new(rows, kv_heads, dim), new(rows, kv_heads, dim)
        self.out, self.weights = torch.zeros_like(self.q), new(heads * dim, vocab)
        self.logits = torch.zeros(rows, vocab, device="cuda")
        full = lambda v, t=torch.float32: torch.full((rows,), v, dtype=t, device="cuda")  # noqa: E731
        self.sampling = [full(0.8), full(20, torch.int32), full(0.9), full(0.01), torch.rand(rows, generator=g, device="cuda")]
        self.ids = full(-5, torch.int32)
        self.attention = api.PagedAttention8(self.cache.layout, heads)

    def run(self):
        self.plan.build(self.start, self.n, self.free)
        for layer in (0, 1):
            self.cache.write(self.plan, self.k, self.v, layer=layer)
            self.attention.run_device(self.q, self.out, self.cache, self.plan, layer=layer, max_seq_rows=16, max_context=160)
        torch.matmul(self.out.flatten(1), self.weights, out=self.logits)
        api.sample(self.ctx, self.logits, *self.sampling, self.ids)

    def give(self, start, n):
        self.start.copy_(i32(start))
        self.n.copy_(i32(n))
        for t in (self.q, self.k, self.v):
            t.normal_(generator=self.g)

    def state(self):
        return [t.clone() for t in (self.cache.codes, self.cache.scales, self.plan.tables, self.out, self.ids, self.plan.slots)]


STEPS = [([0] * 6, [16, 1, 9, 0, 3, 5]), ([16, 1, 9, 0, 3, 5], [1, 1, 1, 12, 1, 0]), ([17, 2, 10, 12, 4, 5], [1, 1, 1, 1, 1, 1])]


def walk(step, run):
    states, free = [], 0
    for start, n in STEPS:
        step.give(start, n)
        step.out.zero_()
        before = step.cache.codes[1].clone(), step.cache.scales[1].clone()
        run()
        torch.cuda.synchronize()
        states.append(step.state() + list(before))
        free += int(step.plan.counts[1])
        assert step.plan.counts.tolist()[::2] == [sum(n), 0]
        step.free[: -int(step.plan.counts[1]) or None].copy_(step.free[int(step.plan.counts[1]):].clone())
    return states


def test_a_whole_step(ctx):
    step = Step(ctx, 1)
    for (start, n), state in zip(STEPS, walk(step, step.run)):
        out, slots, rows = state[3], state[5], sum(n)
        assert (slots[rows:] == -1).all() and (slots[:rows] >= 0).all() and (out[rows:] == 0).all()
        assert len(set(slots[:rows].tolist())) == rows
    # the last step against the references
    codes, scales, tables, out, ids, slots, before_c, before_s = state
    rows = sum(STEPS[-1][1])
    want_c, want_s = write_reference(before_c.view(torch.uint8).cpu().numpy(), before_s.cpu().numpy(), step.k.cpu().numpy(), step.v.cpu().numpy(), slots.cpu().numpy(), "int8", 16)
    assert np.array_equal(codes[1].view(torch.uint8).cpu().numpy(), want_c) and np.array_equal(scales[1].cpu().numpy(), want_s)
    given = dict(tables=tables.cpu().numpy(), lens=step.plan.lens.cpu().numpy(), cu=step.plan.cu_rows.cpu().numpy(), pos=step.plan.row_pos.cpu().numpy(), block=16, kind="int8")
    want, most, mass = attention_reference(step.q[:rows].cpu().numpy(), want_c, want_s, **given)
    assert (np.abs(out[:rows].cpu().numpy() - want) <= attention_tolerance(want, most, mass, 64, "f32")).all()
    logits = step.logits.cpu().numpy()
    for r in range(rows):
        assert ids[r].item() == sample_reference(logits[r], *(v[r].item() for v in step.sampling))[0]


def captured(step, stream):
    step.run()                                           # a first call outside a capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step.run()
    return graph


def test_a_captured_step_replays_on_new_lengths(ctx):
    a = Step(ctx, 2)
    eager = walk(a, a.run)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = api.Context(0, stream=stream.cuda_stream)
        b = Step(other, 2)
        graph = captured(b, stream)
        again = walk(b, graph.replay)
    for x, y in zip(eager, again):
        for s, t in zip(x, y):
            assert torch.equal(s, t)


def test_graphs_of_two_contexts_at_the_same_time(ctx):
    """Two captured steps replayed side by side on two streams: nothing is shared between them."""
    steps, graphs, streams, wants = [], [], [], []
    for seed in (3, 4):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            s = Step(api.Context(0, stream=stream.cuda_stream), seed)
            s.give(*STEPS[0])
            graphs.append(captured(s, stream))
            stream.synchronize()
            wants.append(s.state())
        steps.append(s)
        streams.append(stream)
    for _ in range(20):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for s, want in zip(steps, wants):
        for x, y in zip(s.state(), want):
            assert torch.equal(x, y)


def test_a_context_of_its_own_stream(ctx):
    """The context's own stream: the caller orders it against torch's."""
    mine = api.Context(0)
    a, b = Step(ctx, 6), Step(mine, 6)
    for s in (a, b):
        s.give(*STEPS[0])
        torch.cuda.synchronize()
        s.plan.build(s.start, s.n, s.free)
        s.cache.write(s.plan, s.k, s.v)
        s.attention.run_device(s.q, s.out, s.cache, s.plan, max_seq_rows=16)
        s.ctx.synchronize()
        torch.cuda.synchronize()
    assert torch.equal(a.out, b.out) and torch.equal(a.cache.codes, b.cache.codes) and torch.equal(a.plan.slots, b.plan.slots)
    assert mine.kernel_launches() >= 3
