"""What the device-side serving step over an 8-bit KV cache is timed on, operator by operator.

Operators (each one call of the public Python API)
  plan    block tables, row positions and cache slots of a step, from request lengths and a list of free blocks
  write   keys and values of the step's rows into a cache of 8-bit codes with a scale per block of tokens, head and side (K or V)
  attend  paged attention over that cache: decoded tokens, portions of prompts, or both in one ragged batch
  sample  a token per row of logits: temperature, top-k, min-p and top-p, from given random numbers

Cache: codes [layers][blocks][kv_heads][2][block][pitch] (int8, or float8 e4m3 bytes), scales [layers][blocks][kv_heads][2] f32; a
row of `head_dim` codes is padded with zeros to `pitch` bytes.  A value is code * scale.  Model sizes are those of this
repository's benchmark.  Lengths of a case's sequences are evenly spaced between its bounds, in an order that the seed draws.
"""
import math

import numpy as np
import torch

own = False

LAYERS, LAYER = 2, 1                       # of the pools: the second of two layers is used
TOP = {"int8": 127.0, "e4m3": 448.0}       # the largest code
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a lightly loaded server's step: eight sequences, a token each
        dict(name="plan_8", op="plan", seqs=8, lo=100, hi=1000, new_lo=1, new_hi=1, block=16),
        # the largest step: prompts in portions beside decoded tokens
        dict(name="plan_mixed_1024", op="plan", seqs=1024, lo=1, hi=4000, new_lo=1, new_hi=64, block=16),
        # one decoded token for each of 64 sequences, a layer of the benchmark's model
        dict(name="write_decode_64", op="write", codes="int8", dtype="f32", seqs=64, lo=256, hi=2048, new_lo=1, new_hi=1, block=16, kv_heads=4, dim=64),
        # prompts of a larger model's layer, some of them behind a cached prefix that ends inside a block
        dict(name="write_prompts_4", op="write", codes="e4m3", dtype="bf16", seqs=4, lo=0, hi=50, new_lo=700, new_hi=1400, block=16, kv_heads=8, dim=128),
        # one user, short context: latency
        dict(name="attend_one_short", op="attend", codes="int8", dtype="f32", seqs=1, lo=200, hi=200, new_lo=1, new_hi=1, block=16, heads=32, kv_heads=4, dim=64, window=0),
        # the loaded server of the benchmark
        dict(name="attend_decode_64", op="attend", codes="int8", dtype="f32", seqs=64, lo=256, hi=2048, new_lo=1, new_hi=1, block=16, heads=32, kv_heads=4, dim=64, window=0),
        # a larger model's layer over long contexts
        dict(name="attend_decode_16_long", op="attend", codes="e4m3", dtype="bf16", seqs=16, lo=3000, hi=4096, new_lo=1, new_hi=1, block=16, heads=32, kv_heads=8, dim=128, window=0),
        # one very long context
        dict(name="attend_one_131072", op="attend", codes="int8", dtype="bf16", seqs=1, lo=131072, hi=131072, new_lo=1, new_hi=1, block=32, heads=64, kv_heads=8, dim=128, window=0),
        # a portion of a prompt behind a long cached part
        dict(name="attend_chunk_512", op="attend", codes="int8", dtype="bf16", seqs=1, lo=4096, hi=4096, new_lo=512, new_hi=512, block=16, heads=32, kv_heads=8, dim=128, window=0),
        # a ragged batch with a window and blocks of an odd size
        dict(name="attend_mixed_16", op="attend", codes="int8", dtype="f32", seqs=16, lo=300, hi=1500, new_lo=1, new_hi=256, block=24, heads=32, kv_heads=4, dim=64, window=1024),
        # one user's token out of a small vocabulary
        dict(name="sample_1", op="sample", dtype="f32", rows=1, vocab=32000),
        # a loaded server's tokens out of a large one
        dict(name="sample_64", op="sample", dtype="f32", rows=64, vocab=128256),
    ]


def _between(rng, lo, hi):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 260e6 and w["flops"] <= 30e9:     # no more than the largest listed ones
            return case


def _draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "attend", "sample", "sample"])
    if op == "sample":
        vocab = _between(rng, 50, 128256)
        return dict(op=op, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), rows=_between(rng, 1, min(512, 64 * 128256 // vocab)), vocab=vocab)
    block = rng.choice([16, 16, 16, 32, 64, 128, 1, 8, 20, 24])
    if op == "plan":
        lo = rng.randint(0, 2000)
        new = _between(rng, 1, 64)
        return dict(op=op, seqs=_between(rng, 1, 1024), lo=lo, hi=lo + rng.randint(0, 2000), new_lo=rng.randint(0, new), new_hi=new, block=block)
    codes, dtype, dim = rng.choice(["int8", "e4m3"]), rng.choice(["f32", "bf16", "f16"]), rng.choice([64, 64, 128, 128, 96, 80, 24, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "write":
        seqs = _between(rng, 1, 64)
        lo, new = rng.randint(0, 300), _between(rng, 1, 3000 // seqs)
        return dict(op=op, codes=codes, dtype=dtype, seqs=seqs, lo=lo, hi=lo + rng.randint(0, 300), new_lo=rng.randint(1, new), new_hi=new, block=block, kv_heads=kv_heads, dim=dim)
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12])
    window = rng.choice([0, 0, 0, 100, 1024])
    if rng.random() < 0.6:
        hi = _between(rng, 1, 16384)
        seqs = _between(rng, 1, max(1, min(64, 65536 // hi)))
        return dict(op=op, codes=codes, dtype=dtype, seqs=seqs, lo=rng.randint(max(1, hi // 4), hi), hi=hi, new_lo=1, new_hi=1, block=max(block, 8), heads=heads, kv_heads=kv_heads, dim=dim, window=window)
    new = _between(rng, 2, 512)
    seqs = _between(rng, 1, max(1, min(8, 512 // new)))
    lo = new + rng.randint(0, 1000)
    return dict(op=op, codes=codes, dtype=dtype, seqs=seqs, lo=lo, hi=lo + rng.randint(0, 2000), new_lo=rng.randint(1, new), new_hi=new, block=max(block, 8), heads=heads, kv_heads=kv_heads, dim=dim, window=window)


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens ahead of the step and new tokens, per sequence, unshuffled."""
    n = case["seqs"]
    lo = np.linspace(case["lo"], case["hi"], n).astype(np.int64)
    new = np.linspace(case["new_lo"], case["new_hi"], n).astype(np.int64)
    if case["op"] == "attend":             # the bounds are those of the whole context, the new tokens in it
        lo = np.maximum(lo - new, 0)
    return lo, new


def _pitch(dim):
    return next(p for p in (32, 64, 96, 128, 192, 256) if p >= dim)


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _codes(g, shape, kind):
    """Codes as the write leaves them for values whose largest is a few deviations out."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    return (x * 35).round_().clamp_(-127, 127).to(torch.int8) if kind == "int8" else (x * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _arrays(case, seed):
    """The step's device arrays: what `plan` makes of the lengths, made here with numpy."""
    rng = np.random.default_rng(int(seed) + 31)
    start, new = _lengths(case)
    order = rng.permutation(len(start))
    start, new, bs = start[order], new[order], case["block"]
    held, after = -(-start // bs), -(-(start + new) // bs)
    wide = int(max(1, after.max()))
    blocks = int(after.sum()) + 3
    ids = rng.permutation(blocks)
    tables = np.full((len(start), wide), -1, np.int32)
    first = np.concatenate([[0], np.cumsum(after)])
    tables[np.arange(wide)[None, :] < after[:, None]] = ids[: first[-1]]
    cu = np.concatenate([[0], np.cumsum(new)])
    rows = int(cu[-1])
    seq = np.repeat(np.arange(len(start)), new)
    pos = start[seq] + np.arange(rows) - cu[seq]
    slots = tables[seq, pos // bs].astype(np.int64) * bs + pos % bs
    return dict(start=start, new=new, held=held, after=after, wide=wide, blocks=blocks, tables=tables, cu=cu, rows=rows, seq=seq, pos=pos, slots=slots, rng=rng)


def _pool(case, g, blocks):
    shape = (LAYERS, blocks, case["kv_heads"], 2, case["block"], _pitch(case["dim"]))
    codes = _codes(g, shape, case["codes"])
    codes[..., case["dim"]:] = 0
    scales = (1 / 35 if case["codes"] == "int8" else 1 / 110) * (1 + 0.2 * torch.randn(shape[:4], generator=g, device="cuda").clamp_(-3, 3))
    return codes, scales


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case, op=case["op"])
    if case["op"] == "sample":
        return s | _logits(case, seed, g)
    a = _arrays(case, seed)
    if case["op"] == "plan":
        known = np.where(np.arange(a["wide"])[None, :] < a["held"][:, None], a["tables"], -1)
        free = np.concatenate([a["tables"][b, a["held"][b]:a["after"][b]] for b in range(case["seqs"])] + [np.setdiff1d(np.arange(a["blocks"]), a["tables"])])
        cap = max(1, case["seqs"] * case["new_hi"])            # rows that the step's buffers have
        return s | dict(start=_device(a["start"]), new=_device(a["new"]), free=_device(free), tables=_device(known), cap=cap)
    codes, scales = _pool(case, g, a["blocks"])
    rows = a["rows"]
    s |= dict(codes=codes, scales=scales, tables=_device(a["tables"]), lens=_device(a["after"]), cu=_device(a["cu"]), pos=_device(a["pos"]), seq=_device(a["seq"]),
              slots=torch.from_numpy(a["slots"]).cuda(), rows=rows, most=int(a["new"].max()), longest=int((a["start"] + a["new"]).max()))
    t = TYPES[case["dtype"]]
    if case["op"] == "write":
        s["k"], s["v"] = (torch.randn(rows, case["kv_heads"], case["dim"], generator=g, device="cuda").to(t) for _ in range(2))
    else:
        s["q"] = torch.randn(rows, case["heads"], case["dim"], generator=g, device="cuda").to(t)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    # what a program keeps beside its tensors: its context, the step's arrays, the cache's handle
    from paged_infer_b200 import api
    s["api"], s["ctx"] = api, _context(api)
    if case["op"] == "sample":
        return s
    arrays = dict(tables=s["tables"], lens=s.get("lens"), cu_rows=s.get("cu"), row_seq=s.get("seq"), row_pos=s.get("pos"), slots=s.get("slots"))
    new = lambda n, t=torch.int32: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    if case["op"] == "plan":
        B, cap = case["seqs"], s["cap"]
        arrays |= dict(lens=new(B), cu_rows=new(B + 1), row_seq=new(cap), row_pos=new(cap), slots=new(cap, torch.int64), counts=new(3))
    s["plan"] = api.StepPlan(s["ctx"], block_size=case["block"], **arrays)
    if case["op"] != "plan":
        layout = api.KvLayout(LAYERS, s["codes"].shape[1], case["block"], case["kv_heads"], case["dim"])
        s["cache"] = api.KvCache8(s["ctx"], layout, codes=s["codes"], scales=s["scales"])
    if case["op"] == "attend":
        s["attention"] = api.PagedAttention8(layout, case["heads"])
        s["out"] = torch.empty_like(s["q"])
    return s


_contexts = {}                             # a server has one for each of its streams, whatever steps it runs there


def _context(api):
    """The context of torch's current stream (handle 1 is the legacy default stream)."""
    key = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream or 1
    if key not in _contexts:
        _contexts[key] = api.Context(key[0], stream=key[1])
    return _contexts[key]


def _logits(case, seed, g):
    """A model's logits: a broad heap and a few hundred likely tokens; sampling parameters as requests bring them."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.2
    likely = torch.rand(rows, vocab, generator=g, device="cuda") < 300 / max(vocab, 3000)
    x += likely * torch.randn(rows, vocab, generator=g, device="cuda").abs_() * 4
    rng = np.random.default_rng(int(seed) + 47)
    t, k, p, m = (np.empty(rows, d) for d in (np.float32, np.int32, np.float32, np.float32))
    for r in range(rows):
        kind = rng.integers(0, 6) if r else 1
        t[r] = 0 if kind == 0 else rng.uniform(0.5, 1.3)           # greedy requests among the others
        k[r] = rng.choice([1, 5, 20, 50, 200, 1000]) if kind in (2, 5) else 0
        p[r] = rng.uniform(0.6, 0.99) if kind in (1, 3, 5) else 1  # nucleus alone, or behind top-k
        m[r] = rng.uniform(0.01, 0.2) if kind in (3, 4) else 0
    u = rng.random(rows, dtype=np.float32)
    d = {n: torch.from_numpy(v).cuda() for n, v in dict(temperature=t, top_k=k, top_p=p, min_p=m, u=u).items()}
    return d | dict(logits=x.to(TYPES[case["dtype"]]), ids=torch.empty(rows, dtype=torch.int32, device="cuda"), probs=torch.empty(rows, device="cuda"))


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["op"]
    if own:
        if op == "plan":
            p = s["plan"]
            p.build(s["start"], s["new"], s["free"])
            return dict(tables=p.tables, lens=p.lens, cu_rows=p.cu_rows, row_seq=p.row_seq, row_pos=p.row_pos, slots=p.slots, counts=p.counts)
        if op == "write":
            s["cache"].write(s["plan"], s["k"], s["v"], layer=LAYER)
            return dict(codes=s["codes"], scales=s["scales"])
        if op == "attend":
            s["attention"].run_device(s["q"], s["out"], s["cache"], s["plan"], layer=LAYER, window=s["case"]["window"] or None, max_seq_rows=s["most"], max_context=s["longest"])
            return s["out"]
        s["api"].sample(s["ctx"], s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["u"], s["ids"], s["probs"])
        return dict(ids=s["ids"], probs=s["probs"])
    return {"plan": _plan, "write": _write, "attend": _attend, "sample": _sample}[op](s)


def _plan(s):
    start, new, free, bs, cap = s["start"].long(), s["new"].long(), s["free"], s["case"]["block"], s["cap"]
    B, wide = s["tables"].shape
    dev = start.device
    held, after = (start + bs - 1) // bs, (start + new + bs - 1) // bs
    need = after - held
    ahead = need.cumsum(0) - need
    col = torch.arange(wide, device=dev)[None, :]
    at = ahead[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < after[:, None])
    tables = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], s["tables"])
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    r = torch.arange(cap, device=dev)
    used = r < cu[-1]
    seq = torch.searchsorted(cu, r, right=True).clamp_(1, B) - 1
    pos = start[seq] + r - cu[seq]
    block = tables[seq, (pos // bs).clamp_(0, wide - 1)].long()
    slots = torch.where(used, block * bs + pos % bs, -1)
    counts = torch.stack([cu[-1], need.sum(), torch.zeros_like(cu[0])])
    i = torch.int32
    return dict(tables=tables, lens=after.to(i), cu_rows=cu.to(i), row_seq=torch.where(used, seq, -1).to(i), row_pos=torch.where(used, pos, -1).to(i), slots=slots, counts=counts.to(i))


def _round(y, kind):
    """To the nearest code: halves away from zero (int8), to even (e4m3)."""
    if kind == "e4m3":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn)
    t = y.trunc()
    return (t + torch.sign(y) * ((y - t).abs() >= 0.5)).clamp(-127, 127).to(torch.int8)


def _write(s):
    case, kind, bs, dim = s["case"], s["case"]["codes"], s["case"]["block"], s["case"]["dim"]
    codes, scales = s["codes"][LAYER], s["scales"][LAYER]
    x = torch.stack([s["k"], s["v"]], 2).float()                                  # [rows][kv_heads][2][dim]
    rows = x.shape[0]
    block, off = s["slots"] // bs, s["slots"] % bs
    lead = torch.ones_like(block, dtype=torch.bool)
    lead[1:] = block[1:] != block[:-1]
    unit = lead.cumsum(0) - 1                                                     # rows of one block are one unit; units behind the last repeat it
    first = torch.searchsorted(unit, torch.arange(rows, device=x.device)).clamp_(max=rows - 1)
    first = torch.where(torch.arange(rows, device=x.device) <= unit[-1], first, first[unit[-1]])
    ub, uo = block[first], off[first]                                             # its block and its first token's place
    index = unit[:, None, None].expand(-1, *x.shape[1:3])
    most = torch.zeros(x.shape[:3], device=x.device).scatter_reduce_(0, index, x.abs().amax(-1), "amax")
    most = torch.where((torch.arange(rows, device=x.device) <= unit[-1])[:, None, None], most, most[unit[-1]][None])
    old = torch.where((uo > 0)[:, None, None], scales[ub], 0.0)
    scale = torch.maximum(old, most / TOP[kind])
    safe = torch.where(scale > 0, scale, 1.0)
    kept = codes[ub].float() * old[..., None, None] / safe[..., None, None]       # [units][kv_heads][2][block][pitch]
    keep = torch.arange(bs, device=x.device)[None, :] < uo[:, None]
    b8 = codes.view(torch.int8)
    b8[ub] = torch.where(keep[:, None, None, :, None], _round(kept, kind).view(torch.int8), b8[ub])
    b8[block, :, :, off, :dim] = _round(x / safe[unit][..., None], kind).view(torch.int8)
    scales[ub] = scale
    return dict(codes=s["codes"], scales=s["scales"])


def _attend(s):
    case, bs, dim, H, KH = s["case"], s["case"]["block"], s["case"]["dim"], s["case"]["heads"], s["case"]["kv_heads"]
    B, rows, n = case["seqs"], s["rows"], s["most"]
    ids = s["tables"].long().clamp(min=0)
    kv = s["codes"][LAYER][ids].float() * s["scales"][LAYER][ids][..., None, None]  # [B][wide][kv_heads][2][block][pitch]
    k, v = (kv[:, :, :, i, :, :dim].permute(0, 2, 1, 3, 4).reshape(B, KH, 1, -1, dim) for i in (0, 1))
    cu, seq, pos = s["cu"].long(), s["seq"].long(), s["pos"].long()
    place = torch.arange(rows, device=k.device) - cu[seq]
    q = torch.zeros(B, n, H, dim, device=k.device)
    q[seq, place] = s["q"].float()
    p = torch.full((B, n), -1, device=k.device, dtype=torch.long)
    p[seq, place] = pos
    q = q.view(B, n, KH, H // KH, dim).permute(0, 2, 3, 1, 4)                        # [B][kv_heads][group][n][dim]
    score = q @ k.transpose(-1, -2) / math.sqrt(dim)
    key = torch.arange(k.shape[-2], device=k.device)
    seen = (key <= p[..., None]) & (key > p[..., None] - (case["window"] or 1 << 40)) & (key // bs < s["lens"].long()[:, None, None])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.exp(score - most)
    out = (w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, H, dim)[seq, place].to(s["q"].dtype)


def _sample(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    rows, vocab = x.shape
    most = x.amax(-1, keepdim=True)
    best = (x == most).int().argmax(-1)                                             # the lowest of equals
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    w = torch.exp((x.double() - most.double()) / t)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(-1, order)
    rank = torch.arange(vocab, device=x.device)[None, :]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    keep = (rank < k) & (ws >= s["min_p"].double()[:, None])
    ws = torch.where(keep, ws, 0.0)
    ahead = ws.cumsum(-1) - ws
    p = s["top_p"].double()[:, None]
    keep &= (ahead < p * ws.sum(-1, keepdim=True)) | (p >= 1)
    kept = torch.zeros_like(w).scatter_(-1, order, torch.where(keep, ws, 0.0))
    upto = kept.cumsum(-1)
    total = kept.sum(-1, keepdim=True)
    last = (torch.where(kept > 0, rank, -1)).amax(-1)
    ids = torch.minimum((upto <= s["u"].double()[:, None] * total).sum(-1), last)
    probs = kept.gather(-1, ids[:, None]) / total
    return dict(ids=torch.where(greedy, best, ids).int(), probs=torch.where(greedy, 1.0, probs[:, 0]).float())


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 28 * case["rows"], "flops": 4 * n}
    start, new = _lengths(case)
    rows, B, bs = int(new.sum()), case["seqs"], case["block"]
    after = -(-(start + new) // bs)
    if case["op"] == "plan":
        taken = int((after - -(-start // bs)).sum())
        return {"bytes": 8 * B + 8 * taken + 4 * (2 * B + 1) + 16 * case["seqs"] * case["new_hi"], "flops": 4 * rows}
    KH, dim, size = case["kv_heads"], case["dim"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "write":
        touched = int((after - start // bs).sum())
        n = rows * KH * 2 * dim
        return {"bytes": n * (size + 1) + touched * KH * 2 * 8 + 8 * rows, "flops": 3 * n}
    w = case["window"] or 1 << 40
    keys = np.minimum(start + new, w + new - 1)                    # read: the union of the rows' windows
    pairs = sum(int(np.minimum(np.arange(a + 1, a + n + 1), w).sum()) for a, n in zip(start.tolist(), new.tolist()))
    scales = int((after - np.maximum(start + 1 - w, 0) // bs).sum()) * KH * 2 * 4
    return {"bytes": int(keys.sum()) * KH * 2 * dim + scales + 2 * rows * case["heads"] * dim * size + 4 * int(after.sum()), "flops": 4 * pairs * case["heads"] * dim}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = _inputs(case, seed)
    if case["op"] == "sample":
        return dict(ids=None, probs=torch.tensor([_exact_prob(s, r) for r in range(case["rows"])], dtype=torch.float64))
    return _exact_write(s) if case["op"] == "write" else _exact_attend(s)


def _exact_prob(s, r):
    """Row r of the sampling, token by token in the order of their weights."""
    t, k, p, m, u = (s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    if t <= 0:
        return 1.0
    x = s["logits"][r].double().cpu().numpy()
    w = np.exp((x - x.max()) / t)
    order = np.lexsort((np.arange(x.size), -x))
    if k > 0:
        order = order[:k]
    order = order[w[order] >= m]
    if p < 1:
        sums = np.cumsum(w[order])
        order = order[: int(np.searchsorted(sums, p * sums[-1])) + 1]
    order = np.sort(order)
    sums = np.cumsum(w[order])
    return float(w[order[min(int(np.searchsorted(sums, u * sums[-1], side="right")), order.size - 1)]] / sums[-1])


def _exact_write(s):
    """The scales, block by block; codes are a rounding of their own and are compared as they are."""
    case, bs = s["case"], s["case"]["block"]
    scales = s["scales"].double().cpu().numpy()
    x = np.stack([s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy()], 2)
    most = np.abs(x).max(-1) / TOP[case["codes"]]
    block, off = (s["slots"] // bs).cpu().numpy(), (s["slots"] % bs).cpu().numpy()
    for r in range(len(block)):
        before = scales[LAYER, block[r]] if off[r] > 0 else 0.0
        scales[LAYER, block[r]] = np.maximum(before, most[r])
    return dict(codes=None, scales=torch.from_numpy(scales))


def _exact_attend(s):
    case, bs, dim, G = s["case"], s["case"]["block"], s["case"]["dim"], s["case"]["heads"] // s["case"]["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, pos, lens = (s[n].tolist() for n in ("cu", "pos", "lens"))
    for b in range(case["seqs"]):
        a, z = cu[b], cu[b + 1]
        if a == z:
            continue
        ids = s["tables"][b, : lens[b]].long()
        codes, scale = s["codes"][LAYER][ids].double(), s["scales"][LAYER][ids].double()
        p = torch.tensor(pos[a:z], device="cuda")
        for h in range(case["kv_heads"]):
            k, v = ((codes[:, h, i] * scale[:, h, i, None, None]).reshape(-1, codes.shape[-1])[:, :dim] for i in (0, 1))
            key = torch.arange(k.shape[0], device="cuda")[None, :]
            seen = key <= p[:, None]
            if case["window"]:
                seen &= key + case["window"] > p[:, None]
            for j in range(h * G, h * G + G):
                score = torch.where(seen, s["q"][a:z, j].double() @ k.T * dim ** -0.5, -math.inf)
                out[a:z, j] = torch.softmax(score, -1) @ v
    return out
