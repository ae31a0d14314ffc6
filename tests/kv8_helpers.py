"""Plain references of the device-side step over an 8-bit KV cache, in whole numbers and 64 bits (numpy; torch on the CPU for the
e4m3 rounding)."""
import numpy as np
import torch

TOP = {"int8": np.float32(127), "e4m3": np.float32(448)}
TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def pitch_of(dim):
    return next(p for p in (32, 64, 96, 128, 192, 256) if p >= dim)


def plan_reference(start, n, free, tables, block, max_rows):
    """What a plan makes, sequence by sequence: (tables, lens, cu_rows, row_seq, row_pos, slots, counts)."""
    tables = tables.copy()
    wide = tables.shape[1]
    used = missing = rows = 0
    cu, seq, pos, slots, lens = [0], [], [], [], []
    for b, (s, m) in enumerate(zip(start, n)):
        m = max(int(m), 0)
        held, after = -(-int(s) // block), -(-(int(s) + m) // block)
        for j in range(held, after):
            if j >= wide:
                missing += 1
                continue
            if used < len(free):
                tables[b, j] = free[used]
                used += 1
            else:
                tables[b, j] = -1
                missing += 1
        lens.append(min(after, wide))
        for i in range(m):
            if rows + i >= max_rows:
                break
            p = int(s) + i
            t = tables[b, p // block] if p // block < wide else -1
            seq.append(b)
            pos.append(p)
            slots.append(int(t) * block + p % block if t >= 0 else -1)
        rows += m
        cu.append(min(rows, max_rows))
    pad = max_rows - len(seq)
    return (tables, np.array(lens), np.array(cu), np.array(seq + [-1] * pad), np.array(pos + [-1] * pad), np.array(slots + [-1] * pad, np.int64),
            np.array([rows, used, missing]))


def encode(x, scale, kind):
    """Codes of f32 values under an f32 scale, as bytes."""
    if not scale > 0:
        return np.zeros(x.shape, np.uint8)
    y = (x / scale).astype(np.float32)
    if kind == "e4m3":
        return torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    t = np.trunc(y)
    return np.clip(t + np.sign(y) * (np.abs(y - t) >= 0.5), -127, 127).astype(np.int8).view(np.uint8)


def decode(codes, kind):
    t = torch.from_numpy(np.ascontiguousarray(codes))
    return t.view(TORCH[kind]).to(torch.float32).numpy()


def write_reference(codes, scales, k, v, slots, kind, block):
    """codes [blocks][heads][2][block][pitch] bytes and scales [blocks][heads][2] of one layer after a write of k, v [rows][heads][dim] (f32)."""
    codes, scales = codes.copy(), scales.copy()
    dim, r = k.shape[2], 0
    while r < len(slots):
        b = slots[r] // block if slots[r] >= 0 else -1
        if b < 0 or b >= codes.shape[0]:
            r += 1
            continue
        end = r
        while end < len(slots) and slots[end] >= 0 and slots[end] // block == b:
            end += 1
        first = slots[r] % block
        for h in range(k.shape[1]):
            for side, x in enumerate((k, v)):
                rows = x[r:end, h]
                old = scales[b, h, side] if first else np.float32(0)
                s = np.maximum(old, np.abs(rows).max() * (np.float32(1) / TOP[kind]))
                if not np.isfinite(rows).all():
                    s = np.float32(np.nan)
                if first and s != old and s == s:
                    codes[b, h, side, :first] = encode(decode(codes[b, h, side, :first], kind) * old, s, kind)
                for i in range(r, end):
                    line = np.zeros(codes.shape[-1], np.uint8)
                    line[:dim] = encode(x[i, h], s, kind)
                    codes[b, h, side, slots[i] % block] = line
                scales[b, h, side] = s
        r = end
    return codes, scales


def attention_reference(q, codes, scales, tables, lens, cu, pos, block, kind, window=0, scale=None):
    """(out, what the weights multiply at most, the largest sum of |q||k| scale) in 64 bits; q [rows][heads][dim] of one layer."""
    rows, H, dim = q.shape
    KH = codes.shape[1]
    values = decode(codes, kind).astype(np.float64)[..., :dim] * scales.astype(np.float64)[..., None, None]
    out, most, mass = np.zeros((rows, H, dim)), np.zeros((rows, H)), np.zeros((rows, H))
    scale = dim ** -0.5 if scale is None else scale
    for b in range(len(lens)):
        for r in range(cu[b], min(cu[b + 1], rows)):
            lo = max(0, pos[r] + 1 - window) if window else 0
            keys = [t for t in range(lo, pos[r] + 1) if t // block < lens[b] and 0 <= tables[b, t // block] < codes.shape[0]]
            if not keys:
                continue
            keys = np.array(keys)
            ids, off = tables[b, keys // block], keys % block
            for h in range(H):
                k, v = values[ids, h // (H // KH), 0, off], values[ids, h // (H // KH), 1, off]
                s = k @ q[r, h].astype(np.float64) * scale
                w = np.exp(s - s.max())
                out[r, h] = (w / w.sum()) @ v
                most[r, h] = np.abs(v).max()
                mass[r, h] = (np.abs(k) @ np.abs(q[r, h]).astype(np.float64)).max() * scale
    return out, most, mass


def attention_tolerance(out, most, mass, dim, dtype):
    """Per element.  Scores: both planes of an f32 query keep 22 bits (2^-22 of a product; bf16 and f16 queries are exact but for channels
    2^-14 below the largest, 2^-24 of it), f32 sums of dim terms round or truncate dim + 8 times (2^-23 each), the factor twice more, and
    2^-22 for the exponential and its argument's rounding per unit of score: delta = mass (2^-22 + (dim + 12) 2^-23), a relative error of
    every weight of up to 2 delta.  Weights: 2^-21 (two planes) or half an f16 step, 2^-11 (one plane); sums of the weights and of the
    products over tiles: below 2^-17 for the few thousand terms of a test.  Then the result's own rounding."""
    delta = mass * (2.0 ** -22 + (dim + 12) * 2.0 ** -23)
    rel = 4 * delta + (2.0 ** -21 if dtype == "f32" else 2 * 2.0 ** -11) + 2.0 ** -17
    return (most * rel)[..., None] + HALF_STEP[dtype] * np.abs(out) + 1e-30


def sample_reference(x, t, k, p, m, u):
    """(id, probability) of one row, token by token, in 64 bits; weights are whole multiples of 2^-45."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    if x.max() == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / np.float64(t)))
        w = np.where(w < (min(float(m), 1.0) if m > 0 else 0), 0.0, np.rint(w * 2.0 ** 45) * 2.0 ** -45)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[: k] if k > 0 else order
    if m > 0:
        order = order[w[order] > 0]
    if p < 1:
        sums = np.cumsum(w[order])
        order = order[: max(1, int(np.searchsorted(sums, np.float64(p) * sums[-1])) + 1)]
    order = np.sort(order)
    order = order[w[order] > 0]
    sums = np.cumsum(w[order])
    i = min(int(np.searchsorted(sums, np.float64(u) * sums[-1], side="right")), order.size - 1)
    return int(order[i]), float(w[order[i]] / sums[-1])
