"""Inputs on which f32 attention over the 8-bit cache shows whether queries and weights are held in one f16 plane (11 bits) or in two (22).

`query`: every query channel is 1 +- 2^-12, which f16 rounds to 1; keys +-112 so that the rounded channels cancel and scores are
made of the residues alone, +-0.8 by turns.  `weight`: scores 0 and ln(w) by turns, with 2^7 w halfway between two numbers of f16, and
values +-96.  All sums of products are exact in f32 (multiples of 2^-9 below 2^12), so that what a result may be off is two planes'
rounding of a weight (2^-21), the exponential's and its argument's (14 x 2^-23 for scores below 1) and sums over tiles (2^-17)."""
import numpy as np

from kv8_helpers import attention_tolerance


def plane_case(which, dim, tokens, rows, heads, kv_heads):
    """(q [rows][heads][dim], codes as values [tokens][kv_heads][2][dim], K scale, V scale); softmax scale dim ** -0.5."""
    codes = np.zeros((tokens, kv_heads, 2, dim), np.float32)
    turn = np.where(np.arange(tokens) % 2 == 0, 1.0, -1.0)[:, None, None]
    half = np.where(np.arange(dim) % 2 == 0, 1.0, -1.0)
    codes[:, :, 1] = 96 * turn
    q = np.ones((rows, heads, dim), np.float32)
    if which == "query":
        q += np.float32(2.0 ** -12) * half.astype(np.float32)
        codes[:, :, 0] = 112 * half * turn
        k_scale = 0.8 * 2.0 ** 12 / (dim * 112 * dim ** -0.5)
    else:
        q[..., 1:] = 0
        codes[:, :, 0, 0] = np.where(turn[:, :, 0] < 0, -112, 0)
        k_scale = -np.log(89.59375 / 128) / (112 * dim ** -0.5)      # f16 has 89.5625 and 89.625
    return q, codes, np.float32(k_scale), np.float32(2.0 ** -5)


def plane_reference(q, codes, k_scale, v_scale, pos, planes=None):
    """(out, sum of weight x |v|) in 64 bits; with `planes`, queries and weights as that many f16 planes hold them."""
    def held(x):
        if planes is None:
            return x
        hi = x.astype(np.float16).astype(np.float64)
        return hi if planes == 1 else hi + (x - hi).astype(np.float16).astype(np.float64)

    rows, heads, dim = q.shape
    group = heads // codes.shape[1]
    out, weighed = np.zeros(q.shape), np.zeros((rows, heads))
    seen = np.arange(len(codes))[None] <= pos[:, None]
    for h in range(heads):
        k, v = codes[:, h // group, 0].astype(np.float64), codes[:, h // group, 1].astype(np.float64) * np.float64(v_scale)
        s = held(q[:, h].astype(np.float64)) @ k.T * np.float64(k_scale) * dim ** -0.5
        s[~seen] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True)) * 2.0 ** 7
        out[:, h], weighed[:, h] = held(w) @ v / w.sum(1, keepdims=True), (w @ np.abs(v).max(1)) / w.sum(1)
    return out, weighed


def plane_tolerance(want, weighed):
    return attention_tolerance(want, weighed, np.ones(weighed.shape), 2, "f32")
