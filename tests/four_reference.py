"""The four-bit operators in 64 bits (numpy and torch on the CPU), written from the format's definition."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def toward(v, way):
    """fp64 values to fp16's grid, downwards (-1) or upwards (1)."""
    h = np.array(v, np.float16)
    off = h.astype(np.float64) > v if way < 0 else h.astype(np.float64) < v
    h[off] = np.nextafter(h[off], np.float16(way * np.inf))
    return h


def quantize(rows, group):
    """(codes [..][k], scales [..][groups][2]) of fp64 rows [..][k]; the last group of a row may be short."""
    rows = np.clip(np.where(np.isnan(rows), 0.0, rows), -65504.0, 65504.0)
    k = rows.shape[-1]
    codes, scales = np.zeros(rows.shape, np.uint8), np.zeros((*rows.shape[:-1], -(-k // group), 2), np.float16)
    for i in range(scales.shape[-2]):
        g = rows[..., i * group:(i + 1) * group]
        low = toward(g.min(-1), -1)
        scale = toward((g.max(-1) - low.astype(np.float64)) / 15.0, 1)
        step = scale.astype(np.float64)
        q = (g - low.astype(np.float64)[..., None]) / np.where(step > 0, step, 1.0)[..., None]
        codes[..., i * group:(i + 1) * group] = np.where(step[..., None] > 0, np.clip(np.rint(q), 0, 15), 0)
        scales[..., i, 0], scales[..., i, 1] = scale, low
    return codes, scales


def pack(codes):
    """[..][k] codes to bytes [..][ceil(k/32)*16]."""
    k = codes.shape[-1]
    full = np.zeros((*codes.shape[:-1], -(-k // 32) * 32), np.uint8)
    full[..., :k] = codes
    return full[..., 0::2] | full[..., 1::2] << 4


def unpack(packed, k):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], 2 * packed.shape[-1])[..., :k]


def values(packed, scales, group, k, centre=0):
    """(value, |low + centre * scale| + scale * |code - centre|) of packed rows, fp64 [..][k]: the second is what rounding errors are
    relative to (values of attention, and all of fp32 calls, are summed around the middle, centre 8)."""
    codes = unpack(np.asarray(packed), k).astype(np.float64)
    s, low = (np.repeat(np.asarray(scales)[..., i].astype(np.float64), group, -1)[..., :k] for i in (0, 1))
    return low + s * codes, np.abs(low + centre * s) + np.abs(s) * np.abs(codes - centre)


def find(table, lengths, counts, tokens, page, pages):
    """{(sequence, row): (page, place)} of the rows that stand for a token."""
    found = {}
    for b, length in enumerate(lengths):
        count = tokens if counts is None else counts[b]
        for i in range(min(tokens, count)):
            at = length - count + i
            if 0 <= at < len(table[b]) * page and 0 <= table[b][at // page] < pages:
                found[b, i] = (table[b][at // page], at % page)
    return found


def attend(q, k_packed, k_scales, v_packed, v_scales, table, lengths, counts, group, scale, window, centre=0):
    """(out, lse, bound) in fp64: [batch][tokens][heads][dim], [batch][tokens][heads], and per output the sum of weights times the values'
    magnitudes, which errors of weights are relative to, with the largest magnitude of a score of the row."""
    batch, tokens, heads, dim = q.shape
    pages, kv_heads, page = k_packed.shape[:3]
    out, lse = np.zeros(q.shape), np.full(q.shape[:3], -math.inf)
    size, score = np.zeros(q.shape), np.zeros(q.shape[:3])
    share = heads // kv_heads
    for b in range(batch):
        count = tokens if counts is None else counts[b]
        there = [j for j in range(min(lengths[b], len(table[b]) * page)) if 0 <= table[b][j // page] < pages]
        at = (np.array([table[b][j // page] for j in there], int), np.array([j % page for j in there], int))
        where = np.array(there, int)
        for h in range(kv_heads):
            k, k_size = values(k_packed[at[0], h, at[1]], k_scales[at[0], h, at[1]], group, dim, centre)
            v, v_size = values(v_packed[at[0], h, at[1]], v_scales[at[0], h, at[1]], group, dim, 8)
            for i in range(min(tokens, count)):
                own = lengths[b] - count + i
                seen = (where <= own) & ((where > own - window) if window else True)
                if not seen.any():
                    continue
                for x in range(h * share, (h + 1) * share):
                    s = scale * (k[seen] @ q[b, i, x])
                    top = s.max()
                    w = np.exp(s - top)
                    out[b, i, x] = w @ v[seen] / w.sum()
                    lse[b, i, x] = top + math.log(w.sum())
                    size[b, i, x] = w @ v_size[seen] / w.sum()
                    score[b, i, x] = abs(scale) * (k_size[seen] @ np.abs(q[b, i, x])).max()
    return out, lse, size, score
