"""Plain 64-bit restatement of the quantised key/value cache: its rounding, the
order of a block's bytes, and attention over it.  numpy, element by element where
that is clearest; written from the format's definition (include/vla_b200.h), not
from the kernels."""
import math

import numpy as np

PAGE = 64
DIM = 64
GROUP = 32


def bf16_bits(x):
    """uint16 bits of float64 values that bf16 holds exactly (NaN as 0x7FC0)."""
    u = np.asarray(x, dtype=np.float32).view(np.uint32)
    assert not np.any((u & 0xFFFF)[~np.isnan(np.asarray(x))]), "not a bf16 number"
    return np.where(np.isnan(np.asarray(x)), 0x7FC0, u >> 16).astype(np.uint16)


def group_scale(g, bits):
    """Scale of one group of 32 values."""
    top = max(abs(float(v)) if not math.isnan(v) else math.inf for v in g)
    if not top < 2.0 ** 127:
        return math.nan
    if bits == 4:
        if top == 0:
            return 2.0 ** -100
        unit = 2.0 ** (math.frexp(top / 8)[1] - 5)  # the last place of 5 significant bits
        d = max(math.ceil(top / 8 / unit) * unit, 2.0 ** -100)
        negative = any(v == top for v in g) and not any(v == -top for v in g)
        return -d if negative else d
    e = -100
    while 127 * 2.0 ** e < top:
        e += 1
    return 2.0 ** e


def quantise(x, bits):
    """x [..., 64] -> integer codes [..., 64] and scales [..., 2] (float64)."""
    x = np.asarray(x, dtype=np.float64)
    flat = x.reshape(-1, GROUP)
    codes, scales = np.zeros(flat.shape, dtype=np.int64), np.zeros(len(flat))
    for i, g in enumerate(flat):
        d = scales[i] = group_scale(g, bits)
        if not math.isnan(d):
            c = np.rint(g / d)  # ties to even
            codes[i] = np.clip(c, -8, 7) if bits == 4 else c
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], 2)


def held(x, bits):
    """What the cache stands for once x [..., 64] is written."""
    c, s = quantise(x, bits)
    return (c.reshape(*c.shape[:-1], 2, GROUP) * s[..., None]).reshape(c.shape)


def block_bytes(bits):
    return 2 * PAGE * DIM * bits // 8 + PAGE * 8


def code_place(bits, keys, token, dim):
    """(byte, shift) of an element's code in a block."""
    tile, tok = divmod(token, 16)
    group, e = divmod(dim, GROUP)
    quad, r = divmod(tok, 4)
    base = (0 if keys else PAGE * DIM * bits // 8) + tile * 16 * DIM * bits // 8
    if bits == 4:
        if keys:  # 16 bytes: (token, group) words of 8 elements for tokens b and b + 2
            lane, inner = divmod(e, 8)
            word = base + (2 * quad + r % 2) * 64 + lane * 16 + (r // 2) * 8 + group * 4
        else:  # 16 bytes: a word of 4 + 4 elements for each of 4 tokens
            lane, inner = divmod(e, 4)
            inner += 4 * group
            word = base + quad * 128 + lane * 16 + r * 4
        bit = 4 * (inner // 2) + 16 * (inner % 2)
        return word + bit // 8, bit % 8
    base += group * 512
    if keys:
        lane, inner = divmod(e, 8)
        word = base + (2 * quad + r % 2) * 64 + lane * 16 + (r // 2) * 8 + inner // 4 * 4
    else:
        lane, inner = divmod(e, 4)
        word = base + quad * 128 + lane * 16 + r * 4
    return word + (0, 2, 1, 3)[inner % 4], 0


def scale_place(bits, keys, token, group):
    """Byte of a group's scale (2 bytes, little endian)."""
    tile, tok = divmod(token, 16)
    quad, r = divmod(tok, 4)
    return (2 * PAGE * DIM * bits // 8 + tile * 128 + (2 * quad + r % 2) * 16 + (r // 2) * 8
            + (0 if keys else 4) + 2 * group)


def write_token(block, bits, token, k, v):
    """Writes one token's keys and values [64] into a block (uint8 array)."""
    for keys, x in ((True, k), (False, v)):
        codes, scales = quantise(x, bits)
        for dim in range(DIM):
            at, shift = code_place(bits, keys, token, dim)
            if bits == 4:
                block[at] = block[at] & (0xF0 >> shift) | (int(codes[dim]) + 8) << shift
            else:
                block[at] = int(codes[dim]) & 0xFF
        for group, raw in enumerate(bf16_bits(scales)):
            at = scale_place(bits, keys, token, group)
            block[at:at + 2] = (raw & 0xFF, raw >> 8)


def sees(position, key, window, sinks):
    return key <= position and (window == 0 or key > position - window or key < sinks)


def attend(q, k, v, lens, causal=True, window=0, sinks=0, scale=0.125, q_len=None):
    """q [B, Lq, Hq, 64] over the held keys and values k, v [B][tokens, Hkv, 64].
    Returns the output, and the parts of its error bound: sum_j p_j |v_j| per
    element and the largest scale * sum_d |q_d k_jd| per row."""
    q = np.asarray(q, dtype=np.float64)
    B, Lq, Hq, _ = q.shape
    out, mag, big = np.zeros_like(q), np.zeros_like(q), np.zeros((B, Lq, Hq, 1))
    for b in range(B):
        n, ql = int(lens[b]), Lq if q_len is None else int(q_len[b])
        Hkv = k[b].shape[1]
        for i in range(ql):
            pos = n - ql + i if causal else n - 1
            at = [j for j in range(min(n, pos + 1)) if sees(pos, j, window, sinks)]
            if not at:
                continue
            for h in range(Hq):
                kk, vv = k[b][at, h * Hkv // Hq], v[b][at, h * Hkv // Hq]
                s = scale * kk @ q[b, i, h]
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h], mag[b, i, h] = p @ vv, p @ np.abs(vv)
                big[b, i, h] = (scale * np.abs(kk) @ np.abs(q[b, i, h])).max()
    return out, mag, big


def attend_bound(out, mag, big):
    """Largest error of an element.  bf16 has 8 significant bits, so a rounding to
    it is off by at most 2^-8 of the number: the output once, and each
    probability with its value scale once.  64-term fp32 scores are off by 2^-18
    of sum |q k|, in numerator and denominator; the exponential and the fp32 sums
    by 2^-18.  A probability below fp32's 2^-126 of the largest counts as 0: with
    up to 2^13 keys of magnitude 2^13 that is 2^-100."""
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -8 + 2.0 ** -17 * big + 2.0 ** -18) * mag + 2.0 ** -100
