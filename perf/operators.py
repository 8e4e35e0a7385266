"""Timed cases of the quantised key/value cache: writing it, reading it back and attending over it.

The cache holds the keys and values of sequences that grow step by step (the
prefix tokens of a stream of observations) in pages of 64 tokens.  One block of
a page, for one key/value head, is

    key codes | value codes | scales        (4 bits: 2048 + 2048 + 512 bytes,
                                             8 bits: 4096 + 4096 + 512 bytes)

Each token's 64 key elements (and its 64 value elements) are two groups of 32
with one scale each.  In 4 bits the scale is the group's value of largest
magnitude over -8, its magnitude rounded up to 5 significant bits; in 8 bits it
is the smallest power of two whose 127-fold reaches the largest magnitude.  A
code is x / scale rounded to the nearest integer (ties to even), in 4 bits
limited to [-8, 7] and stored plus 8.  Code times scale is a bfloat16 number
exactly.  Scales are at least 2^-100; a group with a NaN or a magnitude of 2^127
and more has the scale NaN.

A block's tokens come in tiles of 16, in the order in which a warp's matrix
fragments take them (``_fields`` and ``_address`` say where each element lies).

Attention: query row i of sequence b has the position lens[b] - q_len + i (causal)
or lens[b] - 1, and sees key j <= position if j > position - window (window > 0)
or j < sinks; a row that sees no key gives zeros.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DIM = 64


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    def append(name, batch, tokens, start, bits, heads=15, kv_heads=5):
        return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "start": start, "bits": bits,
                "heads": heads, "kv_heads": kv_heads}

    def read(name, batch, length, bits, kv_heads=5):
        return {"name": name, "op": "read", "batch": batch, "length": length, "bits": bits, "kv_heads": kv_heads}

    def attend(name, batch, rows, length, bits, causal=True, window=0, sinks=0, heads=15, kv_heads=5):
        return {"name": name, "op": "attend", "batch": batch, "rows": rows, "length": length, "bits": bits,
                "causal": causal, "window": window, "sinks": sinks, "heads": heads, "kv_heads": kv_heads}

    return [
        # one token of one robot is written: launch latency
        append("append_token", 1, 1, 113, 4),
        # the prefix (113 tokens) of a full batch of observations joins caches of uneven lengths
        append("append_prefix_batch", 256, 113, 1000, 4),
        # a long instruction or recorded episode is loaded, in the finer type
        append("append_episode_8bit", 16, 4001, 0, 8),
        # one observation's prefix goes back to bfloat16, for a layer that wants it so
        read("read_prefix", 1, 113, 4),
        # whole caches are exported, of uneven lengths
        read("read_history_batch", 32, 8001, 4),
        # text generation for one robot right after its prefix: latency
        attend("token_after_prefix", 1, 1, 114, 4),
        # one token over a very long cache: the work has to be split along it
        attend("token_long", 1, 1, 131071, 4),
        # one token each for a batch with uneven histories: memory bound
        attend("token_batch", 64, 1, 16001, 4),
        # streaming control: an instruction that stays visible and a window of recent tokens, 8 bits, more heads
        attend("token_window_8bit", 96, 1, 24001, 8, window=4096, sinks=113, heads=32, kv_heads=8),
        # the action expert's 50 rows read one observation's prefix each
        attend("chunk_prefix_batch", 256, 50, 113, 4, causal=False),
        # the action expert's 50 rows read a history of observations
        attend("chunk_history", 16, 50, 7232, 4, causal=False, window=3616, sinks=113),
        # a long chunk joins a longer history: compute bound
        attend("prefill_long", 4, 1024, 8192, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    heads, kv_heads = rng.choice([(15, 5), (15, 5), (6, 2), (32, 8), (12, 12), (8, 1)])
    bits = rng.choice([4, 4, 8])
    if op == "append":
        tokens = _log(rng, 1, 4001)
        batch = _log(rng, 1, max(1, min(256, 300000 // (tokens * kv_heads))))
        return {"op": op, "batch": batch, "tokens": tokens, "start": rng.randrange(0, 1200), "bits": bits,
                "heads": heads, "kv_heads": kv_heads}
    if op == "read":
        length = _log(rng, 16, 20000)
        batch = _log(rng, 1, max(1, min(64, 1000000 // (length * kv_heads))))
        return {"op": op, "batch": batch, "length": length, "bits": bits, "kv_heads": kv_heads}
    rows = rng.choice([1, 1, 2, 3, _log(rng, 4, 64), _log(rng, 4, 1024)])
    length = max(rows, _log(rng, 16, 130000))
    held, pairs = 3000000 // kv_heads, 400000000 // (rows * heads)  # tokens of all sequences, by memory and by work
    length = min(length, max(rows, held), max(rows, pairs))
    batch = _log(rng, 1, max(1, min(128, held // length, pairs // length)))
    window, sinks = 0, 0
    if rng.random() < 0.4:
        window, sinks = _log(rng, 33, 8192), rng.choice([0, 1, 4, 113])
    return {"op": op, "batch": batch, "rows": rows, "length": length, "bits": bits, "causal": rng.random() < 0.7,
            "window": window, "sinks": sinks, "heads": heads, "kv_heads": kv_heads}


# ---------------------------------------------------------------------------
# what a case needs
# ---------------------------------------------------------------------------
def _uneven(n, batch, least):
    """Lengths between a quarter of n and n, the first one n."""
    at = np.arange(batch, dtype=np.float64) * 0.6180339887498949 % 1.0
    return np.maximum(least, np.round(n * (1.0 - 0.75 * at))).astype(np.int64)


def _token_bytes(bits):
    return 2 * DIM * bits // 8 + 8  # codes and scales of a token's key and value, per head


def work(case):
    b, hkv = case["batch"], case["kv_heads"]
    plain = 2 * 2 * DIM * hkv  # a token's key and value in bfloat16
    held = _token_bytes(case["bits"]) * hkv
    if case["op"] == "append":  # the rows in, the cache written, and what was written read back
        return {"bytes": b * case["tokens"] * (2 * plain + 2 * held), "flops": 0}
    if case["op"] == "read":
        return {"bytes": int(_uneven(case["length"], b, 1).sum()) * held + b * case["length"] * plain, "flops": 0}
    rows = case["rows"]
    lens = _uneven(case["length"], b, rows)
    keys = pairs = 0
    for n in lens.tolist():
        pos = np.arange(n - rows, n) if case["causal"] else np.full(rows, n - 1)
        first = np.maximum(0, pos - case["window"] + 1) if case["window"] else np.zeros(rows, dtype=np.int64)
        pairs += int((pos - first + 1 + np.minimum(case["sinks"], first)).sum())
        keys += int(n - first[0] + min(case["sinks"], first[0]))
    return {"bytes": keys * held + 2 * 2 * b * rows * case["heads"] * DIM, "flops": 4 * DIM * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# plain form: quantisation and layout
# ---------------------------------------------------------------------------
def _quantise(x, bits):
    """Groups of 32 along the last dimension: (codes, scales), both float32."""
    g = x.float().unflatten(-1, (-1, 32))
    hi, lo = g.amax(-1), g.amin(-1)
    top = torch.maximum(hi, -lo)
    m, e = torch.frexp(top / 8 if bits == 4 else top / 127)
    m = torch.ceil(m * 32) / 32 if bits == 4 else torch.where(m > 0.5, 1.0, 0.5)
    d = torch.ldexp(m, e).clamp_min(2.0 ** -100)
    if bits == 4:
        d = torch.where(hi > -lo, -d, d)
    d = torch.where(top < 2.0 ** 127, d, torch.nan)
    code = torch.round(g / d[..., None])
    code = code.clamp(-8, 7) if bits == 4 else code
    return code.flatten(-2), d


def _fields(bits, keys):
    """The shape of a tile's code bytes, and the order that makes them (tokens, dims) of one tile."""
    # q, b, c / r: token 4q + b + 2c, or 4q + r;  h: group;  t, g: 8 or 4 elements of it;  w: 4 of 8;
    # s, u: a word's bytes;  n: a byte's half.  Elements of a word: 4u + 2n + s (4 bits), 2u + s (8 bits)
    if bits == 4 and keys:  # q b t c h s u n -> q c b | h t u n s
        return (4, 2, 4, 2, 2, 2, 2, 2), (0, 3, 1, 4, 2, 6, 7, 5)
    if bits == 4:  # q g r s u n -> q r | u g n s
        return (4, 8, 4, 2, 2, 2), (0, 2, 4, 1, 5, 3)
    if keys:  # h q b t c w s u -> q c b | h t w u s
        return (2, 4, 2, 4, 2, 2, 2, 2), (1, 4, 2, 0, 3, 5, 7, 6)
    return (2, 4, 8, 4, 2, 2), (1, 3, 0, 2, 5, 4)  # h q g r s u -> q r | h g u s


def _blocks(k, v, bits):
    """Keys and values [pages, 64, heads, 64] as blocks [pages, heads, bytes]."""
    pages, _, heads, _ = k.shape
    parts, scales = [], []
    for x, keys in ((k, True), (v, False)):
        code, d = _quantise(x, bits)
        code = torch.nan_to_num(code).to(torch.int16)
        code = (code + 8 if bits == 4 else code & 255).to(torch.uint8)
        shape, order = _fields(bits, keys)
        code = code.view(pages, 4, 16, heads, DIM).permute(0, 3, 1, 2, 4)
        code = code.reshape(pages, heads, 4, *(shape[i] for i in order))
        code = code.permute(0, 1, 2, *(3 + order.index(i) for i in range(len(order))))
        if bits == 4:
            code = code[..., 0] | code[..., 1] << 4
        parts.append(code.reshape(pages, heads, -1))
        scales.append(d.to(torch.bfloat16))
    s = torch.cat(scales, -1)  # [pages, 64, heads, 4]
    s = s.view(pages, 4, 4, 2, 2, heads, 4).permute(0, 5, 1, 2, 4, 3, 6)  # token 4q + 2c + b in the order q b c
    parts.append(s.reshape(pages, heads, -1).contiguous().view(torch.uint8))
    return torch.cat(parts, -1)


def _values(pool, table, bits, keys):
    """Keys or values of the pages in table [b, n] as float32 [b, heads, n * 64, 64]."""
    x = pool[table.long()]
    b, n, heads, _ = x.shape
    size = PAGE * DIM * bits // 8
    code = x[..., :size] if keys else x[..., size:2 * size]
    shape, order = _fields(bits, keys)
    if bits == 4:
        code = torch.stack((code & 15, code >> 4), -1).float() - 8
    else:
        code = code.contiguous().view(torch.int8).float()
    code = code.reshape(b, n, heads, 4, *shape).permute(0, 2, 1, 3, *(4 + i for i in order))
    d = x[..., 2 * size:].contiguous().view(torch.bfloat16).view(b, n, heads, 4, 4, 2, 2, 4)
    d = d[..., :2] if keys else d[..., 2:]
    d = d.permute(0, 2, 1, 3, 4, 6, 5, 7).reshape(b, heads, n * PAGE, 2, 1)
    return (code.reshape(b, heads, n * PAGE, 2, 32) * d).flatten(-2)


def _append(pool, table, bits, k, v, start):
    """Writes k, v [b, n, heads, 64] at the positions start[b] + i, page by page as they are held."""
    b, n, heads, _ = k.shape
    pages = (n + PAGE - 2) // PAGE + 1  # pages that n tokens can touch
    first = (start // PAGE).long()
    at = first[:, None] + torch.arange(pages, device=k.device)
    last = table.shape[1] - 1
    page = table.gather(1, at.clamp_max(last)).long()
    old = pool[page]
    token = (at * PAGE)[..., None] + torch.arange(PAGE, device=k.device) - start[:, None, None]  # [b, pages, 64]
    new = (token >= 0) & (token < n) & (at <= last)[..., None]
    row = token.clamp(0, n - 1).flatten(1)[..., None, None].expand(-1, -1, heads, DIM)
    kk, vv = (x.gather(1, row).view(b * pages, PAGE, heads, DIM) for x in (k, v))
    made = _blocks(kk, vv, bits).view_as(old)
    ones = torch.where(new[..., None, None], 255, 0).to(torch.uint8)
    mask = _mask(ones.view(b * pages, PAGE).expand(heads, -1, -1), bits).view(heads, b, pages, -1).permute(1, 2, 0, 3)
    live = (at <= last).flatten()
    pool[page.flatten()[live]] = torch.where(mask > 0, made, old).flatten(0, 1)[live]


def _mask(token, bits):
    """[heads, pages, 64] per token as [heads, pages, bytes] per byte of a block."""
    out = []
    for keys in (True, False):
        shape, order = _fields(bits, keys)
        x = token.view(*token.shape[:2], 4, 16, 1).expand(-1, -1, -1, -1, DIM)
        x = x.reshape(*token.shape[:2], 4, *(shape[i] for i in order))
        x = x.permute(0, 1, 2, *(3 + order.index(i) for i in range(len(order))))
        out.append((x[..., 0] if bits == 4 else x).flatten(2))
    s = token.view(*token.shape[:2], 4, 4, 2, 2).transpose(-1, -2)
    out.append(s.flatten(2).repeat_interleave(8, -1))
    return torch.cat(out, -1)


def _read(pool, table, bits, start, count, n):
    """Tokens start[b] .. start[b] + n of each sequence as bfloat16 [b, n, heads * 64], zeros from count[b] on."""
    out = []
    for keys in (True, False):
        x = _values(pool, table, bits, keys)
        b, heads, have, _ = x.shape
        i = torch.arange(n, device=x.device)
        at = (start[:, None] + i).clamp_max(have - 1).long()
        x = x.gather(2, at[:, None, :, None].expand(-1, heads, -1, DIM))
        x = torch.where((i < count[:, None])[:, None, :, None], x, 0.0)
        out.append(x.transpose(1, 2).flatten(2).to(torch.bfloat16))
    return out


def _attend(pool, table, bits, q, lens, causal, window, sinks):
    """q [b, rows, heads, 64] over the cache: bfloat16 [b, rows, heads, 64]."""
    k, v = _values(pool, table, bits, True), _values(pool, table, bits, False)
    b, rows, heads, _ = q.shape
    hkv, n = k.shape[1], k.shape[2]
    x = q.float().view(b, rows, hkv, heads // hkv, DIM).permute(0, 2, 3, 1, 4).flatten(2, 3)
    j = torch.arange(n, device=q.device)
    held = j < lens[:, None]
    k, v = (torch.where(held[:, None, :, None], y, 0.0) for y in (k, v))
    s = torch.matmul(x, k.transpose(-1, -2)) * 0.125
    pos = lens[:, None] - rows + torch.arange(rows, device=q.device) if causal else lens[:, None].expand(-1, rows) - 1
    seen = j <= pos[..., None]
    if window:
        seen = seen & ((j > pos[..., None] - window) | (j < sinks))
    seen = seen[:, None, None]
    s = torch.where(seen, s.view(b, hkv, heads // hkv, rows, n), -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38))
    p = torch.where(seen, p, 0.0)
    o = torch.matmul(p.flatten(2, 3), v).view(b, hkv, heads // hkv, rows, DIM)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total == 0, 0.0, o / total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, rows, heads, DIM).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _keys_values(gen, shape, heads, dev):
    """Keys and values as projections give them: a few strong key channels, tokens of uneven size."""
    strong = 1 + 6 * (torch.rand(heads, DIM, generator=gen, device=dev) > 0.94)
    k = torch.randn(*shape, heads, DIM, generator=gen, device=dev, dtype=torch.bfloat16) * strong.to(torch.bfloat16)
    v = torch.randn(*shape, heads, DIM, generator=gen, device=dev, dtype=torch.bfloat16)
    size = torch.rand(*shape, heads, 1, generator=gen, device=dev).add_(0.5).to(torch.bfloat16)
    return k, v * size


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    b, hkv, bits = case["batch"], case["kv_heads"], case["bits"]
    if case["op"] == "append":
        start = torch.from_numpy(_uneven(case["start"], b, 0)).to(dev, torch.int32)
        need = case["start"] + case["tokens"]
    else:
        lens = _uneven(case["length"], b, case.get("rows", 1))
        start, need = torch.zeros(b, dtype=torch.int32, device=dev), case["length"]
    per_seq = -(-need // PAGE)
    pages = b * per_seq
    table = torch.randperm(pages, generator=gen, device=dev).view(b, per_seq).to(torch.int32)  # pages in no order
    state = {"case": dict(case), "table": table, "start": start}
    if case["op"] == "append":
        # a used pool: what the pages held before is not zero
        size = 2 * PAGE * DIM * bits // 8 + 512
        state["pool"] = torch.randint(0, 256, (pages, hkv, size), generator=gen, device=dev, dtype=torch.uint8)
        # the rows lie in a layer's joint output [rows, Q | K | V]
        width = (case["heads"] + 2 * hkv) * DIM
        rows = torch.empty(b * case["tokens"], width, dtype=torch.bfloat16, device=dev)
        k, v = _keys_values(gen, (b * case["tokens"],), hkv, dev)
        rows[:, -2 * hkv * DIM:-hkv * DIM] = k.flatten(1)
        rows[:, -hkv * DIM:] = v.flatten(1)
        state["k"], state["v"] = rows[:, -2 * hkv * DIM:-hkv * DIM], rows[:, -hkv * DIM:]
        state["count"] = torch.full((b,), case["tokens"], dtype=torch.int32, device=dev)
    else:
        pool = torch.empty(pages, hkv, 2 * PAGE * DIM * bits // 8 + 512, dtype=torch.uint8, device=dev)
        for at in range(0, pages, 2048):
            n = min(2048, pages - at)
            pool[at:at + n] = _blocks(*_keys_values(gen, (n, PAGE), hkv, dev), bits)
        state["pool"], state["count"] = pool, torch.from_numpy(lens).to(dev, torch.int32)
        if case["op"] == "attend":
            state["q"] = torch.randn(b, case["rows"], case["heads"], DIM, generator=gen, device=dev,
                                     dtype=torch.bfloat16)
    if own:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "vla-to-npu_b200"))
        from vla_b200.kvcache import KVCache
        state["cache"] = KVCache.wrap(state["pool"], table, kv_heads=hkv, bits=bits)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    b, hkv, bits = case["batch"], case["kv_heads"], case["bits"]
    if own:
        cache = state["cache"]
        if case["op"] == "append":
            cache.append(state["k"], state["v"], state["start"], case["tokens"])
            return cache.read(case["tokens"], state["count"], start=state["start"])
        if case["op"] == "read":
            return cache.read(case["length"], state["count"])
        return cache.attend(state["q"], state["count"], causal=case["causal"], window=case["window"],
                            sinks=case["sinks"])
    pool, table = state["pool"], state["table"]
    if case["op"] == "append":
        k, v = (x.unflatten(0, (b, -1)).unflatten(-1, (hkv, DIM)) for x in (state["k"], state["v"]))
        _append(pool, table, bits, k, v, state["start"])
        return _read(pool, table, bits, state["start"], state["count"], case["tokens"])
    if case["op"] == "read":
        return _read(pool, table, bits, state["start"], state["count"], case["length"])
    return _attend(pool, table, bits, state["q"], state["count"], case["causal"], case["window"], case["sinks"])


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _address(bits, keys):
    """Byte and shift of the code of (token, dim) in a block, and the byte of a token's first scale."""
    tok, dim = np.arange(PAGE)[:, None], np.arange(DIM)[None, :]
    tile, tok = tok // 16, tok % 16
    group, e = dim // 32, dim % 32
    shift = 0 * (tok + dim)
    if bits == 4:
        at = tile * 512
        if keys:  # 16 bytes: 8 elements of each group, for a token and the second next
            at = at + (2 * (tok // 4) + tok % 2) * 64 + e // 8 * 16 + tok % 4 // 2 * 8 + group * 4
            e = e % 8
        else:  # 4 bytes: 4 elements of each group
            at = at + tok // 4 * 128 + e // 4 * 16 + tok % 4 * 4
            e = e % 4 + 4 * group
        nibble = e // 2 + 4 * (e % 2)  # a word's even elements come first
        at, shift = at + nibble // 2, shift + 4 * (nibble % 2)
    else:
        at = tile * 1024 + group * 512
        if keys:  # 16 bytes: 8 elements of one group, for a token and the second next
            at = at + (2 * (tok // 4) + tok % 2) * 64 + e // 8 * 16 + tok % 4 // 2 * 8 + e % 8 // 4 * 4
        else:  # 4 bytes: 4 elements
            at = at + tok // 4 * 128 + e // 4 * 16 + tok % 4 * 4
        at = at + np.array([0, 2, 1, 3])[e % 4]
    size = PAGE * DIM * bits // 8
    first = 2 * size + tile * 128 + (2 * (tok // 4) + tok % 2) * 16 + tok % 4 // 2 * 8 + (0 if keys else 4)
    return at + (0 if keys else size), shift, first[:, 0]


def _decode(block, bits, keys):
    """Blocks [n, bytes] of one head as float64 [n * 64, 64]."""
    at, shift, first = (torch.from_numpy(x).to(block.device) for x in _address(bits, keys))
    code = block[:, at].to(torch.int64) >> shift
    code = code % 16 - 8 if bits == 4 else (code + 128) % 256 - 128
    d = block[:, first[:, None] + torch.arange(4, device=block.device)].contiguous().view(torch.bfloat16).double()
    return (code.double() * d.repeat_interleave(32, -1)).flatten(0, 1)


def _rounded(x, bits):
    """What the cache holds for x [..., 64], from the definition in float64."""
    g = x.double().reshape(*x.shape[:-1], 2, 32)
    top = g.abs().amax(-1)
    least = torch.tensor(2.0 ** -100, dtype=torch.float64, device=x.device)
    want = torch.maximum(top / (8 if bits == 4 else 127), least)
    unit = torch.exp2(torch.floor(torch.log2(want)))
    unit = torch.where(unit > want, unit / 2, torch.where(2 * unit <= want, 2 * unit, unit))  # 2^floor(log2), exactly
    if bits == 4:
        d = torch.maximum(torch.ceil(want / unit * 16) * unit / 16, least)
        d = torch.where((g == top[..., None]).any(-1) & ~(g == -top[..., None]).any(-1), -d, d)
        code = torch.round(g / d[..., None]).clamp(-8, 7)
    else:
        d = torch.where(unit < want, 2 * unit, unit)
        code = torch.round(g / d[..., None])
    bad = ~(top < 2.0 ** 127)
    return torch.where(bad[..., None], torch.nan, code * d[..., None]).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    b, hkv, bits = case["batch"], case["kv_heads"], case["bits"]
    if case["op"] == "append":
        return [_rounded(x.reshape(b, case["tokens"], hkv, DIM), bits).flatten(2) for x in (state["k"], state["v"])]
    pool, table, lens = state["pool"], state["table"].long(), state["count"].tolist()
    if case["op"] == "read":
        out = []
        for keys in (True, False):
            x = torch.zeros(b, case["length"], hkv, DIM, dtype=torch.float64, device=pool.device)
            for i, n in enumerate(lens):
                for h in range(hkv):
                    x[i, :n, h] = _decode(pool[table[i], h], bits, keys)[:n]
            out.append(x.flatten(2))
        return out
    q, rows, heads = state["q"].double(), case["rows"], case["heads"]
    out = torch.zeros(b, rows, heads, DIM, dtype=torch.float64, device=pool.device)
    for i, n in enumerate(lens):
        first = 0
        if case["window"]:  # what no row sees is left out
            first = max(0, (n - rows if case["causal"] else n - 1) - case["window"] + 1) // PAGE
        pages = torch.arange(-(-n // PAGE), device=pool.device)
        pages = pages[(pages >= first) | (pages * PAGE < case["sinks"])]
        key = (pages[:, None] * PAGE + torch.arange(PAGE, device=pool.device)).flatten()
        for row in range(0, rows, 256):
            part = slice(row, min(rows, row + 256))
            pos = torch.arange(part.start, part.stop, device=pool.device) + (n - rows)
            pos = pos if case["causal"] else torch.full_like(pos, n - 1)
            hidden = key[None] > pos[:, None]
            if case["window"]:
                hidden |= (key[None] <= pos[:, None] - case["window"]) & (key[None] >= case["sinks"])
            for h in range(hkv):
                k, v = (_decode(pool[table[i][pages], h], bits, keys)[key < n] for keys in (True, False))
                for head in range(h * heads // hkv, (h + 1) * heads // hkv):
                    s = (q[i, part, head] @ k.T / 8).masked_fill(hidden[:, key < n], -math.inf)
                    out[i, part, head] = torch.softmax(s, -1) @ v
    return out
