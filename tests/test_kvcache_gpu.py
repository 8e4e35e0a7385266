"""The quantised key/value cache on the GPU against its 64-bit restatement
(oracle/kvcache_ref.py): bytes and values bit for bit, attention within the bound
that its roundings give (oracle.kvcache_ref.attend_bound)."""
import numpy as np
import pytest
import torch

from oracle import kvcache_ref as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rows_like(gen, *shape):
    """bf16 rows with uneven sizes and a few strong channels."""
    x = torch.randn(*shape, generator=gen) * (0.25 + 4 * torch.rand(*shape[:-1], 1, generator=gen))
    return (x * (1 + 5 * (torch.rand(shape[-1], generator=gen) > 0.9))).to(BF16)


def garbage(pool, gen):
    """What unwritten memory may hold: any bytes, among the scales NaN and infinities."""
    pool.copy_(torch.randint(0, 256, pool.shape, generator=gen, dtype=torch.uint8))
    pool[..., -512:].view(torch.int16)[..., ::3] = 0x7FC0
    pool[..., -512:].view(torch.int16)[..., 1::7] = 0x7F80


def make(batch, max_len, kv_heads, bits, seed=0, layers=1, spare=0):
    """A cache with shuffled pages in used memory."""
    from vla_b200.kvcache import KVCache
    gen = torch.Generator().manual_seed(seed)
    per = -(-max_len // 64)
    cache = KVCache(batch, max_len, kv_heads=kv_heads, layers=layers, bits=bits, pages=batch * per + spare)
    cache.table.copy_(torch.randperm(batch * per + spare, generator=gen)[:batch * per].view(batch, per))
    garbage(cache.pool, gen)
    return cache, gen


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def f64(x):
    return x.detach().float().cpu().double().numpy()


def check_clean():
    from vla_b200 import device as dev
    dev.sync_check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kv_heads,n,starts,counts", [
    (1, 1, [0], None),
    (5, 1, [63, 64, 113], None),
    (2, 70, [0, 61, 5], [70, 69, 1]),
    (3, 131, [1, 2, 3], [0, 131, 64]),
])
def test_append_writes_the_bytes_and_nothing_else(cuda, bits, kv_heads, n, starts, counts):
    B = len(starts)
    cache, gen = make(B, max(starts) + n, kv_heads, bits, spare=2)
    want = cache.pool[0].cpu().numpy().copy()
    k, v = rows_like(gen, B, n, kv_heads * 64), rows_like(gen, B, n, kv_heads * 64)
    cache.append(k.cuda(), v.cuda(), i32(starts), n, count=None if counts is None else i32(counts))
    table = cache.table.cpu().numpy()
    for b in range(B):
        for i in range(n if counts is None else counts[b]):
            at = starts[b] + i
            for h in range(kv_heads):
                R.write_token(want[table[b, at // 64], h], bits, at % 64, f64(k)[b, i, 64 * h:64 * h + 64],
                              f64(v)[b, i, 64 * h:64 * h + 64])
    np.testing.assert_array_equal(cache.pool[0].cpu().numpy(), want)
    check_clean()


def special_rows():
    """Groups where a rounding can go wrong, as bf16 [n, 64] rows."""
    inf, nan = float("inf"), float("nan")
    rows = []
    for base in ([0.0], [1.0], [-1.0], [1.0, -1.0], [3.0, -3.0, 0.5], [2.0 ** -133, 0.0], [-2.0 ** -126], [2.0 ** -98],
                 [2.0 ** 126], [-1.99 * 2.0 ** 126, 2.0 ** 120], [2.0 ** 127], [-3.38e38, 1.0], [inf, 1.0], [-inf],
                 [nan, 2.0], [127.0, 63.5, 0.5, 1.5], [254.0, 1.0, 3.0], [128.0, 0.5], [-0.0, 0.0]):
        rows.append((base * 32)[:32] + [0.75, -0.25] * 16)
    # every tie of 4-bit codes, for the 16 significands of a scale and both signs of the peak
    for m in range(16, 32):
        for sign in (1, -1):
            d = m / 16
            ties = [(c + 0.5) * d for c in range(-8, 8)]
            rows.append([sign * 8 * d] + ties + [c * d for c in range(-7, 8)] + [-x for x in ties] + ties)
    x = torch.tensor(rows, dtype=torch.float64).to(BF16)
    assert x.shape[1] == 64
    return x


@pytest.mark.parametrize("bits", [4, 8])
def test_special_values_round_as_defined(cuda, bits):
    from vla_b200.kvcache import KVCache
    x = special_rows()
    y = x.roll(32, dims=1)
    n = len(x)
    cache = KVCache(1, n, kv_heads=1, bits=bits)
    cache.append(x.cuda(), y.cuda(), i32([0]), n)
    for got, want in zip(cache.read(n), (x, y)):
        np.testing.assert_array_equal(f64(got[0]), R.held(f64(want), bits))


@pytest.mark.parametrize("bits", [4, 8])
def test_every_bf16_magnitude_quantises_as_defined(cuda, bits):
    """One group per bf16 bit pattern as its peak, against fractions of it."""
    from vla_b200.kvcache import KVCache
    peak = torch.arange(0, 65536, 7, dtype=torch.int32).to(torch.int16).view(BF16)
    frac = torch.linspace(-1, 1, 63)
    x = torch.cat([peak[:, None].float(), peak[:, None].float() * frac], 1).to(BF16)
    n = len(x)
    cache = KVCache(1, n, kv_heads=1, bits=bits)
    cache.append(x.cuda(), x.cuda(), i32([0]), n)
    k, v = cache.read(n)
    want = R.held(f64(x), bits)
    np.testing.assert_array_equal(f64(k[0]), want)
    np.testing.assert_array_equal(f64(v[0]), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_read_ranges_layers_and_strided_rows(cuda, bits):
    B, n, H = 3, 90, 2
    cache, gen = make(B, 200, H, bits, layers=2)
    qkv = rows_like(gen, B * n, 6 * 64 + 2 * H * 64).cuda()  # Q | K | V rows of a layer
    k, v = qkv[:, 6 * 64:6 * 64 + H * 64], qkv[:, 6 * 64 + H * 64:]
    start = i32([0, 37, 110])
    cache.append(k, v, start, n, layer=1)
    hk, hv = R.held(f64(k).reshape(B, n, H, 64), bits), R.held(f64(v).reshape(B, n, H, 64), bits)
    # a part of them, from the middle, into a wider buffer
    first, m, counts = 13, 71, [71, 0, 50]
    wide = torch.full((2, B, m, H * 64 + 64), 7.0, dtype=BF16, device="cuda")
    out = cache.read(m, count=i32(counts), start=start + first, layer=1, out=(wide[0, :, :, :H * 64], wide[1, :, :, :H * 64]))
    for got, want in zip(out, (hk, hv)):
        want = want[:, first:first + m].reshape(B, m, H * 64).copy()
        for b in range(B):
            want[b, counts[b]:] = 0
        np.testing.assert_array_equal(f64(got), want)
    assert (wide[..., H * 64:] == 7).all()
    check_clean()


CASES = [
    # rows, q heads, kv heads, lens, q_len, causal, window, sinks
    (1, 3, 1, [1], None, True, 0, 0),
    (1, 15, 5, [114, 64, 65, 1], None, True, 0, 0),
    (1, 4, 4, [0, 63, 200], None, True, 0, 0),
    (1, 32, 2, [129, 31], None, True, 50, 0),
    (2, 6, 2, [300, 2, 1], None, True, 33, 5),
    (7, 15, 5, [200, 3, 0], None, True, 0, 0),
    (5, 6, 2, [97, 160], [5, 2], True, 0, 0),
    (9, 8, 1, [150, 40], [0, 9], False, 32, 70),
    (50, 15, 5, [113, 20], None, False, 0, 0),
    (50, 6, 2, [400, 49, 10], None, True, 64, 3),
    (3, 3, 1, [257], None, True, 1, 0),
    (33, 12, 12, [33, 90], [33, 1], True, 0, 0),
    (150, 3, 1, [260, 150], [150, 130], True, 100, 1),
    (1, 3, 1, [500], None, True, 10, 490),
    (4, 6, 2, [500], None, False, 1, 1),
    (33, 8, 8, [1 + 37 * i % 128 for i in range(96)], None, True, 0, 0),  # many short sequences per CTA
    (40, 4, 4, [37 * i % 300 for i in range(70)], None, False, 0, 0),
]


def run_case(case, bits, seed=1, max_len=0, room=None):
    rows, hq, hkv, lens, q_len, causal, window, sinks = case
    B, n = len(lens), max(max(lens), 1)
    cache, gen = make(B, room or n, hkv, bits, seed)
    k, v = rows_like(gen, B, n, hkv * 64), rows_like(gen, B, n, hkv * 64)
    cache.append(k.cuda(), v.cuda(), i32([0] * B), n, count=i32(lens))
    q = rows_like(gen, B, rows, hq, 64)
    got = cache.attend(q.cuda(), i32(lens), causal=causal, window=window, sinks=sinks, max_len=max_len,
                       q_len=None if q_len is None else i32(q_len))
    hk, hv = R.held(f64(k).reshape(B, n, hkv, 64), bits), R.held(f64(v).reshape(B, n, hkv, 64), bits)
    want, mag, big = R.attend(f64(q), hk, hv, lens, causal, window, sinks, q_len=q_len)
    err, bound = np.abs(f64(got) - want), R.attend_bound(want, mag, big)
    assert np.all(err <= bound), f"error {err.max()} at most {(err / np.maximum(bound, 1e-30)).max()} times its bound"
    check_clean()
    return cache, q, got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"r{c[0]}_h{c[1]}.{c[2]}_n{c[3][0]}_c{int(c[5])}_w{c[6]}_s{c[7]}")
def test_attend_matches_the_definition(cuda, case, bits):
    run_case(case, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case,max_len", [
    ((1, 3, 1, [3001], None, True, 0, 0), 0),
    ((1, 6, 2, [2000, 5000, 0, 1], None, True, 0, 0), 0),
    ((1, 6, 2, [2000, 5000, 0, 1], None, True, 0, 0), 64),  # the hint may be too small
    ((2, 8, 1, [4097, 1500], None, True, 1200, 100), 0),
    ((20, 3, 1, [3000], [7], False, 0, 0), 0),
])
def test_attend_splits_long_caches(cuda, case, max_len, bits):
    run_case(case, bits, max_len=max_len)


def test_attend_repeats_bit_for_bit_and_leaves_the_cache(cuda):
    cache, q, got = run_case((1, 6, 2, [2000, 5000], None, True, 0, 0), 4)
    before = cache.pool.clone()
    for _ in range(3):
        assert torch.equal(cache.attend(q.cuda(), i32([2000, 5000])), got)
    assert torch.equal(cache.pool, before)


def test_rows_layouts_agree(cuda):
    cache, q, got = run_case((5, 6, 2, [97, 160], None, True, 0, 0), 4)
    lens = i32([97, 160])
    wide = torch.zeros(2, 7, 9 * 64, dtype=BF16, device="cuda")  # strided rows of a wider buffer
    wide[:, 1:6, 64:448] = q.cuda().flatten(2)
    out = torch.full((2, 6, 8 * 64), 3.0, dtype=BF16, device="cuda")
    cache.attend(wide[:, 1:6, 64:448], lens, out=out[:, :5, 128:])
    assert torch.equal(out[:, :5, 128:], got.flatten(2))
    assert (out[:, 5] == 3).all() and (out[:, :, :128] == 3).all()


def test_seen_nan_reaches_its_rows_only(cuda):
    B, n, H = 2, 70, 1
    cache, gen = make(B, n, H, 4)
    k, v = rows_like(gen, B, n, 64), rows_like(gen, B, n, 64)
    k[0, 60, 3] = float("nan")  # group 0 of token 60 of sequence 0
    cache.append(k.cuda(), v.cuda(), i32([0, 0]), n)
    q = rows_like(gen, B, 20, 3, 64)
    got = cache.attend(q.cuda(), i32([n, n]))  # positions 50 .. 69
    assert torch.isfinite(got[0, :10].float()).all() and torch.isfinite(got[1].float()).all()
    assert torch.isnan(got[0, 10:].float()).all()
    # every score of a row NaN
    k[1] = float("nan")
    cache.append(k.cuda(), v.cuda(), i32([0, 0]), n)
    assert torch.isnan(cache.attend(q.cuda(), i32([n, n]))[1].float()).all()
    # a value's NaN group spoils its dims alone
    v[0, 65, 40] = float("inf")
    k[0, 60, 3] = 0
    cache.append(k.cuda(), v.cuda(), i32([0, 0]), n)
    got = cache.attend(q.cuda(), i32([n, n]))[0].float()
    assert torch.isfinite(got[:15]).all() and torch.isfinite(got[..., :32]).all()
    assert torch.isnan(got[15:, :, 32:]).all()


def test_large_scores_and_equal_scores(cuda):
    """Scores of hundreds (one key takes all) and all alike (a plain mean)."""
    from vla_b200.kvcache import KVCache
    gen = torch.Generator().manual_seed(5)
    n = 300
    k, v = rows_like(gen, 1, n, 64), rows_like(gen, 1, n, 64)
    for kk, factor in ((k * 40, 40.0), (torch.ones_like(k), 1.0)):
        cache = KVCache(1, n, kv_heads=1, bits=8)
        cache.append(kk.cuda(), v.cuda(), i32([0]), n)
        q = (rows_like(gen, 1, 1, 3, 64) * factor).to(BF16)
        hk, hv = R.held(f64(kk).reshape(1, n, 1, 64), 8), R.held(f64(v).reshape(1, n, 1, 64), 8)
        want, mag, big = R.attend(f64(q), hk, hv, [n])
        assert np.all(np.abs(f64(cache.attend(q.cuda(), i32([n]))) - want) <= R.attend_bound(want, mag, big))


def test_offsets_past_32_bits(cuda):
    """Pages behind the first 2^32 bytes of a pool."""
    from vla_b200.kvcache import KVCache, block_bytes
    pages = 2 ** 32 // (5 * block_bytes(4)) + 40
    cache = KVCache(1, 128, kv_heads=5, bits=4, pages=pages)
    cache.table.copy_(torch.tensor([[pages - 1, 3]]))
    gen = torch.Generator().manual_seed(9)
    k, v = rows_like(gen, 1, 100, 320), rows_like(gen, 1, 100, 320)
    cache.append(k.cuda(), v.cuda(), i32([0]), 100)
    got = cache.read(100)[0]
    np.testing.assert_array_equal(f64(got), R.held(f64(k).reshape(1, 100, 5, 64), 4).reshape(1, 100, 320))
    q = rows_like(gen, 1, 1, 15, 64)
    o = cache.attend(q.cuda(), i32([100]))
    small = KVCache(1, 128, kv_heads=5, bits=4)
    small.append(k.cuda(), v.cuda(), i32([0]), 100)
    assert torch.equal(o, small.attend(q.cuda(), i32([100])))
    check_clean()


def test_bad_pages_and_positions_are_skipped_and_reported(cuda):
    from vla_b200 import _lib, device as dev
    cache, gen = make(1, 192, 1, 4)
    k, v = rows_like(gen, 1, 192, 64), rows_like(gen, 1, 192, 64)
    cache.append(k.cuda(), v.cuda(), i32([0]), 192)
    check_clean()
    good = cache.table.clone()
    q = rows_like(gen, 1, 1, 3, 64).cuda()

    def reported():
        with pytest.raises(_lib.VlaError) as e:
            dev.sync_check()
        assert e.value.code == _lib.VLA_E_DEVICE_RANGE
        dev.sync_check()  # read once, then clear

    for bad in (-1, 3, 2 ** 30):
        cache.table[0, 1] = bad
        got = cache.attend(q, i32([192]))
        reported()
        hk, hv = (R.held(f64(x).reshape(1, 192, 1, 64), 4) for x in (k, v))
        keep = [j for j in range(192) if j // 64 != 1]  # the page's keys are not seen
        want, mag, big = R.attend(f64(q), hk[:, keep], hv[:, keep], [128])
        assert np.all(np.abs(f64(got) - want) <= R.attend_bound(want, mag, big))
        assert (cache.read(192)[0][0, 64:128] == 0).all()
        reported()
    cache.table.copy_(good)
    cache.append(k.cuda(), v.cuda(), i32([150]), 192, count=i32([60]))  # 42 fit
    reported()
    cache.append(k[:, :1].cuda(), v[:, :1].cuda(), i32([-1]), 1)
    reported()
    cache.attend(q, i32([193]))
    reported()
    cache.attend(q, i32([-5]))
    reported()
    assert torch.isfinite(cache.attend(q, i32([150])).float()).all()
    check_clean()


def test_other_streams_and_graph_replays_as_the_sequence_grows(cuda):
    from vla_b200.kvcache import KVCache
    gen = torch.Generator().manual_seed(3)
    H, steps = 2, 70
    k, v = rows_like(gen, steps, 1, 1, H * 64).cuda(), rows_like(gen, steps, 1, 1, H * 64).cuda()
    q = rows_like(gen, steps, 1, 1, 6, 64).cuda()
    plain = KVCache(1, 128, kv_heads=H)
    want = []
    for i in range(steps):
        plain.append(k[i], v[i], i32([i]), 1)
        want.append(plain.attend(q[i], i32([i + 1]), window=16, sinks=2))
    cache = KVCache(1, 128, kv_heads=H)
    kk, vv, qq = k[0].clone(), v[0].clone(), q[0].clone()
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(kk, vv, lens, 1)  # warm-up
        cache.attend(qq, lens + 1, window=16, sinks=2)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.append(kk, vv, lens, 1)
        lens += 1
        out = cache.attend(qq, lens, window=16, sinks=2)
    lens.zero_()
    for i in range(steps):
        kk.copy_(k[i]), vv.copy_(v[i]), qq.copy_(q[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
    check_clean()


def test_empty_calls_do_nothing(cuda):
    from vla_b200.kvcache import KVCache
    cache = KVCache(2, 64, kv_heads=1)
    z = torch.empty(2, 0, 64, dtype=BF16, device="cuda")
    cache.append(z, z, i32([0, 0]), 0)
    assert cache.read(0)[0].shape == (2, 0, 64)
    assert cache.attend(torch.empty(2, 0, 3, 64, dtype=BF16, device="cuda"), i32([0, 0])).shape == (2, 0, 3, 64)
    none = KVCache(0, 64, kv_heads=1)
    assert none.attend(torch.empty(0, 1, 3, 64, dtype=BF16, device="cuda"), i32([])).shape == (0, 1, 3, 64)
    check_clean()


def test_refusals(cuda):
    from vla_b200 import _lib
    from vla_b200.kvcache import KVCache
    with pytest.raises(_lib.VlaError, match="4 or 8 bits"):
        KVCache(1, 64, bits=3)
    cache = KVCache(2, 64, kv_heads=2)
    x = torch.zeros(2, 3, 128, dtype=BF16, device="cuda")
    lens = i32([3, 3])
    for bad in (x.float(), x[:, :2], x.cpu(), x[..., :64], x.transpose(0, 1)):
        with pytest.raises(ValueError, match="k:"):
            cache.append(bad, x, lens, 3)
    for bad in (lens.long(), lens[:1], lens.cpu(), i32([[1], [2]])):
        with pytest.raises(ValueError, match="start:"):
            cache.append(x, x, bad, 3)
    with pytest.raises(_lib.VlaError, match="alignment"):
        y = torch.zeros(2 * 3 * 128 + 1, dtype=BF16, device="cuda")[1:].view(2, 3, 128)
        cache.append(y, x, lens, 3)
    with pytest.raises(_lib.VlaError, match="stride"):
        cache.append(x[:, :1].expand(2, 3, 128), x, lens, 3)
    q = torch.zeros(2, 1, 4, 64, dtype=BF16, device="cuda")
    for bad in (q[..., :32], q.float(), q[:1], q[0]):
        with pytest.raises(ValueError, match="q:"):
            cache.attend(bad, lens)
    with pytest.raises(_lib.VlaError, match="kv heads"):
        cache.attend(q[:, :, :3], lens)
    for kw in ({"window": -1}, {"sinks": 2 ** 31}, {"max_len": -2}):
        with pytest.raises(ValueError, match="window"):
            cache.attend(q, lens, **kw)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(_lib.VlaError, match="scale"):
            cache.attend(q, lens, scale=scale)
    with pytest.raises(ValueError, match="out:"):
        cache.attend(q, lens, out=torch.empty(2, 1, 3, 64, dtype=BF16, device="cuda"))
    with pytest.raises(IndexError):
        cache.attend(q, lens, layer=1)
    with pytest.raises(ValueError, match="pool"):
        KVCache.wrap(torch.empty(1, 2, 100, dtype=torch.uint8, device="cuda"), i32([[0]]), 2, 4)
    with pytest.raises(ValueError, match="table"):
        KVCache.wrap(cache.pool, cache.table.long(), 2, 4)


def test_many_rows_bad_pages_and_shared_queries(cuda):
    """The kernel for many rows: a page that is not there, a page count that is odd, and
    one sequence's queries for all (a zero stride)."""
    from vla_b200 import _lib, device as dev
    B, n, H = 3, 300, 2
    cache, gen = make(B, n, H, 4)
    k, v = rows_like(gen, B, n, H * 64), rows_like(gen, B, n, H * 64)
    cache.append(k.cuda(), v.cuda(), i32([0] * B), n)
    q = rows_like(gen, 1, 50, 6, 64).expand(B, 50, 6, 64)
    hk, hv = (R.held(f64(x).reshape(B, n, H, 64), 4) for x in (k, v))
    lens = [300, 193, 64]
    got = cache.attend(q.cuda()[:1].expand(B, 50, 6, 64), i32(lens), causal=False)
    want, mag, big = R.attend(f64(q), hk, hv, lens, causal=False)
    assert np.all(np.abs(f64(got) - want) <= R.attend_bound(want, mag, big))
    check_clean()
    cache.table[0, 2] = 10 ** 6
    got = cache.attend(q.cuda(), i32(lens), causal=False)
    with pytest.raises(_lib.VlaError) as e:
        dev.sync_check()
    assert e.value.code == _lib.VLA_E_DEVICE_RANGE
    keep = [j for j in range(n) if j // 64 != 2]
    first, mag0, big0 = R.attend(f64(q)[:1], hk[:1, keep], hv[:1, keep], [len(keep)], causal=False)
    want[0], mag[0], big[0] = first[0], mag0[0], big0[0]
    assert np.all(np.abs(f64(got) - want) <= R.attend_bound(want, mag, big))


@pytest.mark.parametrize("rows", [3, 60])
def test_values_of_the_largest_size_do_not_leak_from_hidden_keys(cuda, rows):
    """A key that a row does not see may hold values near bf16's end."""
    cache, gen = make(1, 128, 1, 8)
    k, v = rows_like(gen, 1, 100, 64), rows_like(gen, 1, 100, 64)
    v[0, 99] = 1.6e38
    cache.append(k.cuda(), v.cuda(), i32([0]), 100)
    q = rows_like(gen, 1, rows, 3, 64)
    got = cache.attend(q.cuda(), i32([100]))
    hk, hv = (R.held(f64(x).reshape(1, 100, 1, 64), 8) for x in (k, v))
    want, mag, big = R.attend(f64(q)[:, :-1], hk, hv, [99])
    assert np.all(np.abs(f64(got)[:, :-1] - want) <= R.attend_bound(want, mag, big))


def test_query_layouts_that_share_a_kernel_agree(cuda):
    """The same row in a call of few rows and in one of many: within the two kernels' roundings."""
    cache, gen = make(2, 500, 2, 4)
    k, v = rows_like(gen, 2, 500, 128), rows_like(gen, 2, 500, 128)
    cache.append(k.cuda(), v.cuda(), i32([0, 0]), 500)
    q = rows_like(gen, 2, 40, 6, 64).cuda()
    many = cache.attend(q, i32([500, 333]), window=100, sinks=5)
    hv = R.held(f64(v).reshape(2, 500, 2, 64), 4)
    for i in (0, 17, 39):
        few = cache.attend(q[:, i:i + 1], i32([500 - 39 + i, 333 - 39 + i]), window=100, sinks=5)
        assert np.all(np.abs(f64(few[:, 0]) - f64(many[:, i])) <= 2.0 ** -6 * np.abs(hv).max())


@pytest.mark.parametrize("rows", [1, 60])
def test_value_scales_of_very_different_size(cuda, rows):
    """Values that grow and shrink by powers of two along the sequence, over bf16's range."""
    n = 700
    cache, gen = make(1, n, 1, 4)
    k, v = rows_like(gen, 1, n, 64), rows_like(gen, 1, n, 64)
    step = torch.randint(-12, 13, (1, n // 20, 1), generator=gen).float().repeat_interleave(20, 1)
    for power in (-80.0, 0.0, 100.0):
        vv = (v.float() * 2 ** (step + power)).to(BF16)
        cache.append(k.cuda(), vv.cuda(), i32([0]), n)
        q = (rows_like(gen, 1, rows, 3, 64) * 0.25).to(BF16)
        hk, hv = (R.held(f64(x).reshape(1, n, 1, 64), 4) for x in (k, vv))
        want, mag, big = R.attend(f64(q), hk, hv, [n])
        err = np.abs(f64(cache.attend(q.cuda(), i32([n]))) - want)
        assert np.all(err <= R.attend_bound(want, mag, big))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows", [1, 2, 8, 40])
def test_a_nan_value_group_leaves_the_other_group(cuda, rows, bits):
    """One token's second value group is NaN: the first 32 dims stay right, the rest is NaN where it is seen."""
    n = 90
    cache, gen = make(1, n, 1, bits)
    k, v = rows_like(gen, 1, n, 64), rows_like(gen, 1, n, 64)
    v[0, 20, 50] = float("inf")
    cache.append(k.cuda(), v.cuda(), i32([0]), n)
    q = rows_like(gen, 1, rows, 3, 64)
    got = f64(cache.attend(q.cuda(), i32([n])))
    hk, hv = (R.held(f64(x).reshape(1, n, 1, 64), bits) for x in (k, v))
    want, mag, big = R.attend(f64(q), hk, np.nan_to_num(hv), [n])
    bound = R.attend_bound(want, mag, big)
    assert np.all(np.abs(got[..., :32] - want[..., :32]) <= bound[..., :32])
    assert np.isnan(got[..., 32:]).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("room", [300, 700])
@pytest.mark.parametrize("lens,q_len", [
    ([0] * 37, None),
    ([1 + 61 * i % 300 if i % 3 else 0 for i in range(130)] + [0] * 30, None),
    ([0] * 50 + [113] * 40, [i % 18 for i in range(90)]),
    ([300], [7]),
])
def test_many_rows_short_caches_with_empty_sequences(cuda, lens, q_len, room, bits):
    """Items that are dealt out whole (room for few pages) or in units, empty ones at a
    share's start, middle and end; rows that do not fill a block."""
    run_case((17, 6, 3, lens, q_len, True, 0, 0), bits, room=room)
    run_case((17, 6, 2, lens, q_len, False, 70, 3), bits, room=room)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,heads", [(1, 3), (5, 12), (90, 3)])
@pytest.mark.parametrize("raw", [0x7F00, 0x7F7F, 0xFF7F, 0x7E00])
def test_hidden_slots_that_no_append_wrote(cuda, rows, heads, bits, raw):
    """Only the first tokens and the newest part of a stream were moved into the cache: the slots below the
    length that nothing wrote, and that the masks hide, may hold finite scales whose values overflow."""
    n, window, sinks = 330, 20, 9
    first = n - rows - window  # the oldest key that the window shows, and one to spare
    outs = []
    for fill in (raw, 0):
        cache, gen = make(1, n, 1, bits, seed=4)
        cache.pool[..., -512:].view(torch.int16).fill_(fill - 65536 if fill > 32767 else fill)
        k, v = rows_like(gen, 1, n, 64), rows_like(gen, 1, n, 64)
        q = rows_like(gen, 1, rows, heads, 64)
        cache.append(k[:, :sinks].cuda(), v[:, :sinks].cuda(), i32([0]), sinks)
        cache.append(k[:, first:].cuda(), v[:, first:].cuda(), i32([first]), n - first)
        outs.append(cache.attend(q.cuda(), i32([n]), window=window, sinks=sinks))
    hk, hv = (R.held(f64(x).reshape(1, n, 1, 64), bits) for x in (k, v))
    want, mag, big = R.attend(f64(q), hk, hv, [n], True, window, sinks)
    assert np.all(np.abs(f64(outs[0]) - want) <= R.attend_bound(want, mag, big))
    assert torch.equal(outs[0], outs[1])
    check_clean()


def test_an_expired_wait_outranks_a_skipped_page(cuda):
    """A page that was skipped must not hide that a kernel gave up, whichever came first."""
    import ctypes
    from vla_b200 import _lib
    from vla_b200.kvcache import KVCache
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    cache = KVCache(1, 64, kv_heads=1, pages=1)  # its table holds no page
    q = torch.zeros(1, 1, 3, 64, dtype=BF16, device="cuda")
    check_clean()
    for order in ("page wait", "wait page"):
        for what in order.split():
            if what == "page":
                cache.attend(q, i32([5]))
            else:
                _lib.check(lib.vla_test_expired_wait(1000, stream))  # 1 ms limit
            torch.cuda.synchronize()
        code = ctypes.c_uint(0)
        _lib.check(lib.vla_peek_device_error(ctypes.byref(code)))
        assert code.value == 0x1FF
        assert lib.vla_sync_check() == _lib.VLA_E_DEVICE_TIMEOUT
        assert "0x1ff" in _lib.last_error()
        check_clean()
    cache.attend(q, i32([5]))
    torch.cuda.synchronize()
    _lib.check(lib.vla_peek_device_error(ctypes.byref(code)))
    assert code.value == 0x301
    assert lib.vla_sync_check() == _lib.VLA_E_DEVICE_RANGE
    check_clean()


def test_outputs_may_lie_between_each_other(cuda):
    """Keys and values in one buffer, and the rows of all sequences in turn (token-major): no element has two writers."""
    from vla_b200 import _lib
    B, n, H = 3, 20, 2
    cache, gen = make(B, n, H, 4)
    k, v = rows_like(gen, B, n, H * 64), rows_like(gen, B, n, H * 64)
    cache.append(k.cuda(), v.cuda(), i32([0] * B), n)
    buf = torch.zeros(n, B, 2, H * 64, dtype=BF16, device="cuda")
    views = buf[:, :, 0].transpose(0, 1), buf[:, :, 1].transpose(0, 1)
    for got, want in zip(cache.read(n, out=views), cache.read(n)):
        assert torch.equal(got, want)
    q, lens = rows_like(gen, B, n, 6, 64).cuda(), i32([n] * B)
    out = torch.zeros(n, B, 6 * 64, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(cache.attend(q, lens, out=out), cache.attend(q, lens).flatten(2))
    one = torch.zeros(1, n, 6 * 64, dtype=BF16, device="cuda").expand(B, n, 6 * 64)
    with pytest.raises(_lib.VlaError, match="overlap"):
        cache.attend(q, lens, out=one)
    with pytest.raises(_lib.VlaError, match="overlap"):
        cache.read(n, out=(one[..., :128], torch.zeros(B, n, 128, dtype=BF16, device="cuda")))
    check_clean()


def test_a_refused_call_leaves_the_next_one_alone(cuda):
    """A call whose arguments are refused says nothing about the workspace of valid ones of its sizes."""
    from vla_b200 import _lib
    cache, gen = make(1, 3000, 1, 4)
    k, v = rows_like(gen, 1, 3000, 64), rows_like(gen, 1, 3000, 64)
    cache.append(k.cuda(), v.cuda(), i32([0]), 3000)
    for rows in (1, 40):  # either kernel, both split along the cache
        q, lens = rows_like(gen, 1, rows, 3, 64).cuda(), i32([3000])
        for scale in (float("nan"), 0.0):
            with pytest.raises(_lib.VlaError, match="scale"):
                cache.attend(q, lens, scale=scale)
        got = cache.attend(q, lens)
        assert torch.equal(got, cache.attend(q, lens, max_len=3001))  # a plan of its own


@pytest.mark.parametrize("bits", [4, 8])
def test_special_values_are_written_as_defined(cuda, bits):
    """The bytes of groups where a rounding or a sign can go wrong: the scales, and the
    codes wherever the scale is a number."""
    from vla_b200.kvcache import KVCache
    x = special_rows()
    y = x.roll(32, dims=1)
    n = len(x)
    cache = KVCache(1, n, kv_heads=1, bits=bits)
    cache.append(x.cuda(), y.cuda(), i32([0]), n)
    got = cache.pool[0, :, 0].cpu().numpy()
    want = got.copy()
    for i in range(n):
        R.write_token(want[i // 64], bits, i % 64, f64(x)[i], f64(y)[i])
    for i in range(n):
        for keys, rows in ((True, x), (False, y)):
            for group in range(2):
                at = R.scale_place(bits, keys, i % 64, group)
                np.testing.assert_array_equal(got[i // 64, at:at + 2], want[i // 64, at:at + 2], f"{rows[i]}")
                if got[i // 64, at + 1] == 0x7F and got[i // 64, at] & 0x80:
                    continue  # NaN
                places = {R.code_place(bits, keys, i % 64, 32 * group + d) for d in range(32)}
                for byte, shift in places:
                    m = 15 << shift if bits == 4 else 255
                    assert got[i // 64, byte] & m == want[i // 64, byte] & m, (rows[i], byte, shift)
    for back, rows in zip(cache.read(n), (x, y)):  # zeros with their signs
        held = R.held(f64(rows), bits)
        same = np.signbit(f64(back[0])) == np.signbit(held)
        assert np.all(same | np.isnan(held))


@pytest.mark.parametrize("scale", [1e-36, 1e-38, 1e-42])
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 3000), (7, 700), (40, 300)])
def test_scales_near_zero_give_the_mean(cuda, rows, n, scale):
    """Every positive finite scale counts, also one whose reciprocal is not finite."""
    cache, gen = make(1, n, 1, 4)
    k, v = rows_like(gen, 1, n, 64), rows_like(gen, 1, n, 64)
    cache.append(k.cuda(), v.cuda(), i32([0]), n)
    q = rows_like(gen, 1, rows, 3, 64)
    hk, hv = (R.held(f64(x).reshape(1, n, 1, 64), 4) for x in (k, v))
    want, mag, big = R.attend(f64(q), hk, hv, [n], scale=scale)
    got = cache.attend(q.cuda(), i32([n]), scale=scale)
    assert np.all(np.abs(f64(got) - want) <= R.attend_bound(want, mag, big))


def test_the_longest_window_with_rows_before_the_first_key(cuda):
    """Queries at negative positions see nothing; their window reaches almost to -2^31."""
    from vla_b200.kvcache import KVCache
    gen = torch.Generator().manual_seed(6)
    room, n = 2 ** 31 - 512, 90
    cache = KVCache(2, room, kv_heads=1, pages=4)
    cache.table[:, :2] = torch.tensor([[3, 0], [1, 2]])
    k, v = rows_like(gen, 2, n, 64), rows_like(gen, 2, n, 64)
    lens = [30, 90]
    cache.append(k.cuda(), v.cuda(), i32([0, 0]), n, count=i32(lens))
    q = rows_like(gen, 2, 100, 3, 64)
    hk, hv = (R.held(f64(x).reshape(2, n, 1, 64), 4) for x in (k, v))
    want, mag, big = R.attend(f64(q), hk, hv, lens)
    got = f64(cache.attend(q.cuda(), i32(lens), window=room - 1))
    assert np.all(np.abs(got - want) <= R.attend_bound(want, mag, big))
    assert np.abs(got[0, 70:]).max() > 0 and (got[0, :70] == 0).all()
    check_clean()


@pytest.mark.parametrize("bits", [4, 8])
def test_append_and_read_of_calls_that_fill_the_gpu(cuda, bits):
    """Four groups of positions per warp (calls of 64 warps per SM and more): bytes and values, uneven starts and counts."""
    B, n, H = 320, 113, 5
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert B * H * -(-((n + 6) // 4) // 4) >= 64 * sms
    starts = [37 * b % 70 for b in range(B)]
    counts = [n if b % 40 == 3 else b % 7 for b in range(B)]
    cache, gen = make(B, 70 + n, H, bits, spare=3)
    want = cache.pool[0].cpu().numpy().copy()
    k, v = rows_like(gen, B, n, H * 64), rows_like(gen, B, n, H * 64)
    cache.append(k.cuda(), v.cuda(), i32(starts), n, count=i32(counts))
    table, kk, vv = cache.table.cpu().numpy(), f64(k).reshape(B, n, H, 64), f64(v).reshape(B, n, H, 64)
    held = np.zeros((2, B, n, H, 64))
    for b in range(B):
        for i in range(counts[b]):
            at = starts[b] + i
            for h in range(H):
                R.write_token(want[table[b, at // 64], h], bits, at % 64, kk[b, i, h], vv[b, i, h])
        held[0, b, :counts[b]], held[1, b, :counts[b]] = R.held(kk[b, :counts[b]], bits), R.held(vv[b, :counts[b]], bits)
    np.testing.assert_array_equal(cache.pool[0].cpu().numpy(), want)
    for got, x in zip(cache.read(n, count=i32(counts), start=i32(starts)), held):
        np.testing.assert_array_equal(f64(got), x.reshape(B, n, H * 64))
    check_clean()


@pytest.mark.parametrize("room", [64, 700])
@pytest.mark.parametrize("bits", [4, 8])
def test_many_rows_with_many_items_per_cta(cuda, bits, room):
    """More than twenty items for each CTA, so that the entries by which its warps hear of them are used again and
    again: items dealt out whole (room for one page) and in units."""
    lens = [1 + 5 * b % 12 if b % 29 else 0 for b in range(640)]
    run_case((11, 15, 5, lens, None, True, 0, 0), bits, room=room)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", [
    (120, 3, 1, [1500, 700], None, True, 0, 0),       # two blocks of rows
    (200, 3, 1, [1290, 777], [200, 90], True, 600, 70),
    (300, 2, 2, [900], None, False, 400, 0),
    (260, 1, 1, [2000, 0, 261], None, True, 64, 1),
], ids=lambda c: f"r{c[0]}_w{c[6]}")
def test_several_blocks_of_rows_over_caches_that_are_cut(cuda, case, bits):
    run_case(case, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", [
    (10, 3, 1, [3000, 1500], None, True, 0, 0),       # 30 rows
    (8, 6, 2, [2500, 40], [8, 3], True, 900, 33),     # 24 rows
    (3, 15, 5, [2000, 2000, 1], None, False, 0, 0),   # 9 rows
    (1, 32, 1, [4000], None, True, 0, 0),             # 32 rows
    (4, 12, 3, [700, 90], None, True, 0, 0),          # 16 rows
], ids=lambda c: f"r{c[0] * c[1] // c[2]}")
def test_nine_to_32_rows_over_caches_that_are_cut(cuda, case, bits):
    run_case(case, bits)
