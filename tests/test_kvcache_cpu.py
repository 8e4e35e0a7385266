"""The quantised key/value cache without a GPU: the C entry points' refusals, the
ctypes mirrors, and the restatement's own properties."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kvcache_ref as R
from vla_b200 import _lib


def cache_desc(**kw):
    d = _lib.KVCacheDesc()
    d.pool = d.table = 256
    d.table_ld, d.pages, d.max_pages, d.batch, d.kv_heads, d.head_dim, d.bits = 4, 8, 4, 2, 5, 64, 4
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def attention_args(**kw):
    a = _lib.KVAttentionArgs()
    a.q = a.o = a.lens = 256
    a.q_row = a.q_batch = a.o_row = a.o_batch = 960
    a.Lq, a.Hq, a.scale = 1, 15, 0.125
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_struct_sizes():
    assert ctypes.sizeof(_lib.KVCacheDesc) == 48
    assert ctypes.sizeof(_lib.KVAttentionArgs) == 112


@pytest.mark.parametrize("bits", [4, 8])
def test_block_bytes(bits):
    assert _lib.load().vla_kv_block_bytes(bits) == R.block_bytes(bits)
    assert _lib.load().vla_kv_block_bytes(bits + 1) == 0


@pytest.mark.parametrize("change,code,word", [
    ({"bits": 2}, "INVALID", "bits"), ({"head_dim": 128}, "INVALID", "head_dim"), ({"pool": None}, "INVALID", "null"),
    ({"table": None}, "INVALID", "null"), ({"kv_heads": 0}, "INVALID", "shape"), ({"table_ld": 3}, "INVALID", "stride"),
    ({"max_pages": 1 << 25, "table_ld": 1 << 25}, "INVALID", "2^31"), ({"pool": 264}, "ALIGN", "16-byte"),
])
def test_bad_caches_are_refused(change, code, word):
    lib, want = _lib.load(), getattr(_lib, "VLA_E_" + code)
    d = ctypes.byref(cache_desc(**change))
    assert lib.vla_kv_append_bf16(d, 256, 320, 320, 256, 320, 320, 1, 256, None, None) == want
    assert word in _lib.last_error()
    assert lib.vla_kv_read_bf16(d, 256, 320, 320, 256, 320, 320, 1, None, None, None) == want
    assert lib.vla_kv_attention_bf16(d, ctypes.byref(attention_args()), None) == want
    assert lib.vla_kv_attention_workspace(d, ctypes.byref(attention_args())) == 0


def test_bad_rows_are_refused():
    lib, d = _lib.load(), ctypes.byref(cache_desc())
    assert lib.vla_kv_append_bf16(None, 256, 320, 320, 256, 320, 320, 1, 256, None, None) == _lib.VLA_E_INVALID
    for k, row, batch, n, start, rc in ((None, 320, 320, 1, 256, "INVALID"), (256, 312, 320, 1, 256, "INVALID"),
                                        (256, 324, 320, 1, 256, "ALIGN"), (256, 320, 321, 1, 256, "ALIGN"),
                                        (258, 320, 320, 1, 256, "ALIGN"), (256, 320, 320, -1, 256, "INVALID"),
                                        (256, 320, 320, 1, None, "INVALID"), (256, 320, -320, 1, 256, "INVALID")):
        assert lib.vla_kv_append_bf16(d, k, row, batch, 256, 320, 320, n, start, None, None) == getattr(
            _lib, "VLA_E_" + rc)
    assert lib.vla_kv_append_bf16(d, None, 0, 0, None, 0, 0, 0, None, None, None) == _lib.VLA_OK  # nothing to do


@pytest.mark.parametrize("change,code", [
    ({"Hq": 14}, "INVALID"), ({"Hq": 0}, "INVALID"), ({"Lq": -1}, "INVALID"), ({"window": -1}, "INVALID"),
    ({"sinks": -1}, "INVALID"), ({"max_len": -1}, "INVALID"), ({"scale": 0.0}, "INVALID"),
    ({"scale": float("nan")}, "INVALID"), ({"lens": None}, "INVALID"), ({"q": None}, "INVALID"),
    ({"o_row": 952}, "INVALID"), ({"q_row": 964}, "ALIGN"), ({"Lq": 1 << 29}, "INVALID"),
])
def test_bad_attention_arguments_are_refused(change, code):
    rc = _lib.load().vla_kv_attention_bf16(ctypes.byref(cache_desc()), ctypes.byref(attention_args(**change)), None)
    assert rc == getattr(_lib, "VLA_E_" + code), _lib.last_error()


def test_workspace_is_asked_for_and_checked():
    lib = _lib.load()
    d = cache_desc(batch=1, max_pages=2048, table_ld=2048)
    a = attention_args()
    need = lib.vla_kv_attention_workspace(ctypes.byref(d), ctypes.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = 256, need - 1
    assert lib.vla_kv_attention_bf16(ctypes.byref(d), ctypes.byref(a), None) == _lib.VLA_E_WORKSPACE
    a.window = 64  # a short window needs no split
    assert lib.vla_kv_attention_workspace(ctypes.byref(d), ctypes.byref(a)) == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_places_cover_a_block_once(bits):
    seen = set()
    for keys in (True, False):
        for token in range(R.PAGE):
            for dim in range(R.DIM):
                seen.add(R.code_place(bits, keys, token, dim))
            for group in range(2):
                at = R.scale_place(bits, keys, token, group)
                seen |= {(at, 0), (at + 1, 0)}
    assert len(seen) == 2 * R.PAGE * R.DIM + R.PAGE * 8
    assert max(at for at, _ in seen) == R.block_bytes(bits) - 1


@pytest.mark.parametrize("bits,most", [(4, 0.5), (8, 0.5)])
def test_held_values_are_bf16_and_near(bits, most):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((200, 64)).astype(np.float32) * np.exp(rng.uniform(-30, 30, (200, 1)))
    x = (x.astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32).astype(np.float64)
    codes, d = R.quantise(x, bits)
    held = R.held(x, bits)
    R.bf16_bits(held)  # asserts that bf16 holds each
    step = np.abs(np.repeat(d, 32, axis=-1))
    off = np.abs(held - x) / step
    clipped = (codes == 7) & (bits == 4)  # the sign without a code 8 may lose up to a whole step
    assert off[~clipped].max() <= most and off.max() <= 1.0


def test_tables_with_overlapping_rows_are_refused():
    """The kernels take row b at b * stride: one row for all sequences has no such stride."""
    from vla_b200.kvcache import KVCache, block_bytes
    pool = torch.zeros(4, 1, block_bytes(4), dtype=torch.uint8)
    row = torch.arange(3, dtype=torch.int32)
    for table in (row.expand(5, 3), torch.arange(8, dtype=torch.int32).as_strided((3, 4), (2, 1))):
        with pytest.raises(ValueError, match="overlap"):
            KVCache.wrap(pool, table, 1, 4)
    for table in (row.expand(1, 3), torch.zeros(2, 4, dtype=torch.int32)[:, :3], row.expand(5, 3).contiguous()):
        with pytest.raises(ValueError, match="CUDA"):  # nothing but the device is wrong
            KVCache.wrap(pool, table, 1, 4)


@pytest.mark.parametrize("n,row,batch", [
    (1, 320, 0), (4, 320, 0),          # one sequence's rows for all
    (1, 320, 312), (4, 320, 1272),     # the last 8 elements are shared
    (4, 640, 312), (4, 632, 320),      # rows of all sequences in turn, too close
])
def test_outputs_that_overlap_are_refused(n, row, batch):
    """Two sequences with a row in common would be written by two writers."""
    lib, d = _lib.load(), ctypes.byref(cache_desc())
    assert lib.vla_kv_read_bf16(d, 256, row, batch, 4096, 320, 1280, n, None, None, None) == _lib.VLA_E_INVALID
    assert "k overlap" in _lib.last_error()
    assert lib.vla_kv_read_bf16(d, 256, 320, 1280, 4096, row, batch, n, None, None, None) == _lib.VLA_E_INVALID
    assert "v overlap" in _lib.last_error()
    a = attention_args(Lq=n, Hq=5, q_row=320, q_batch=0, o_row=row, o_batch=batch)
    assert lib.vla_kv_attention_bf16(d, ctypes.byref(a), None) == _lib.VLA_E_INVALID
    assert "o overlap" in _lib.last_error()


def test_one_output_for_keys_and_values_is_refused():
    lib, d = _lib.load(), ctypes.byref(cache_desc())
    assert lib.vla_kv_read_bf16(d, 256, 320, 1280, 256, 320, 1280, 4, None, None, None) == _lib.VLA_E_INVALID
    assert "one output" in _lib.last_error()


def test_a_scale_that_overflows_in_base_two_is_refused():
    """Exponentials are taken to base 2: the scale times log2(e) has to be a number, too."""
    a = attention_args(scale=3e38)
    assert _lib.load().vla_kv_attention_bf16(ctypes.byref(cache_desc()), ctypes.byref(a), None) == _lib.VLA_E_INVALID
    assert "scale" in _lib.last_error()


def test_tables_whose_windows_could_wrap_are_refused():
    """A row 255 positions before the first key, less a window of the whole table, has to fit 32 bits."""
    d = cache_desc(max_pages=(1 << 25) - 7, table_ld=1 << 25)
    assert _lib.load().vla_kv_attention_bf16(ctypes.byref(d), ctypes.byref(attention_args()), None) == _lib.VLA_E_INVALID
    assert "2^31 - 512" in _lib.last_error()
    d.max_pages -= 1
    a = attention_args()
    assert _lib.load().vla_kv_attention_workspace(ctypes.byref(d), ctypes.byref(a)) > 0
    assert -255 - (64 * d.max_pages - 1) + 1 >= -(1 << 31)
