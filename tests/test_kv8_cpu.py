"""The rotary and 8-bit-cache operators without a GPU: what the entry points refuse,
the host check of page tables and lengths (the bounds that the kernels use), and
the rotary frequency tables."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def kv8(qtts):
    import qtts_b200.kv8 as m
    m._lib()
    return m


def _cache(kv8, **kw):
    c = kv8.Kv8(0, 0, 1, 2, 128, 10, 3, 4, *([4096] * 7))   # addresses that are never read: every call below is refused first
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def _err(kv8):
    return kv8.lib().qtts_create_error().decode()


@pytest.mark.parametrize("field,value", [("device", -1), ("code", 2), ("row_type", 0), ("head_dim", 96), ("n_kv_heads", 0), ("n_pages", 0),
                                         ("n_seqs", -1), ("max_pages", 0), ("k", None), ("v_scale", None), ("k_open", None), ("k", 4100)])
def test_a_cache_that_is_none_is_refused_everywhere(kv8, field, value):
    L = kv8.lib()
    c = C.byref(_cache(kv8, **{field: value}))
    a = kv8.Kv8Attend(4096, 4096, None, 4096, 4096, 0, 0, 0, 0, 3, 1, 4, 0, 1.0)
    assert L.qtts_op_kv8_append(c, 4096, 4096, None, 4096, 4096, 256, 128, 256, 128, 3, 1, None) == 0 and "append" in _err(kv8)
    assert L.qtts_op_kv8_read(c, 4096, 4096, None, 1, 4096, 4096, 3, 1, None) == 0
    assert L.qtts_op_kv8_attend(c, C.byref(a), None) == 0 and L.qtts_kv8_attend_ws(c, C.byref(a)) == -1
    assert L.qtts_op_kv8_evict(c, 4096, 4096, 8192, 1, 4096, 256, 16, 0, 0, 4096, 4096, 4096, None) == 0
    t = np.zeros(12, np.int32)
    assert L.qtts_kv8_check(c, t.ctypes.data, t.ctypes.data, None, 3, 1) == -1


def test_refusals_of_append_and_read(kv8):
    L, c = kv8.lib(), C.byref(_cache(kv8))
    ok = [c, 4096, 4096, None, 4096, 4096, 256, 128, 256, 128, 3, 1, None]
    for at, bad in [(1, None), (2, None), (4, None), (5, None), (4, 4097), (10, -1), (10, 2), (11, -1)]:
        args = list(ok)
        args[at] = bad
        assert L.qtts_op_kv8_append(*args) == 0, (at, bad)
    ok = [c, 4096, None, None, 1, 4096, 4096, 3, 1, None]
    for at, bad in [(1, None), (4, 8), (5, None), (6, 4104), (7, -1), (7, 2), (8, -1)]:
        args = list(ok)
        args[at] = bad
        assert L.qtts_op_kv8_read(*args) == 0, (at, bad)


def test_refusals_of_attend(kv8):
    L, c = kv8.lib(), C.byref(_cache(kv8))

    def call(**kw):
        a = kv8.Kv8Attend(4096, 4096, None, 4096, 4096, 512, 128, 512, 128, 3, 1, 4, 0, 1.0)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.qtts_op_kv8_attend(c, C.byref(a), None)

    for kw in [dict(table=None), dict(lens=None), dict(q=None), dict(out=None), dict(q=4097), dict(n_heads=3), dict(n_heads=0), dict(n_rows=2),
               dict(n_rows=-1), dict(max_q=-1), dict(window=-1), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(weight_in=4096), dict(weight_out=4096),
               dict(weight_in=4096, weight_out=4096, weight_stride=255), dict(weight_in=4096, weight_out=4096, weight_stride=256)]:
        assert call(**kw) == 0, kw
    assert L.qtts_op_kv8_attend(c, None, None) == 0


def test_refusals_of_evict(kv8):
    L, c = kv8.lib(), C.byref(_cache(kv8))
    ok = [c, 4096, 4096, 8192, 1, 4096, 256, 32, 4, 8, 8192, 4096, 8192, None]
    for at, bad in [(1, None), (2, None), (3, None), (3, 4096), (4, 0), (5, None), (6, 255), (7, 24), (7, 0), (7, 128), (8, -1), (8, 25), (9, -1), (9, 29),
                    (10, None), (10, 4096), (11, None), (12, None), (12, 4096)]:
        args = list(ok)
        args[at] = bad
        assert L.qtts_op_kv8_evict(*args) == 0, (at, bad)


def test_refusals_of_rope(kv8):
    L = kv8.lib()

    def call(**kw):
        a = kv8.RopeArgs(0, 1, 3, 4, 2, 128, 64, 0, 1.0, 4096, 4096, 4096, 8192, 4096, 8192, 512, 128, 256, 128, 512, 128, 256, 128)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.qtts_op_rope(C.byref(a), None)

    for kw in [dict(type=2), dict(rows=-1), dict(q_heads=0), dict(k_heads=-1), dict(dim=0), dict(rot=0), dict(rot=65), dict(rot=130), dict(k=None),
               dict(k_heads=0), dict(pos=None), dict(freq=None), dict(q=None), dict(q_out=None), dict(k_out=None), dict(q=4097), dict(freq=4100),
               dict(qo_row=256), dict(ko_head=64)]:
        assert call(**kw) == 0, kw
    assert L.qtts_op_rope(None, None) == 0


def test_tensors_on_the_cpu_are_refused(kv8):
    x = torch.zeros(2, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError):
        kv8.rope(x, None, torch.zeros(2, dtype=torch.int32), torch.ones(64, dtype=torch.float64))
    with pytest.raises(ValueError):
        kv8.KvCache8.empty(4, 1, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        kv8.KvCache8.empty(4, 1, 2, 128, code="int4", device="cpu")


@pytest.mark.parametrize("table,lens,cu,rows,most,want", [
    ([[0, 1, 9, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 100, 1], None, 3, 1, 0),
    ([[0, 1, 10, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 100, 1], None, 3, 1, 1),      # page 10 of 10
    ([[0, 1, 10, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [128, 100, 1], None, 3, 1, 0),      # ... past the length: not looked at
    ([[0, 1, -1, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [129, 100, 1], None, 3, 1, 1),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [257, 100, 1], None, 3, 1, 2),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, -1, 1], None, 3, 1, 2),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 0, 1], None, 3, 1, 4),         # a row for an empty sequence
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 0, 1], [0, 9, 9, 10], 10, 9, 0),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 0, 1], [0, 9, 9, 10], 9, 9, 4),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 0, 1], [0, 9, 9, 10], 10, 8, 4),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 9, 1], [0, 9, 8, 9], 9, 9, 4),
    ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 0, 0, 0]], [256, 9, 1], [-2147483648, 2147483647, 8, 9], 9, 9, 4),
])
def test_check_of_host_copies(kv8, table, lens, cu, rows, most, want):
    t, n = np.array(table, np.int32), np.array(lens, np.int32)
    u = None if cu is None else np.array(cu, np.int32)
    c = _cache(kv8)
    assert kv8.lib().qtts_kv8_check(C.byref(c), t.ctypes.data, n.ctypes.data, None if u is None else u.ctypes.data, rows, most) == want


def test_frequencies(kv8):
    f, m = kv8.rope_freqs(128, 1e6)
    assert m == 1.0
    assert torch.allclose(f, 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128), rtol=1e-13, atol=0)
    g, m = kv8.rope_freqs(128, 1e6, "linear", 4.0)
    assert m == 1.0 and torch.equal(g, f / 4)
    g, m = kv8.rope_freqs(64, 1e4, "ntk", 8.0)
    # the slowest pair turns 8 times slower, the fastest as before
    f, _ = kv8.rope_freqs(64, 1e4)
    assert m == 1.0 and g[0] == 1.0 and abs(float(f[-1] / g[-1]) - 8.0) < 1e-9
    g, m = kv8.rope_freqs(64, 1e4, "yarn", 8.0, original_len=4096)
    assert m == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-6)
    turns = f * 4096 / (2 * math.pi)
    ratio = g / f
    assert bool((ratio[turns > 34] == 1.0).all()) and bool((abs(ratio[turns < 0.9] - 1 / 8) < 1e-15).all())
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all())
    for bad in [dict(rot=7), dict(rot=0), dict(theta=1.0), dict(theta=math.inf), dict(scaling="cubic"), dict(scaling="yarn", factor=0.5),
                dict(scaling="yarn", factor=math.nan), dict(scaling="yarn", factor=2.0, beta_fast=1.0, beta_slow=1.0)]:
        with pytest.raises(ValueError):
            kv8.rope_freqs(**{**dict(rot=64, theta=1e4), **bad})
