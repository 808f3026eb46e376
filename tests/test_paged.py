"""CPU tests of the paged cache operators' host side: the operators take device tensors only,
the C entries refuse a null context, and the plain forms of paged_ref.py agree with one another."""
import ctypes

import pytest
import torch

import paged_ref as ref
import tabinfer_b200 as tb
from tabinfer_b200._lib import LIB, PagedKV


def test_host_tensors_are_refused():
    c = ref.Cache(1, 1, 2, 16, 2, 64)
    kv, lens = (c.Kq, c.Ks, c.Vq, c.Vs), torch.tensor([5], dtype=torch.int32)
    q = torch.randn(1, 256)
    w = torch.ones(64, dtype=torch.float16)
    with pytest.raises(tb.TabInferError):
        tb.attention_decode_paged_q8(q, kv, c.table, lens, 4, 2, 64)
    with pytest.raises(tb.TabInferError):
        tb.attention_prefill_paged_q8(q, kv, c.table, torch.tensor([0, 1], dtype=torch.int32), lens, 4, 2, 64)
    with pytest.raises(tb.TabInferError):
        tb.attn_prep_paged_q8(q, q[:, :128], q[:, :128], w, w, kv, c.table, lens, lens, lens, 4, 2, 64, 1e6, 1e-6)
    with pytest.raises(tb.TabInferError):
        tb.kv_evict_paged_q8(kv, c.table, lens, torch.zeros(1, 2, 32), c.table, 4, 0, 0, 2, 64)


def test_null_context_is_refused():
    s, n = PagedKV(), ctypes.c_size_t()
    assert LIB.tb_attn_prep_paged_q8(None, ctypes.byref(s), *[None] * 6, 1, 1, None, None, None, 1.0, 0.0) == 1
    assert LIB.tb_attn_decode_paged_ws(None, ctypes.byref(s), 1, 0, ctypes.byref(n)) == 1
    assert LIB.tb_attn_decode_paged_q8(None, ctypes.byref(s), None, None, None, 1, 0, 0, None, None, 0) == 1
    assert LIB.tb_attn_prefill_paged_ws(None, ctypes.byref(s), 1, 1, ctypes.byref(n)) == 1
    assert LIB.tb_attn_prefill_paged_q8(None, ctypes.byref(s), None, None, None, None, 1, 1, 0, 0, None, 0) == 1
    assert LIB.tb_kv_evict_paged_ws(None, ctypes.byref(s), ctypes.byref(n)) == 1
    assert LIB.tb_kv_evict_paged_q8(None, ctypes.byref(s), ctypes.byref(s), None, None, None, None, None, 1, 0, 0,
                                    None, 0) == 1


def test_reference_attention():
    c = ref.Cache(2, 1, 4, 16, 2, 64)
    q = torch.randn(4 * 64, generator=c.g)
    full, w, _, _ = ref.attend(c, 0, q, 40, 4)
    wide = ref.attend(c, 0, q, 40, 4, window=41)[0]
    assert torch.equal(full, wide) and torch.allclose(w.sum(1), torch.full((2,), 2.0, dtype=torch.float64))
    all_sinks = ref.attend(c, 0, q, 40, 4, window=1, sinks=41)[0]
    assert torch.equal(full, all_sinks)
    own = ref.attend(c, 0, q, 40, 4, window=1)[0]
    assert torch.allclose(own[0], c.head(0, 41, 0)[1][40])


def test_reference_eviction():
    w = torch.tensor([[5.0, 1, 9, 2, 2, 2, 0, 0]])
    assert ref.evict(w, 8, 5, 1, 1) == [0, 2, 3, 4, 7]     # ties to the lower row
    assert ref.evict(w, 3, 5, 1, 1) == [0, 1, 2]
