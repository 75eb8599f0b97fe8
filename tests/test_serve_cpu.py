"""Host side of the serving operators (no GPU calls): the C entry points refuse
bad sizes, pointers and shapes before they touch a device, and the Python
functions refuse tensors that are not on a GPU."""
import ctypes

import pytest
import torch

L = pytest.importorskip("hif4x._lib")
from hif4x import serve  # noqa: E402

P = 0x10000   # never read: every call below is refused on the host


def lin(**kw):
    a = dict(x=P, ldx=128, meta=P, codes=P, T=4, N=8, C=128, bias=None, bias_dtype=0, act=0, res=None, ldr=8, y=P, ldy=8)
    a.update(kw)
    return L.lib().hif4x_linear_packed(*a.values(), None)


def test_linear_refusals():
    assert lin(T=0) == L.OK                                    # nothing to do
    for kw in (dict(x=None), dict(meta=None), dict(codes=None), dict(y=None), dict(T=-1), dict(N=0), dict(C=0),
               dict(C=96), dict(ldx=120), dict(ldx=132), dict(x=P + 2), dict(codes=P + 8), dict(ldy=7), dict(act=5),
               dict(act=-1), dict(res=P, ldr=7), dict(bias=P, bias_dtype=2)):
        assert lin(**kw) == L.ERR_ARG, kw
    assert lin(T=2 ** 31) == L.ERR_UNSUPPORTED


def cache(**kw):
    a = dict(k_codes=P, k_meta=P, v_codes=P, v_meta=P, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return L.KVCacheDesc(*a.values())


def batch(**kw):
    a = dict(cu_new=P, kv_len=P, pages=P, sequences=2, max_pages=3, ld_pages=3)
    a.update(kw)
    return L.KVBatchDesc(*a.values())


def calls(kv, b, rows=2):
    lib, r = L.lib(), ctypes.byref
    yield lib.hif4x_kv_append(r(kv), r(b), P, 128, 64, P, 128, 64, L.DT_BF16, rows, None)
    yield lib.hif4x_kv_read(r(kv), r(b), rows, P, P, L.DT_BF16, None)
    yield lib.hif4x_paged_attention(r(kv), r(b), P, 256, 64, 4, rows, 0.1, 0, 0, 1, P, 256, 64, None, 0, None)


def test_cache_and_batch_refusals():
    for kw in (dict(k_codes=None), dict(v_meta=None), dict(num_pages=0), dict(kv_heads=0), dict(k_meta=P + 4)):
        assert set(calls(cache(**kw), batch())) == {L.ERR_ARG}, kw
    for kw in (dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(head_dim=96), dict(head_dim=256),
               dict(kv_heads=70000)):
        assert set(calls(cache(**kw), batch())) == {L.ERR_UNSUPPORTED}, kw
    for kw in (dict(cu_new=None), dict(kv_len=None), dict(pages=None), dict(sequences=0), dict(max_pages=0),
               dict(ld_pages=2)):
        assert set(calls(cache(), batch(**kw))) == {L.ERR_ARG}, kw
    assert set(calls(cache(), batch(), rows=-1)) == {L.ERR_ARG}


def test_attention_refusals():
    lib, r, need = L.lib(), ctypes.byref, L.i64()
    ok = dict(page=16, kvh=2, dh=64, B=2, most=3, qh=4, rows=2, window=0, sinks=0, max_new=1)
    for kw in (dict(kvh=0), dict(dh=80), dict(B=0), dict(most=0), dict(qh=3), dict(qh=1), dict(rows=-1), dict(window=-1),
               dict(sinks=-1), dict(window=2 ** 30 + 1), dict(sinks=2 ** 30 + 1), dict(max_new=0), dict(rows=2 ** 30)):
        assert lib.hif4x_paged_attention_work(*{**ok, **kw}.values(), r(need)) == L.ERR_ARG, kw
    assert lib.hif4x_paged_attention_work(*{**ok, "rows": 0}.values(), r(need)) == L.OK and need.value == 0


def test_python_refuses_host_tensors():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    meta, codes = torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        serve.linear(x, meta, codes)
    with pytest.raises(TypeError):
        serve.linear(x.float(), meta, codes)
    with pytest.raises(ValueError, match="CUDA"):
        serve.PagedKV.empty(4, 16, 2, 64, "cpu")
    with pytest.raises(ValueError, match="head_dim"):
        serve.PagedKV.empty(4, 16, 2, 80, "cpu")


def test_overlap_of_spans():
    t = torch.zeros(100)
    assert serve._overlap(t[:10], t[9:12]) and not serve._overlap(t[:10], t[10:12])
    assert serve._overlap(t.view(10, 10)[:, :2], t.view(10, 10)[:, 2:])     # spans, not elements
    assert not serve._overlap(t.view(10, 10)[:5, :2], t.view(10, 10)[5:])
