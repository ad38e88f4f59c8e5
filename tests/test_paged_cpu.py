"""Refusals of the paged-cache entry points, without a GPU: what the C ABI answers
before any launch, and what the Python front end raises."""
import ctypes

import pytest
import torch

import dial_cuda as D
from dial_cuda import paged as P

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: checks fail first


def kv(**kw):
    v = dict(k_pages=0x1000, v_pages=0x1000, k_scale=None, v_scale=None, format=1, n_kv_heads=8, head_dim=128,
             page_size=64, n_pages=100)
    v.update(kw)
    return ctypes.byref(P._PagedKv(*v.values()))


def batch(**kw):
    v = dict(block_table=0x1000, kv_len=0x1000, q_start=0x1000, n_seqs=2, max_pages=8, max_q=4, max_kv=100)
    v.update(kw)
    return ctypes.byref(P._PagedBatch(*v.values()))


def axes(n=1, section=(64, 0, 0, 0), inter=0):
    return ctypes.byref(P._RopeAxes(n, (ctypes.c_int32 * 4)(*section), inter))


def attention(k=None, b=None, q=FAKE, out=FAKE, dt=D.F16, tokens=8, hq=32, scale=0.1):
    return D.lib().dial_paged_attention(q, k or kv(), b or batch(), out, dt, tokens, hq, scale, None)


def append(k=None, b=None, qkv=FAKE, qn=None, kn=None, rows=100, pos=FAKE, ax=None, dt=D.F16, tokens=8, hq=32):
    return D.lib().dial_paged_kv_append(qkv, qn, kn, FAKE, FAKE, rows, pos, ax or axes(), k or kv(), b or batch(), FAKE, dt,
                                        tokens, hq, 1e-6, None)


def verify(logits=FAKE, dt=D.F16, probs=None, n=2, rows=8, vocab=100, max_q=4, ws=FAKE, nbytes=1 << 40, ids=FAKE):
    return D.lib().dial_verify_drafts(logits, dt, ids, probs, FAKE, n, FAKE, FAKE, FAKE, FAKE, FAKE, None, rows, vocab, max_q,
                                      ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(format=3), 1), (dict(format=2), 2), (dict(format=0), 2),
    (dict(format=7), 2), (dict(head_dim=64), 4), (dict(page_size=8), 4), (dict(page_size=48), 4), (dict(page_size=512), 4),
    (dict(page_size=0), 4), (dict(n_pages=0), 1), (dict(n_kv_heads=0), 1), (dict(n_pages=1 << 23), 4),
    (dict(n_pages=1 << 62), 4), (dict(k_pages=0x1008), 3), (dict(v_pages=0x1004), 3),
    (dict(format=3, k_scale=0x1000, v_scale=0x1004), 3)])
def test_bad_caches(bad, status):
    for call in (attention, append, lambda k: D.lib().dial_paged_kv_read(k, batch(), FAKE, FAKE, D.F16, 8, None)):
        assert call(kv(**bad)) == status, D.lib().dial_last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(block_table=None), 1), (dict(kv_len=None), 1), (dict(q_start=None), 1), (dict(n_seqs=0), 1), (dict(max_pages=0), 1),
    (dict(max_q=0), 1), (dict(max_kv=-1), 1), (dict(max_pages=1 << 26), 4), (dict(max_q=1 << 31), 4), (dict(n_seqs=1 << 25), 4)])
def test_bad_batches(bad, status):
    for call in (attention, append, lambda b: D.lib().dial_paged_kv_read(kv(), b, FAKE, FAKE, D.F16, 8, None)):
        r = call(b=batch(**bad)) if call in (attention, append) else call(batch(**bad))
        assert r == status, D.lib().dial_last_error()


def test_bad_attention_and_read_arguments():
    assert attention(q=None) == 1 and attention(out=None) == 1
    assert attention(dt=D.F32) == 2 and attention(dt=D.BF16) == 2
    assert attention(tokens=0) == 1 and attention(tokens=1 << 31) == 4
    assert attention(hq=12) == 4 and attention(hq=72) == 4 and attention(hq=0) == 4
    assert attention(scale=0.0) == 1 and attention(scale=float("nan")) == 1 and attention(scale=float("inf")) == 1
    assert attention(q=ctypes.c_void_p(0x1008)) == 3
    L = D.lib()
    assert L.dial_paged_attention(FAKE, None, batch(), FAKE, D.F16, 8, 32, 0.1, None) == 1
    assert L.dial_paged_kv_read(kv(), None, FAKE, FAKE, D.F16, 8, None) == 1
    assert L.dial_paged_kv_read(kv(), batch(), None, FAKE, D.F16, 8, None) == 1
    assert L.dial_paged_kv_read(kv(), batch(), FAKE, ctypes.c_void_p(0x1002), D.F16, 8, None) == 3


def test_bad_append_arguments():
    assert append(qkv=None) == 1 and append(pos=None) == 1 and append(qn=FAKE) == 1 and append(kn=FAKE) == 1
    assert append(rows=0) == 1 and append(rows=1 << 31) == 1
    assert append(hq=33) == 4 and append(dt=D.F32) == 2
    assert append(qkv=ctypes.c_void_p(0x1004)) == 3
    for ax in (axes(0), axes(5), axes(1, (63, 0, 0, 0)), axes(2, (60, 5, 0, 0)), axes(2, (70, -6, 0, 0)),
               axes(3, (0, 32, 32, 0), 1), axes(1, (32, 32, 0, 0))):
        assert append(ax=ax) == 1, D.lib().dial_last_error()
    assert D.lib().dial_paged_kv_append(FAKE, None, None, FAKE, FAKE, 10, FAKE, None, kv(), batch(), FAKE, D.F16, 8, 32, 1e-6, None) == 1


def test_overlapping_results():
    L, at = D.lib(), lambda n: ctypes.c_void_p(0x10000 + n)
    size = 8 * 32 * 256
    for out in (at(0), at(size - 16), at(-size + 16)):
        assert attention(q=at(0), out=out) == 1 and b"overlap" in L.dial_last_error()
    for out in (at(0), at(8 * 8 * 256 - 16), at(-8 * 8 * 256 + 16)):
        assert L.dial_paged_kv_read(kv(), batch(), at(0), out, D.F16, 8, None) == 1 and b"overlap" in L.dial_last_error()
    for x in (FAKE, ctypes.c_void_p(0x1000 + size - 16), ctypes.c_void_p(0x1010)):
        assert append(qkv=x) == 1 and b"overlap" in L.dial_last_error()


def test_bad_verification_arguments():
    assert verify(logits=None) == 1 and verify(ids=None) == 1 and verify(ws=None) == 1
    assert verify(dt=5) == 2
    assert verify(rows=0) == 1 and verify(vocab=0) == 1 and verify(n=0) == 1 and verify(max_q=0) == 1
    assert verify(rows=1 << 31) == 4 and verify(vocab=1 << 31) == 4
    assert verify(vocab=(1 << 30) + 1) == 4 and D.lib().dial_verify_drafts_workspace_bytes(8, (1 << 30) + 1) == 0
    need = D.lib().dial_verify_drafts_workspace_bytes(8, 100)
    assert need > 0 and verify(nbytes=need - 1) == 1
    assert b"workspace" in D.lib().dial_last_error()
    assert verify(logits=ctypes.c_void_p(0x1002)) == 3 and verify(ws=ctypes.c_void_p(0x1008)) == 3
    assert verify(probs=ctypes.c_void_p(0x1004)) == 3
    assert D.lib().dial_verify_drafts_workspace_bytes(0, 5) == 0


def test_structs_have_the_headers_sizes():
    assert ctypes.sizeof(P._PagedKv) == 56 and ctypes.sizeof(P._PagedBatch) == 56 and ctypes.sizeof(P._RopeAxes) == 24


def test_front_end_takes_cuda_tensors_only():
    k = torch.zeros((4, 2, 16, 128), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.PagedKVCache.from_tensors(k, k.clone())
    with pytest.raises(ValueError, match="page_size"):
        P.PagedKVCache.from_tensors(k[:, :, :8].contiguous(), k[:, :, :8].contiguous())
    with pytest.raises(TypeError, match="f16"):
        P.PagedKVCache.from_tensors(k.float(), k.float())
    with pytest.raises(ValueError, match="k_scale"):
        P.PagedKVCache.from_tensors(k.to(torch.int8), k.to(torch.int8))
    t = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.PagedBatch(t, t[0, :2], t[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        P.verify_drafts(torch.zeros((2, 8)), t[0, :2], t[0], t[0, :2].float(), t[0, :2].float(), t[0, :2].float())
