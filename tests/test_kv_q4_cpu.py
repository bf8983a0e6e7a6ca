"""Refusals of the 4-bit KV cache's entry points, before any device work (fake,
aligned addresses that are never dereferenced; CPU tensors at the Python layer)."""
import pytest
import torch

from llamamps_b200 import _lib
from llamamps_b200 import kernels as K

A = 1 << 20
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


def _append(**kw):
    v = {**dict(qkv=A, pos=A, inv=A, q=A, ko=None, vo=None, k=A, v=A, n_pages=4, bt=A, max_pages=2, page=64, hq=12,
                hkv=2, d=128, rows=1, style=0, err=None), **kw}
    return _lib.lib().lmps_rope_kv_append_q4(v["qkv"], v["pos"], v["inv"], v["q"], v["ko"], v["vo"], v["k"], v["v"],
                                             v["n_pages"], v["bt"], v["max_pages"], v["page"], v["hq"], v["hkv"],
                                             v["d"], v["rows"], v["style"], v["err"], None)


def _decode(**kw):
    v = {**dict(q=A, k=A, v=A, n_pages=4, bt=A, lens=A, out=A, ws=None, wsn=0, max_pages=2, page=64, hq=12, hkv=2,
                d=128, batch=1, max_len=128, splits=1), **kw}
    return _lib.lib().lmps_gqa_decode_attention_q4(v["q"], v["k"], v["v"], v["n_pages"], v["bt"], v["lens"], v["out"],
                                                   v["ws"], v["wsn"], v["max_pages"], v["page"], v["hq"], v["hkv"],
                                                   v["d"], v["batch"], v["max_len"], v["splits"], None, None)


def _step(**kw):
    v = {**dict(qkv=A, pos=A, inv=A, style=0, lens=A, max_len=128, splits=1), **kw}
    return _lib.lib().lmps_gqa_decode_attention_rope_q4(v["qkv"], v["pos"], v["inv"], v["style"], A, A, 4, A,
                                                        v["lens"], A, None, 0, 2, 64, 12, 2, 128, 1, v["max_len"],
                                                        v["splits"], None, None)


def _prefill(**kw):
    v = {**dict(q=A, k=A, v=A, n_pages=4, bt=A, starts=None, lens=None, out=A, ws=None, wsn=0, max_pages=2, page=64,
                hq=12, hkv=2, d=128, batch=1, seq=8, max_len=128, splits=1, err=A), **kw}
    return _lib.lib().lmps_prefill_attention_q4(v["q"], v["k"], v["v"], v["n_pages"], v["bt"], v["starts"], v["lens"],
                                                v["out"], v["ws"], v["wsn"], v["max_pages"], v["page"], v["hq"],
                                                v["hkv"], v["d"], v["batch"], v["seq"], v["max_len"], v["splits"],
                                                v["err"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), INVALID), (dict(pos=None), INVALID), (dict(inv=None), INVALID), (dict(q=None), INVALID),
    (dict(k=None), INVALID), (dict(bt=None), INVALID), (dict(rows=0), INVALID), (dict(n_pages=0), INVALID),
    (dict(max_pages=0), INVALID), (dict(page=0), INVALID), (dict(hkv=0), INVALID), (dict(style=2), INVALID),
    (dict(qkv=A + 8), INVALID), (dict(q=A + 2), INVALID), (dict(k=A + 8), INVALID), (dict(ko=A + 4), INVALID),
    (dict(max_pages=1 << 24), INVALID), (dict(d=64), UNSUPPORTED), (dict(page=24), UNSUPPORTED),
])
def test_append_refusals(kw, status):
    assert _append(**kw) == status


@pytest.mark.parametrize("call", [_decode, _prefill])
@pytest.mark.parametrize("kw,status", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(bt=None), INVALID),
    (dict(out=None), INVALID), (dict(batch=0), INVALID), (dict(n_pages=0), INVALID), (dict(max_len=0), INVALID),
    (dict(max_len=129), INVALID), (dict(hkv=5), INVALID), (dict(splits=0), INVALID), (dict(splits=1025), INVALID),
    (dict(q=A + 8), INVALID), (dict(k=A + 8), INVALID), (dict(v=A + 8), INVALID), (dict(out=A + 8), INVALID),
    (dict(max_pages=1 << 24), INVALID), (dict(d=64), UNSUPPORTED), (dict(page=40, max_len=64), UNSUPPORTED),
    (dict(hq=18), UNSUPPORTED), (dict(splits=2), WORKSPACE), (dict(splits=2, ws=A, wsn=100), WORKSPACE),
])
def test_attention_refusals(call, kw, status):
    assert call(**kw) == status


def test_refusals_of_one_form():
    assert _decode(lens=None) == INVALID and _decode(batch=65536) == INVALID
    assert _step(qkv=None) == _step(pos=None) == _step(inv=None) == _step(lens=None) == INVALID
    assert _step(style=-1) == INVALID and _step(max_len=129) == INVALID and _step(splits=2) == WORKSPACE
    assert _prefill(err=None) == INVALID and _prefill(seq=0) == INVALID
    assert _decode(splits=2, ws=A + 8, wsn=1 << 20) == INVALID


def test_sizes():
    assert K.attention_q4_workspace_size(3, 12, 128, 1) == 0
    assert K.attention_q4_workspace_size(3, 12, 128, 4) == 3 * 12 * 4 * (128 * 4 + 8) + 3 * 8
    assert K.attention_q4_splits(0, 2, 100) == K.prefill_q4_splits(0, 1, 12, 2, 100) == 1
    for b, n in ((1, 1), (1, 32768), (64, 8200), (300, 100)):
        assert 1 <= K.attention_q4_splits(b, 2, n) <= 1024


def test_python_layer_refuses_cpu_tensors():
    h, i = torch.float16, torch.int32
    pool, bt = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8), torch.zeros(1, 2, dtype=i)
    q, one = torch.zeros(1, 1536, dtype=h), torch.ones(1, dtype=i)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.gqa_decode_attention_q4(q, pool, pool, bt, one, q.clone(), None, 64, 12, 2, 128, 128, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rope_kv_append_q4(torch.zeros(1, 2048, dtype=h), one, torch.zeros(64), q, pool, pool, bt, 64, 12, 2, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.prefill_attention_q4(q, pool, pool, bt, q.clone(), 1, 1, 64, 12, 2, 128, 128)


def test_cache_rows_round_trip_on_the_host():
    """PagedKVCacheQ4 on CPU tensors: what it reads back is the restatement's quantisation of what was written."""
    import numpy as np

    from llamamps_b200.config import ModelConfig
    from llamamps_b200.kv_cache import PagedKVCacheQ4
    from tests import _kv_q4 as R
    cfg = ModelConfig(n_layers=2, n_q_heads=4, n_kv_heads=2)
    order = list(np.random.default_rng(0).permutation(2 * 4))
    kv = PagedKVCacheQ4(cfg, 2, max_batch=2, max_seq_len=60, page_size=16, device="cpu", page_order=order)
    rng = np.random.default_rng(1)
    k, v = (rng.normal(0, 2, (50, 256)).astype(np.float16) for _ in range(2))
    v[3, 5], k[7] = np.nan, 0
    kv.write_positions(1, 1, 0, torch.from_numpy(k[:20]), torch.from_numpy(v[:20]))
    kv.write_positions(1, 1, 20, torch.from_numpy(k[20:]), torch.from_numpy(v[20:]))
    got = kv.read_positions(1, 1, 50)
    for g, x in zip(got, (k, v)):
        want = R.values(*R.quantise(x.reshape(-1, 128))).reshape(50, 256)
        assert np.array_equal(g.numpy().astype(np.float64), want, equal_nan=True)
    assert kv.k.shape == (2, 8, 2, 16 * 72) and kv.k.dtype == torch.uint8
    blk = kv.k[1, kv.pages(1)[1], 1]                          # positions 16..31 of KV head 1
    codes, scales = R.quantise(k[16:32, 128:])
    cb, sb = R.row_bytes(codes, scales)
    assert np.array_equal(blk[:16 * 64].numpy().reshape(16, 64), cb)
    assert np.array_equal(blk[16 * 64:].numpy().reshape(16, 8), sb)
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCacheQ4(cfg, 1, 1, 64, page_size=40, device="cpu")
    with pytest.raises(ValueError, match="heads of 128"):
        PagedKVCacheQ4(ModelConfig(head_dim=64), 1, 1, 64, device="cpu")
    assert cfg.kv_bytes_per_position(4) * 32 == cfg.kv_bytes_per_position() * 9


def test_launch_counts():
    assert K.attention_q4_launches(1, 100000) == 1 and K.attention_q4_launches(8, 10240) == 1
    assert K.attention_q4_launches(8, 10241) == 2 and K.attention_q4_launches(9, 100) == 2
