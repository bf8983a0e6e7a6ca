"""The 4-bit cache's attention under the tight tolerance of tests/_kv_q4_tight.py."""
import numpy as np
import pytest
import torch

from tests import _kv_q4 as R
from tests import _kv_q4_tight as T
from tests.test_kv_q4_gpu import _cu, _err, _guarded, _guards_ok, _ws

pytestmark = pytest.mark.gpu

D = 128


def _sink_cache(rng, lens, hq, hkv, page, weight, gain):
    """A cache whose rows have a strong first position, and their queries [B, hq, 128]."""
    c = R.Cache(rng, [0] * len(lens), hkv, page, max_len=max(lens))
    q, rows = [], []
    for b, n in enumerate(lens):
        qb, k, v = T.with_sink(rng, n, hq, hkv, weight, gain)
        q.append(qb)
        rows.append((c._write(c.k_np, b, 0, k), c._write(c.v_np, b, 0, v)))
    c.rows, c.k, c.v = rows, _cu(c.k_np), _cu(c.v_np)
    return c, np.stack(q)


@pytest.mark.parametrize("gain", [1.0, 0.1, 0.01, 0.001])
@pytest.mark.parametrize("lens,hq,hkv,page,n_splits,max_len", [
    ([131], 12, 2, 64, 1, 131),                       # one CTA of 8 warps a row
    ([2500] + [40] * 79, 2, 2, 16, 1, 2500),          # one CTA of 4 warps
    ([2049, 700], 6, 1, 64, 4, 2112),                 # clusters
    ([8000, 33, 3000], 12, 2, 64, 9, 12000),          # pieces
])
def test_decode_behind_a_sink(cuda, gain, lens, hq, hkv, page, n_splits, max_len):
    """A first position that takes nearly all of the weight and has a small V, the others' V of any size: their
    share of the result survives (decode in every way of sharing a row out, and the prefill of the same query)."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(len(lens) + lens[0])
    c, q = _sink_cache(rng, lens, hq, hkv, page, 0.98, gain)
    B, max_len = len(lens), min(max_len, c.max_seq_len) if n_splits < 9 else max_len
    c.bt = torch.nn.functional.pad(c.bt, (0, max(0, -(-max_len // page) - c.bt.shape[1])))
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert K.attention_q4_launches(n_splits, max_len) == (2 if n_splits == 9 else 1)
    buf, out = _guarded(B, hq * D)
    e = _err()
    K.gqa_decode_attention_q4(_cu(q.reshape(B, -1)), c.k, c.v, c.bt, seq, out,
                              _ws(K.attention_q4_workspace_size(B, hq, D, n_splits)), page, hq, hkv, D, max_len,
                              n_splits, error=e)
    other = torch.empty_like(out)
    K.prefill_attention_q4(_cu(q.reshape(B, -1)), c.k, c.v, c.bt, other, B, 1, page, hq, hkv, D, max_len,
                           starts=seq - 1, error=e)
    assert e.item() == 0 and _guards_ok(buf)
    for b in sorted({0, 1 % B, B - 1}):
        T.close(out[b].cpu().numpy(), *T.attend(q[b], *c.rows[b], lens[b]), f"decode, length {lens[b]}")
        T.close(other[b].cpu().numpy(), *T.attend(q[b], *c.rows[b], lens[b], 2.0 ** -32, 16), f"prefill, length {lens[b]}")
