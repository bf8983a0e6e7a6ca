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


@pytest.mark.parametrize("size", [40.0, 2000.0, 60000.0])
def test_scores_of_any_size(cuda, size):
    """Scores from some 10^7 to 4 * 10^10, positive and negative: where they differ, they differ by thousands, so
    the result is V of the largest (or the mean over equal ones), off by the roundings of P (2^-11) and of the
    result (2^-11) at most; sums and factors in fp32 are within the rest of 2^-9."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(int(size))
    n, hq, hkv, page = 700, 6, 1, 16
    u = rng.choice([-1.0, 1.0], D)
    c = R.Cache(rng, [0], hkv, page, max_len=n)
    k = (rng.choice([-1.0, 1.0], (n, 1, 1)) * rng.uniform(20000, 60000, (n, 1, 1)) * u).astype(np.float16)
    k[0] = -u * 50000  # the first position sees a negative score alone
    rows = c._write(c.k_np, 0, 0, k), c._write(c.v_np, 0, 0, rng.normal(0, 1, (n, hkv, D)).astype(np.float16))
    c.k, c.v = _cu(c.k_np), _cu(c.v_np)
    q = np.repeat((u * size).astype(np.float16)[None], hq, 0)
    seq = torch.tensor([n], dtype=torch.int32, device="cuda")

    def check(got, length, what):
        want, _ = R.attend(q, *rows, length)
        got = got.cpu().numpy().reshape(hq, D).astype(np.float64)
        assert np.isfinite(got).all(), f"{what}: not finite"
        assert (np.abs(got - want) <= 2.0 ** -9 * np.abs(rows[1][:length]).max(0)).all(), what

    qd = _cu(q.reshape(1, -1))
    for n_splits, max_len in ((1, n), (3, n), (9, c.max_seq_len)):
        out = torch.empty(1, hq * D, dtype=torch.float16, device="cuda")
        K.gqa_decode_attention_q4(qd, c.k, c.v, c.bt, seq, out, _ws(K.attention_q4_workspace_size(1, hq, D, n_splits)),
                                  page, hq, hkv, D, max_len, n_splits)
        check(out, n, f"decode, {n_splits} splits")
    for n_splits in (1, 3):
        e, out = _err(), torch.empty(n, hq * D, dtype=torch.float16, device="cuda")
        K.prefill_attention_q4(qd.repeat(n, 1), c.k, c.v, c.bt, out, 1, n, page, hq, hkv, D, c.max_seq_len,
                               workspace=_ws(K.prefill_q4_workspace_size(1, n, hq, D, n_splits)), n_splits=n_splits,
                               error=e)
        assert e.item() == 0
        for i in [0, 1, 2, 5, 31, 63, 64, 65, 127, 128, 300, n - 1]:
            check(out[i], i + 1, f"prefill, {n_splits} splits, query {i}")


@pytest.mark.parametrize("lens,hq,hkv,page,n_splits,max_len", [
    # one CTA a row: of 8 warps, of 4
    ([1, 31, 33, 300], 12, 2, 16, 1, 300), ([(29 * i) % 700 for i in range(160)], 2, 1, 48, 1, 700),
    # clusters of 2, 3, 8
    ([513, 64, 65], 12, 2, 64, 2, 2560), ([700, 95, 0, 96], 8, 8, 32, 3, 3840), ([1000, 257], 7, 1, 16, 8, 1008),
    # pieces: long shares across the rows, rows shorter than a share, fewer units than shares, one row
    ([20000, 0, 9000], 12, 2, 64, 9, 20032), ([0, 1, 127, 128, 129, 255, 256, 257, 640, 2000, 0, 5], 8, 4, 16, 11, 2016),
    ([(37 * i) % 300 for i in range(250)], 2, 2, 16, 9, 304), ([9000], 16, 2, 64, 1024, 9024),
    ([3] * 40, 6, 1, 16, 10, 16),
    # many shares to a row, and borders inside some of them
    ([3000, 2000, 2500], 8, 4, 32, 100, 3008), ([4000, 3000, 3500, 2500], 6, 1, 64, 30, 4032),
])
def test_decode_loses_and_doubles_no_step(cuda, lens, hq, hkv, page, n_splits, max_len):
    """Every way of sharing rows out, under a tolerance that a step of 32 positions lost, doubled or read from its
    neighbour leaves (test_kv_q4_accuracy_cpu.py)."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(len(lens) + hq)
    c = R.Cache(rng, lens, hkv, page)
    B, max_pages = len(lens), -(-max_len // page)
    c.bt = torch.nn.functional.pad(c.bt, (0, max(0, max_pages - c.bt.shape[1])))
    q = rng.normal(0, 1, (B, hq, D)).astype(np.float16)
    assert K.attention_q4_launches(n_splits, max_len) == (1 if n_splits <= 8 else 2)
    buf, out = _guarded(B, hq * D)
    e = _err()
    K.gqa_decode_attention_q4(_cu(q.reshape(B, -1)), c.k, c.v, c.bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                              out, _ws(K.attention_q4_workspace_size(B, hq, D, n_splits)), page, hq, hkv, D,
                              max(max_len, max(lens)), n_splits, error=e)
    assert e.item() == 0 and _guards_ok(buf)
    got = out.cpu().numpy().reshape(B, hq, D)
    for b in range(B):
        T.close(got[b], *T.attend(q[b], *c.rows[b], lens[b]), f"row {b}, length {lens[b]}")
        if lens[b] == 0:
            assert (got[b] == 0).all()


def test_step_loses_no_position(cuda):
    """The decode step's own position and all before it, in one CTA a row, a cluster and pieces."""
    from llamamps_b200 import kernels as K
    from tests.test_kv_q4_gpu import _inv
    rng = np.random.default_rng(41)
    lens, hq, hkv, page = [1, 33, 1000, 640], 12, 2, 32
    for n_splits, max_len in ((1, 1024), (4, 1024), (9, 1024)):
        c = R.Cache(rng, [n - 1 for n in lens], hkv, page, max_len=max_len)
        qkv = rng.normal(0, 1, (4, hq + 2 * hkv, D)).astype(np.float16)
        seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
        buf, out = _guarded(4, hq * D)
        e = _err()
        K.gqa_decode_attention_rope_q4(_cu(qkv.reshape(4, -1)), seq - 1, _cu(_inv()), c.k, c.v, c.bt, seq, out,
                                       _ws(K.attention_q4_workspace_size(4, hq, D, n_splits)), page, hq, hkv, D,
                                       max_len, n_splits, error=e)
        assert e.item() == 0 and _guards_ok(buf)
        # the rotated q as the append gives it (the step's attention has the same bits)
        q = torch.empty_like(out)
        K.rope_kv_append_q4(_cu(qkv.reshape(4, -1)), seq - 1, _cu(_inv()), q, c.k.clone(), c.v.clone(), c.bt, page, hq,
                            hkv, D)
        q = q.cpu().numpy().reshape(4, hq, D)
        rot = R.rotate(qkv[:, hq:hq + hkv], np.array(lens) - 1, _inv(), 0)
        got = out.cpu().numpy().reshape(4, hq, D)
        for b in range(4):
            k, v = (np.concatenate([old, R.values(*R.quantise(new))[None]])
                    for old, new in zip(c.rows[b], (rot[b], qkv[b, hq + hkv:])))
            T.close(got[b], *T.attend(q[b], k, v, lens[b]), f"length {lens[b]}, {n_splits} splits")
