"""Calls of the 4-bit cache's kernels that fill the GPU: appends of more than 1024 rows (four tokens a CTA), and
prefill attention with several units of work a CTA."""
import numpy as np
import pytest
import torch

from tests import _kv_q4 as R
from tests import _kv_q4_tight as T
from tests.test_kv_q4_gpu import _cu, _err, _guarded, _guards_ok, _inv, _ws

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("rows,hq,hkv,page", [(1025, 12, 2, 64), (1026, 7, 1, 16), (1027, 8, 8, 48), (4099, 6, 1, 32)])
def test_append_of_many_rows(cuda, style, rows, hq, hkv, page):
    """Byte for byte the restatement's cache, values and rotated q, with skipped rows and rows whose page is not
    in the pool among the others of a CTA, and a number of rows that four does not divide."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(rows + style)
    B = 4
    lens = rng.permutation([rows - 3 * (rows // 4)] + [rows // 4] * 3)
    c = R.Cache(rng, [0] * B, hkv, page, max_len=int(lens.max()) + 200)
    start = rng.integers(0, 200, B)
    seq = np.repeat(np.arange(B), lens)
    pos = np.concatenate([s + np.arange(n) for s, n in zip(start, lens)]).astype(np.int32)
    qkv = rng.normal(0, 2, (rows, hq + 2 * hkv, D)).astype(np.float16)
    bt = c.bt_np[seq]
    gone = rng.choice(rows, 9, replace=False)   # their pages are not in the pool; the last row among the skipped
    skip = np.append(rng.choice(rows, 200, replace=False), rows - 1)
    for i, r in enumerate(gone):
        bt[r, pos[r] // page] = -1 if i % 2 else c.k.shape[0]
    pos[skip] = rng.choice([-1, -7, -2 ** 31], len(skip))
    live = np.setdiff1d(np.arange(rows), np.append(gone, skip))
    rot = R.rotate(qkv[live, hq:hq + hkv], pos[live], _inv(), style)
    want = {}
    for name, pool, x in (("k", c.k_np, rot), ("v", c.v_np, qkv[live, hq + hkv:])):
        codes, scales = R.quantise(x.reshape(-1, D))
        want[name] = R.values(codes, scales).reshape(len(live), hkv, D)
        cb, sb = (z.reshape(len(live), hkv, -1) for z in R.row_bytes(codes, scales))
        for i, r in enumerate(live):
            block, off = pool[bt[r, pos[r] // page]], pos[r] % page
            block[:, off * 64:off * 64 + 64] = cb[i]
            block[:, page * 64 + off * 8:page * 64 + off * 8 + 8] = sb[i]
    (qb, q_out), (kb, k_out), (vb, v_out) = _guarded(rows, hq * D), _guarded(rows, hkv * D), _guarded(rows, hkv * D)
    e = _err()
    K.rope_kv_append_q4(_cu(qkv.reshape(rows, -1)), _cu(pos), _cu(_inv()), q_out, c.k, c.v, _cu(bt), page, hq, hkv, D,
                        style, k_out=k_out, v_out=v_out, error=e)
    assert e.item() == (K.Q4_ERR_PAGE if np.setdiff1d(gone, skip).size else 0)
    assert _guards_ok(qb) and _guards_ok(kb) and _guards_ok(vb)
    assert np.array_equal(c.k.cpu().numpy(), c.k_np) and np.array_equal(c.v.cpu().numpy(), c.v_np)
    q, k, v = (x.cpu().numpy().reshape(rows, -1, D).astype(np.float64) for x in (q_out, k_out, v_out))
    assert np.array_equal(k[live], want["k"]) and np.array_equal(v[live], want["v"])
    # q is rotated in fp32: 3 roundings of 2^-24 of |x1| + |x2|, then half a step of fp16
    exact, size = R.rotate_exact(qkv[live, :hq], pos[live], _inv(), style)
    off = np.abs(q[live] - exact)
    assert (off <= np.abs(exact) * 2.0 ** -11 + size * 3 * 2.0 ** -24 * (1 + 2.0 ** -11) + 2.0 ** -25).all()
    rest = np.append(gone, skip)
    assert all((x[rest] == 7).all() for x in (q, k, v))


@pytest.mark.parametrize("starts,q_lens,seq,hq,hkv,page,splits", [
    # units of work: 204 and 400 (148 CTAs); ragged, so that some row blocks have one row tile and some none
    ([0, 500, 7, 129, 64, 1000], [700, 3, 0, 301, 699, 43], 700, 12, 2, 64, (1, 2)),
    ([(211 * i) % 900 for i in range(25)], [(97 * i + 40) % 513 for i in range(25)], 512, 8, 2, 16, (1, 3)),
    # one position a sequence beside one long context: more sequences than CTAs, pieces of all lengths
    ([4000] + [(13 * i) % 90 for i in range(159)], None, 1, 6, 1, 32, (1, 2)),
    # whole prompts, 3 units a CTA and a last round that few CTAs have
    (None, None, 600, 7, 1, 48, (1,)),
])
def test_prefill_with_several_units_a_cta(cuda, starts, q_lens, seq, hq, hkv, page, splits):
    from llamamps_b200 import kernels as K
    B = len(starts) if starts else 30
    s_np, n_np = starts or [0] * B, q_lens or [seq] * B
    units = -(-seq * (hq // hkv) // 256) * hkv * B
    assert units > 148
    rng = np.random.default_rng(B + seq)
    c = R.Cache(rng, [s + n for s, n in zip(s_np, n_np)], hkv, page, max_len=max(s_np) + seq)
    q = rng.normal(0, 1, (B, seq, hq, D)).astype(np.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n_splits in splits:
        buf, out = _guarded(B * seq, hq * D)
        e = _err()
        K.prefill_attention_q4(_cu(q.reshape(B * seq, -1)), c.k, c.v, c.bt, out, B, seq, page, hq, hkv, D,
                               c.max_seq_len, starts=torch.tensor(s_np, **i32) if starts else None,
                               q_lens=torch.tensor(n_np, **i32) if q_lens else None,
                               workspace=_ws(K.prefill_q4_workspace_size(B, seq, hq, D, n_splits)),
                               n_splits=n_splits, error=e)
        assert e.item() == 0 and _guards_ok(buf)
        got = out.cpu().numpy().reshape(B, seq, hq, D)
        for b in range(B):
            n = n_np[b]
            assert (got[b, n:] == 7).all(), "a row behind the sequence was written"
            assert np.isfinite(got[b, :n]).all()
            # the borders of row tiles and blocks, and some between
            at = {0, 1, n - 1, n // 2, *(x // (hq // hkv) + d for x in (127, 255, 511, 1023, 2047) for d in (0, 1))}
            for i in sorted(x for x in at if 0 <= x < n)[:: 1 if B < 10 else 3]:
                T.close(got[b, i], *T.attend(q[b, i], *c.rows[b], s_np[b] + i + 1, 2.0 ** -32, 16),
                        f"sequence {b}, query {i}, {n_splits} splits")
