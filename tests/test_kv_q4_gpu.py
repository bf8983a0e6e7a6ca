"""The 4-bit KV cache's kernels against their 64-bit restatement (tests/_kv_q4.py)."""
import numpy as np
import pytest
import torch

from tests import _kv_q4 as R

pytestmark = pytest.mark.gpu

D = 128


def _inv():
    from llamamps_b200.engine import rope_inv_freq
    return rope_inv_freq(D, 1e6)


def _cu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _err():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _guarded(rows, cols):
    """An fp16 output between guard rows, all 7."""
    buf = torch.full((rows + 2, cols), 7.0, dtype=torch.float16, device="cuda")
    return buf, buf[1:-1]


def _guards_ok(buf):
    return bool((buf[0] == 7).all()) and bool((buf[-1] == 7).all())


def _ws(n):
    return torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")  # stale partials would be NaN


# -- append ------------------------------------------------------------------
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("hq,hkv,page,ends", [
    (12, 2, 64, [1, 2, 64, 65, 1000]), (6, 1, 16, [16, 17, 33]), (16, 2, 48, [48, 49, 500]), (8, 8, 128, [129, 7]),
    (7, 1, 64, [32768]),
])
def test_append_bytes(cuda, style, hq, hkv, page, ends):
    """Cache bytes equal the restatement's everywhere (rows that the call does
    not name keep theirs), the values too; rotated q within its roundings."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(sum(ends) + hq + style)
    c = R.Cache(rng, [min(e - 1, 70) for e in ends], hkv, page, max_len=max(ends))
    B = len(ends)
    pos = np.array(ends, np.int32) - 1
    qkv = rng.normal(0, 2, (B, hq + 2 * hkv, D)).astype(np.float16)
    rot = R.rotate(qkv[:, :hq + hkv], pos, _inv(), style)
    k_vals = np.stack([c._write(c.k_np, b, int(pos[b]), rot[b:b + 1, hq:])[0] for b in range(B)])
    v_vals = np.stack([c._write(c.v_np, b, int(pos[b]), qkv[b:b + 1, hq + hkv:])[0] for b in range(B)])
    buf, q_out = _guarded(B, hq * D)
    k_out, v_out = (torch.zeros(B, hkv * D, dtype=torch.float16, device="cuda") for _ in range(2))
    e = _err()
    K.rope_kv_append_q4(_cu(qkv.reshape(B, -1)), _cu(pos), _cu(_inv()), q_out, c.k, c.v, c.bt, page, hq, hkv, D,
                        style, k_out=k_out, v_out=v_out, error=e)
    assert e.item() == 0 and _guards_ok(buf)
    assert np.array_equal(c.k.cpu().numpy(), c.k_np) and np.array_equal(c.v.cpu().numpy(), c.v_np)
    # q is rotated in fp32: 3 roundings of 2^-24 of |x1| + |x2|, then half a step of fp16
    exact, size = R.rotate_exact(qkv[:, :hq], pos, _inv(), style)
    off = np.abs(q_out.cpu().numpy().reshape(B, hq, D).astype(np.float64) - exact)
    assert (off <= np.abs(exact) * 2.0 ** -11 + size * 3 * 2.0 ** -24 * (1 + 2.0 ** -11) + 2.0 ** -25).all()
    assert np.array_equal(k_out.cpu().numpy().astype(np.float64).reshape(k_vals.shape), k_vals)
    assert np.array_equal(v_out.cpu().numpy().astype(np.float64).reshape(v_vals.shape), v_vals)


def test_append_special_rows(cuda):
    """Zero groups, subnormals, the largest numbers, exact ties, infinities and NaN."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(5)
    hq, hkv, page = 2, 1, 16
    rows = rng.normal(0, 1, (12, D)).astype(np.float16)
    rows[0] = 0
    rows[1, 32:64] = 0
    rows[2] *= np.float16(2.0 ** -20)                         # subnormal inputs
    rows[3] = np.float16(2.0 ** -24)                          # the smallest
    rows[4] = np.float16(65504.0) * np.sign(rows[4])          # 7 steps of 9344 fall short: clamped to +-7
    rows[5, ::2] = np.float16(65504.0)
    rows[6] = (np.arange(D) % 15 - 7) * 0.5                   # ties: scale 0.5, odd halves
    rows[6, :32] = np.where(np.arange(32) % 2, 3.5, 0.25)     # scale 0.5: 0.25 / 0.5 = 0.5 -> 0 (even)
    rows[7] = -0.0
    rows[8, 100] = np.inf
    rows[9, 3] = np.nan
    rows[10, 64] = -np.inf
    rows[11] = np.float16(6.1e-5)
    B = len(rows)
    c = R.Cache(rng, [0] * B, hkv, page, max_len=16)
    qkv = np.zeros((B, hq + 2 * hkv, D), np.float16)
    qkv[:, hq] = rows                                         # K at position 0: no rotation
    qkv[:, hq + 1] = rows[::-1]
    pos = np.zeros(B, np.int32)
    for b in range(B):
        c._write(c.k_np, b, 0, rows[b][None, None])
        c._write(c.v_np, b, 0, rows[::-1][b][None, None])
    k_out = torch.zeros(B, D, dtype=torch.float16, device="cuda")
    q_out = torch.zeros(B, hq * D, dtype=torch.float16, device="cuda")
    K.rope_kv_append_q4(_cu(qkv.reshape(B, -1)), _cu(pos), _cu(_inv()), q_out, c.k, c.v, c.bt, page, hq, hkv, D,
                        k_out=k_out)
    k, v = c.k.cpu().numpy(), c.v.cpu().numpy()
    # NaN scales: any NaN bits
    for got, want in ((k, c.k_np), (v, c.v_np)):
        assert np.array_equal(got[..., :page * 64], want[..., :page * 64])
        gs, ws = (x[..., page * 64:].copy().view(np.float16) for x in (got, want))
        assert np.array_equal(gs, ws, equal_nan=True)
    kv = k_out.cpu().numpy()
    assert np.isnan(kv[[8, 9, 10]]).all()
    fine = [0, 1, 2, 3, 4, 5, 6, 7, 11]
    want = R.values(*R.quantise(rows[fine]))
    assert np.array_equal(kv[fine].astype(np.float64), want)  # code * scale is exact in fp16
    # an element is off by at most half a scale; rounding up to 8 bits on a grid of 2^-24 gives
    # scale <= (max / 7) (1 + 2^-7) + 2^-24; the clamp at 9344 adds 65504 - 7 * 9344 = 96
    x = rows[fine].astype(np.float64)
    top = np.abs(x).reshape(-1, 4, 32).max(-1).repeat(32, -1)
    assert (np.abs(want - x) <= top / 14 * (1 + 2.0 ** -7) + 2.0 ** -25 + (top > 65000) * 96).all()


def test_append_skips_and_reports(cuda):
    """pos < 0 leaves a row alone; positions and pages outside the cache are reported and nothing is written."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(6)
    c = R.Cache(rng, [5, 5, 5, 5], 2, 16, max_len=48)
    c.bt[2, 0] = c.k.shape[0]                                 # one past the pool
    c.bt[3, 0] = -1
    before = c.k.clone(), c.v.clone()
    qkv = torch.randn(4, 16 * D, device="cuda").half()
    buf, q_out = _guarded(4, 12 * D)
    args = (_cu(_inv()), q_out, c.k, c.v, c.bt, 16, 12, 2, D)
    e = _err()
    K.rope_kv_append_q4(qkv, torch.tensor([-1, -5, -1, -2 ** 31], dtype=torch.int32, device="cuda"), *args, error=e)
    assert e.item() == 0 and bool((buf == 7).all())
    K.rope_kv_append_q4(qkv, torch.tensor([48, -1, 5, 5], dtype=torch.int32, device="cuda"), *args, error=e)
    assert e.item() == K.Q4_ERR_PAGE | K.Q4_ERR_POSITION and bool((buf == 7).all())
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])


# -- decode ------------------------------------------------------------------
DECODE = [
    ([1], 12, 2, 64), ([0, 1, 2, 15, 16, 17], 12, 2, 16), ([31, 32, 33, 63, 64, 65], 6, 1, 64),
    ([127, 128, 129, 300], 16, 2, 48), ([5, 700, 0, 96], 8, 8, 128), ([1000, 3], 7, 1, 32), ([4100], 12, 2, 64),
    ([257, 100], 5, 5, 16), ([90, 511], 32, 8, 80),
]


@pytest.mark.parametrize("lens,hq,hkv,page", DECODE)
def test_decode_attention(cuda, lens, hq, hkv, page):
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(sum(lens) * 3 + hq)
    c = R.Cache(rng, lens, hkv, page)
    B = len(lens)
    q = rng.normal(0, 1, (B, hq, D)).astype(np.float16)
    want = [R.attend(q[b], *c.rows[b], lens[b]) for b in range(B)]
    auto = K.attention_q4_splits(B, hkv, c.max_seq_len)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for n_splits in sorted({1, 2, 3, auto, 7, 40}):
        buf, out = _guarded(B, hq * D)
        e = _err()
        K.gqa_decode_attention_q4(_cu(q.reshape(B, -1)), c.k, c.v, c.bt, seq, out,
                                  _ws(K.attention_q4_workspace_size(B, hq, D, n_splits)), page, hq, hkv, D,
                                  c.max_seq_len, n_splits, error=e)
        assert e.item() == 0 and _guards_ok(buf)
        got = out.cpu().numpy().reshape(B, hq, D)
        for b in range(B):
            R.close(got[b], *want[b], f"length {lens[b]}, {n_splits} splits")
        if 0 in lens:
            assert (got[lens.index(0)] == 0).all()


@pytest.mark.parametrize("lens,hq,hkv,page,n_splits,max_len", [
    ([20000, 0, 9000], 12, 2, 64, 9, 20032),                                       # long shares across the rows
    ([0, 1, 127, 128, 129, 255, 256, 257, 640, 2000, 0, 5], 8, 4, 16, 11, 2016),   # shorter than a share
    ([(37 * i) % 300 for i in range(250)], 2, 2, 16, 9, 304),                      # more rows than shares
    ([9000], 16, 2, 64, 1024, 9024), ([3] * 40, 6, 1, 16, 10, 16),                 # fewer units than shares
])
def test_decode_shares_of_ragged_rows(cuda, lens, hq, hkv, page, n_splits, max_len):
    """Rows laid end to end and cut into equal shares: borders inside shares, rows shorter than one, empty ones."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(len(lens) + hq)
    c = R.Cache(rng, lens, hkv, page, max_len=max_len)
    B = len(lens)
    assert K.attention_q4_launches(n_splits, c.max_seq_len) == 2
    q = rng.normal(0, 1, (B, hq, D)).astype(np.float16)
    buf, out = _guarded(B, hq * D)
    e = _err()
    K.gqa_decode_attention_q4(_cu(q.reshape(B, -1)), c.k, c.v, c.bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                              out, _ws(K.attention_q4_workspace_size(B, hq, D, n_splits)), page, hq, hkv, D,
                              c.max_seq_len, n_splits, error=e)
    assert e.item() == 0 and _guards_ok(buf)
    got = out.cpu().numpy().reshape(B, hq, D)
    for b in range(B):
        R.close(got[b], *R.attend(q[b], *c.rows[b], lens[b]), f"length {lens[b]}")


def test_decode_shares_follow_the_lengths_in_a_graph(cuda):
    """The shares are cut from the lengths that the device holds when the call runs: a captured call replayed with
    other lengths gives the bits of an eager call, whatever the replay before it left in the workspace."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(31)
    B, hq, hkv, page, n_splits, longest = 40, 6, 1, 32, 9, 700
    c = R.Cache(rng, [longest] * B, hkv, page)
    q = _cu(rng.normal(0, 1, (B, hq * D)).astype(np.float16))
    seq = torch.full((B,), longest, dtype=torch.int32, device="cuda")
    ws, out = _ws(K.attention_q4_workspace_size(B, hq, D, n_splits)), torch.empty(B, hq * D, dtype=torch.float16, device="cuda")

    def call(o, w):
        K.gqa_decode_attention_q4(q, c.k, c.v, c.bt, seq, o, w, page, hq, hkv, D, 20000, n_splits)

    c.bt = torch.nn.functional.pad(c.bt, (0, 625 - c.bt.shape[1]), value=0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(out, ws)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(out, ws)
    for lens in ([longest] * B, [0] * B, [(61 * i) % longest for i in range(B)], [longest] + [1] * (B - 1), [0] * (B - 1) + [33]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(out)
        call(eager, torch.zeros_like(ws))
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))
        for b in (0, 1, B - 1):
            R.close(out[b].cpu().numpy(), *R.attend(q[b].cpu().numpy().reshape(hq, D), *c.rows[b], lens[b]), f"{b}, {lens[b]}")


def test_decode_large_scores_and_long_flat_softmax(cuda):
    """Scores that differ by hundreds (one position takes all) and equal scores (the mean of V)."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(8)
    lens, hq, hkv, page = [600, 2500], 12, 2, 64
    c = R.Cache(rng, lens, hkv, page, gain=6.0)
    q = np.zeros((2, hq, D), np.float16)
    q[0] = rng.normal(0, 8, (hq, D))
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for n_splits in (1, 5):
        out = torch.empty(2, hq * D, dtype=torch.float16, device="cuda")
        K.gqa_decode_attention_q4(_cu(q.reshape(2, -1)), c.k, c.v, c.bt, seq, out,
                                  _ws(K.attention_q4_workspace_size(2, hq, D, n_splits)), page, hq, hkv, D,
                                  c.max_seq_len, n_splits)
        for b in range(2):
            R.close(out[b].cpu().numpy().reshape(hq, D), *R.attend(q[b], *c.rows[b], lens[b]), f"sequence {b}")


def test_decode_nan_rows_reach_only_those_who_attend(cuda):
    """A NaN row of one sequence (as the append stores it) poisons that sequence's head alone; beyond a
    sequence's end anything may lie."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(9)
    lens, hq, hkv, page = [40, 40, 40], 12, 2, 16
    c = R.Cache(rng, lens, hkv, page)
    nan_k = np.full((1, hkv, D), np.nan, np.float16)
    c._write(c.k_np, 0, 39, nan_k)       # attended by sequence 0
    c._write(c.v_np, 1, 20, nan_k)       # attended by sequence 1
    c._write(c.k_np, 2, 40, nan_k)       # behind sequence 2's end
    c._write(c.v_np, 2, 41, nan_k)
    q = rng.normal(0, 1, (3, hq, D)).astype(np.float16)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for n_splits in (1, 2):
        out = torch.empty(3, hq * D, dtype=torch.float16, device="cuda")
        K.gqa_decode_attention_q4(_cu(q.reshape(3, -1)), _cu(c.k_np), _cu(c.v_np), c.bt, seq, out,
                                  _ws(K.attention_q4_workspace_size(3, hq, D, n_splits)), page, hq, hkv, D,
                                  c.max_seq_len, n_splits)
        got = out.cpu().numpy()
        assert np.isnan(got[0]).all() and np.isnan(got[1]).all()
        R.close(got[2], *R.attend(q[2], *c.rows[2], 40), "sequence 2")


def test_decode_bad_pages_and_lengths(cuda):
    """Pages outside the pool count as absent, lengths outside the cache are cut; both are reported."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(10)
    lens, hq, hkv, page = [100, 100], 12, 2, 16
    c = R.Cache(rng, lens, hkv, page, max_len=112)
    q = rng.normal(0, 1, (2, hq, D)).astype(np.float16)
    k0, v0 = c.rows[0]
    keep = np.r_[0:32, 48:100]
    c.bt[0, 2] = c.k.shape[0] + 5
    for n_splits in (1, 3):
        ws = _ws(K.attention_q4_workspace_size(2, hq, D, n_splits))
        e, out = _err(), torch.empty(2, hq * D, dtype=torch.float16, device="cuda")
        K.gqa_decode_attention_q4(_cu(q.reshape(2, -1)), c.k, c.v, c.bt,
                                  torch.tensor(lens, dtype=torch.int32, device="cuda"), out, ws, page, hq, hkv, D,
                                  c.max_seq_len, n_splits, error=e)
        assert e.item() == K.Q4_ERR_PAGE
        R.close(out[0].cpu().numpy(), *R.attend(q[0], k0[keep], v0[keep], len(keep)), "page left out")
        R.close(out[1].cpu().numpy(), *R.attend(q[1], *c.rows[1], 100), "sequence 1")
        e = _err()
        K.gqa_decode_attention_q4(_cu(q.reshape(2, -1)), c.k, c.v, c.bt,
                                  torch.tensor([-3, 1 << 30], dtype=torch.int32, device="cuda"), out, ws, page, hq,
                                  hkv, D, 96, n_splits, error=e)
        assert e.item() == K.Q4_ERR_POSITION and bool((out[0] == 0).all())
        R.close(out[1].cpu().numpy(), *R.attend(q[1], *c.rows[1], 96), "cut at max_seq_len")


# -- the decode step -----------------------------------------------------------
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("lens,hq,hkv,page,n_splits", [
    ([1, 16, 17], 12, 2, 16, 1), ([65, 1, 200, 128], 6, 1, 64, 3), ([1000, 33], 16, 2, 48, 5), ([129], 8, 8, 128, 2),
    ([300, 4], 7, 1, 32, 9),
])
def test_step_equals_append_then_attention(cuda, style, lens, hq, hkv, page, n_splits):
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(sum(lens) + hq)
    c = R.Cache(rng, [n - 1 for n in lens], hkv, page, max_len=max(lens))
    B = len(lens)
    ka, va = c.k.clone(), c.v.clone()
    qkv = _cu(rng.normal(0, 1, (B, (hq + 2 * hkv) * D)).astype(np.float16))
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = seq - 1
    inv = _cu(_inv())
    ws = _ws(K.attention_q4_workspace_size(B, hq, D, n_splits))
    q, ref = (torch.empty(B, hq * D, dtype=torch.float16, device="cuda") for _ in range(2))
    K.rope_kv_append_q4(qkv, pos, inv, q, ka, va, c.bt, page, hq, hkv, D, style)
    K.gqa_decode_attention_q4(q, ka, va, c.bt, seq, ref, ws, page, hq, hkv, D, c.max_seq_len, n_splits)
    buf, out = _guarded(B, hq * D)
    e = _err()
    K.gqa_decode_attention_rope_q4(qkv, pos, inv, c.k, c.v, c.bt, seq, out, ws, page, hq, hkv, D, c.max_seq_len,
                                   n_splits, style, error=e)
    assert e.item() == 0 and _guards_ok(buf)
    assert torch.equal(c.k, ka) and torch.equal(c.v, va)
    assert torch.equal(out.view(torch.int16), ref.view(torch.int16))
    assert bool(torch.isfinite(out).all())


# -- many queries a sequence ------------------------------------------------------
PREFILL = [
    # starts, q_lens, seq_len, hq, hkv, page
    (None, None, 1, 12, 2, 64), (None, None, 37, 12, 2, 64), ([0, 0], [130, 5], 130, 12, 2, 16),
    ([100, 0, 257], [3, 0, 64], 64, 6, 1, 48), ([63, 64, 65], [1, 1, 1], 1, 16, 2, 64), ([500], [70], 70, 7, 1, 32),
    ([31, 1], [20, 33], 40, 8, 8, 16), ([10], [43], 43, 5, 5, 64), ([2000], [17], 17, 12, 2, 64),
    ([129, 20], [90, 128], 128, 32, 8, 128),
]


@pytest.mark.parametrize("starts,q_lens,seq,hq,hkv,page", PREFILL)
def test_prefill_attention(cuda, starts, q_lens, seq, hq, hkv, page):
    from llamamps_b200 import kernels as K
    B = len(starts) if starts else 2
    s_np, n_np = starts or [0] * B, q_lens or [seq] * B
    rng = np.random.default_rng(seq * 7 + hq + sum(s_np))
    c = R.Cache(rng, [s + n for s, n in zip(s_np, n_np)], hkv, page, max_len=max(s_np) + seq + 5)
    q = rng.normal(0, 1, (B, seq, hq, D)).astype(np.float16)
    q[0, 0] *= 4
    i32 = dict(dtype=torch.int32, device="cuda")
    auto = K.prefill_q4_splits(B, seq, hq, hkv, c.max_seq_len)
    for n_splits in sorted({1, 2, 3, auto}):
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
            for i in range(seq):
                if i >= n_np[b]:
                    assert (got[b, i] == 7).all(), "a row behind the sequence was written"
                    continue
                R.close(got[b, i], *R.attend(q[b, i], *c.rows[b], s_np[b] + i + 1),
                        f"sequence {b}, query {i}, {n_splits} splits")


def test_prefill_nan_rows_and_bad_pages(cuda):
    """Whoever attends to a NaN row gets NaN, nobody before it does (the rows share tiles with it); a page
    outside the pool counts as absent and is reported; rows without a position are zeros."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(11)
    seq, hq, hkv, page = 150, 12, 2, 16
    c = R.Cache(rng, [150, 150, 150], hkv, page, max_len=160)
    nan = np.full((1, hkv, D), np.nan, np.float16)
    c._write(c.k_np, 0, 70, nan)
    c._write(c.v_np, 1, 131, nan)
    c.k, c.v = _cu(c.k_np), _cu(c.v_np)
    c.bt[2, 0] = c.k.shape[0]      # positions 0..15: query 0..15 has nothing left
    c.bt[2, 4] = -7                # positions 64..79
    q = rng.normal(0, 1, (3, seq, hq, D)).astype(np.float16)
    seen = np.ones(150, bool)
    seen[:16] = seen[64:80] = False
    for n_splits in (1, 2):
        e, out = _err(), torch.empty(3 * seq, hq * D, dtype=torch.float16, device="cuda")
        K.prefill_attention_q4(_cu(q.reshape(3 * seq, -1)), c.k, c.v, c.bt, out, 3, seq, page, hq, hkv, D,
                               c.max_seq_len, workspace=_ws(K.prefill_q4_workspace_size(3, seq, hq, D, n_splits)),
                               n_splits=n_splits, error=e)
        assert e.item() == K.Q4_ERR_PAGE
        got = out.cpu().numpy().reshape(3, seq, hq, D)
        for b, at in ((0, 70), (1, 131)):
            assert np.isnan(got[b, at:]).all()
            for i in (0, 1, at - 30, at - 1):
                R.close(got[b, i], *R.attend(q[b, i], *c.rows[b], i + 1), f"sequence {b}, query {i}")
        assert (got[2, :16] == 0).all()
        k, v = c.rows[2]
        for i in (16, 17, 63, 64, 79, 80, 149):
            keep = seen[:i + 1]
            n = int(keep.sum())
            R.close(got[2, i], *R.attend(q[2, i], k[:i + 1][keep], v[:i + 1][keep], n), f"query {i}")


def test_prefill_positions_outside_the_cache(cuda):
    """Queries past max_seq_len see what there is, queries before position 0 nothing; reported, nothing else read."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(12)
    seq, hq, hkv, page = 40, 6, 1, 16
    c = R.Cache(rng, [96, 96, 96], hkv, page)
    q = rng.normal(0, 1, (3, seq, hq, D)).astype(np.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    e = _err()
    buf, out = _guarded(3 * seq, hq * D)
    K.prefill_attention_q4(_cu(q.reshape(3 * seq, -1)), c.k, c.v, c.bt, out, 3, seq, page, hq, hkv, D, 96,
                           starts=torch.tensor([80, -5, 2 ** 31 - 10], **i32),
                           q_lens=torch.tensor([40, 1000, -3], **i32), error=e)
    assert e.item() == K.Q4_ERR_POSITION and _guards_ok(buf)
    got = out.cpu().numpy().reshape(3, seq, hq, D)
    for i in (0, 15, 16, 39):
        R.close(got[0, i], *R.attend(q[0, i], *c.rows[0], min(81 + i, 96)), f"query {i}")
    assert (got[1, :5] == 0).all() and (got[2] == 7).all()
    for i in (5, 39):
        R.close(got[1, i], *R.attend(q[1, i], *c.rows[1], i - 4), f"query {i} from position -5")


def test_prefill_long_context_rows(cuda):
    """Chunk rows behind contexts of thousands of positions, through several tiles and rescales."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(13)
    starts, seq, hq, hkv, page = [3000, 777], 96, 12, 2, 64
    c = R.Cache(rng, [s + seq for s in starts], hkv, page, gain=2.0)
    # scores that grow with the position, so that the running max moves often
    q = rng.normal(0, 2, (2, seq, hq, D)).astype(np.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n_splits in (1, 3, K.prefill_q4_splits(2, seq, hq, hkv, c.max_seq_len)):
        e, out = _err(), torch.empty(2 * seq, hq * D, dtype=torch.float16, device="cuda")
        K.prefill_attention_q4(_cu(q.reshape(2 * seq, -1)), c.k, c.v, c.bt, out, 2, seq, page, hq, hkv, D,
                               c.max_seq_len, starts=torch.tensor(starts, **i32),
                               workspace=_ws(K.prefill_q4_workspace_size(2, seq, hq, D, n_splits)),
                               n_splits=n_splits, error=e)
        assert e.item() == 0
        got = out.cpu().numpy().reshape(2, seq, hq, D)
        for b in range(2):
            for i in range(0, seq, 19):
                R.close(got[b, i], *R.attend(q[b, i], *c.rows[b], starts[b] + i + 1), f"{b}, {i}, {n_splits}")


def test_prefill_many_pieces(cuda):
    """One long context beside two short ones is cut into more pieces than the lanes of a warp; pieces whose pages
    are all bad, the first one of the row among them, weigh nothing."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(14)
    starts, seq, hq, hkv, page, n_splits = [9000, 0, 5], 8, 12, 2, 64, 33
    c = R.Cache(rng, [s + seq for s in starts], hkv, page)
    q = rng.normal(0, 2, (3, seq, hq, D)).astype(np.float16)
    seen = np.ones(9008, bool)
    for bad in (0, 1, 70, 71, 72, 73):  # positions 0..127 and 4480..4735
        c.bt[0, bad] = -1
        seen[bad * page:(bad + 1) * page] = False
    e = _err()
    buf, out = _guarded(3 * seq, hq * D)
    K.prefill_attention_q4(_cu(q.reshape(3 * seq, -1)), c.k, c.v, c.bt, out, 3, seq, page, hq, hkv, D, c.max_seq_len,
                           starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                           workspace=_ws(K.prefill_q4_workspace_size(3, seq, hq, D, n_splits)), n_splits=n_splits,
                           error=e)
    assert e.item() == K.Q4_ERR_PAGE and _guards_ok(buf)
    got = out.cpu().numpy().reshape(3, seq, hq, D)
    for b in range(3):
        for i in range(seq):
            n = starts[b] + i + 1
            keep = seen[:n] if b == 0 else np.ones(n, bool)
            k, v = c.rows[b]
            R.close(got[b, i], *R.attend(q[b, i], k[:n][keep], v[:n][keep], int(keep.sum())), f"{b}, {i}")


# -- the calls around the kernels ---------------------------------------------------
def _all_calls(rng, c, lens, hq, hkv, page, out=None):
    """One call of each entry point on cache c, as functions of replaced arguments."""
    from llamamps_b200 import kernels as K
    B = len(lens)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    t = dict(qkv=_cu(rng.normal(0, 1, (B, (hq + 2 * hkv) * D)).astype(np.float16)), pos=seq - 1, inv=_cu(_inv()),
             q=_cu(rng.normal(0, 1, (B, hq * D)).astype(np.float16)), k=c.k, v=c.v, bt=c.bt, lens=seq,
             out=torch.full((B, hq * D), 7.0, dtype=torch.float16, device="cuda"), ws=None, err=_err(), page=page)

    def append(**kw):
        a = {**t, **kw}
        return K.rope_kv_append_q4(a["qkv"], a["pos"], a["inv"], a["out"], a["k"], a["v"], a["bt"], a["page"], hq, hkv,
                                   D, error=a["err"])

    def decode(**kw):
        a = {**t, **kw}
        return K.gqa_decode_attention_q4(a["q"], a["k"], a["v"], a["bt"], a["lens"], a["out"], a["ws"], a["page"], hq,
                                         hkv, D, c.max_seq_len, 1, error=a["err"])

    def step(**kw):
        a = {**t, **kw}
        return K.gqa_decode_attention_rope_q4(a["qkv"], a["pos"], a["inv"], a["k"], a["v"], a["bt"], a["lens"],
                                              a["out"], a["ws"], a["page"], hq, hkv, D, c.max_seq_len, 1,
                                              error=a["err"])

    def prefill(**kw):
        a = {**t, **kw}
        return K.prefill_attention_q4(a["q"], a["k"], a["v"], a["bt"], a["out"], B, 1, a["page"], hq, hkv, D,
                                      c.max_seq_len, starts=a["pos"], workspace=a["ws"], error=a["err"])
    return t, dict(append=append, decode=decode, step=step, prefill=prefill)


def test_argument_mistakes_are_named_and_nothing_runs(cuda):
    rng = np.random.default_rng(21)
    c = R.Cache(rng, [20, 30], 2, 16, max_len=48)
    t, calls = _all_calls(rng, c, [21, 31], 12, 2, 16)
    before = c.k.clone(), c.v.clone()
    used = dict(append=("qkv", "pos", "inv", "bt", "k", "v", "err"), decode=("q", "lens", "bt", "k", "v", "err"),
                step=("qkv", "pos", "inv", "lens", "bt", "k", "v", "err"), prefill=("q", "pos", "bt", "k", "v", "err"))
    for name, call in calls.items():
        for arg in used[name] + ("out",):
            good = t[arg]
            with pytest.raises(RuntimeError, match="CUDA"):
                call(**{arg: good.cpu()})
            with pytest.raises(TypeError):
                call(**{arg: good.to(torch.float64)})
            if good.dim() == 2:
                with pytest.raises(ValueError, match="contiguous"):
                    call(**{arg: torch.stack([good, good], dim=2)[..., 0]})
            if arg == "bt":
                with pytest.raises(ValueError, match="block_table"):
                    call(bt=good[:1])
            elif arg in ("k", "v"):
                with pytest.raises(ValueError, match="pools"):
                    call(**{arg: good[:, :1].contiguous()})
            elif arg != "err":
                with pytest.raises(ValueError, match="elements"):
                    call(**{arg: good.reshape(-1)[:-1].reshape(1, -1) if arg in ("q", "qkv") else good.reshape(-1)[:-1]})
        with pytest.raises(ValueError, match="pools"):
            call(page=32)
        with pytest.raises(AttributeError):
            call(out=None)
    torch.cuda.synchronize()
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1]) and bool((t["out"] == 7).all())
    with pytest.raises(RuntimeError, match="argument"):   # misaligned: the entry point itself refuses
        buf = torch.zeros(t["q"].numel() + 1, dtype=torch.float16, device="cuda")
        calls["decode"](q=buf[1:].view_as(t["q"]))


def test_side_stream_and_graph_replay(cuda):
    """The calls run on the caller's stream; captured, they follow lengths, positions and inputs that change
    between replays; two graphs may share a workspace."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(22)
    hq, hkv, page, lens = 12, 2, 16, [300, 41]
    c = R.Cache(rng, lens, hkv, page, max_len=400)
    B, n_splits = 2, 11
    i32 = dict(dtype=torch.int32, device="cuda")
    seq, pos = torch.tensor(lens, **i32), torch.tensor(lens, **i32) - 1
    qkv = _cu(rng.normal(0, 1, (B, 16 * D)).astype(np.float16))
    q = _cu(rng.normal(0, 1, (B * 5, hq * D)).astype(np.float16))
    inv, err = _cu(_inv()), _err()
    ws = _ws(max(K.attention_q4_workspace_size(B, hq, D, n_splits), K.prefill_q4_workspace_size(B, 5, hq, D, 3)))
    outs = [torch.zeros(B, hq * D, dtype=torch.float16, device="cuda"),
            torch.zeros(B * 5, hq * D, dtype=torch.float16, device="cuda")]

    def one(i):
        if i == 0:
            K.gqa_decode_attention_rope_q4(qkv, pos, inv, c.k, c.v, c.bt, seq, outs[0], ws, page, hq, hkv, D,
                                           c.max_seq_len, n_splits, error=err)
        else:
            K.prefill_attention_q4(q, c.k, c.v, c.bt, outs[1], B, 5, page, hq, hkv, D, c.max_seq_len, starts=pos - 4,
                                   workspace=ws, n_splits=3, error=err)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in (0, 1):
            one(i)
        want = [o.clone() for o in outs]
        graphs = []
        for i in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                one(i)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        o.zero_()
    for i in (0, 1, 1, 0):
        graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    # the next position, another query
    pos.add_(1)
    seq.add_(1)
    qkv.copy_(torch.randn_like(qkv))
    q.copy_(torch.randn_like(q))
    for g in graphs:
        g.replay()
    got = [o.clone() for o in outs]
    kept = c.k.clone(), c.v.clone()
    for i in (0, 1):
        one(i)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, got)) and err.item() == 0
    assert torch.equal(c.k, kept[0]) and torch.equal(c.v, kept[1])


def test_append_decode_and_chunk_run_as_used(cuda):
    """A prompt appended and attended, a chunk behind it, then decode steps, on one cache: every stage's
    attention against the 64-bit restatement on what the cache holds."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(23)
    hq, hkv, page, B, P, C = 12, 2, 16, 2, 37, 21
    total = P + C + 3
    c = R.Cache(rng, [0] * B, hkv, page, max_len=total)
    inv, err = _cu(_inv()), _err()
    held = [(np.zeros((total, hkv, D)), np.zeros((total, hkv, D))) for _ in range(B)]
    at = 0
    for n in (P, C):
        qkv = rng.normal(0, 1, (B * n, (hq + 2 * hkv) * D)).astype(np.float16)
        pos = torch.arange(at, at + n, dtype=torch.int32, device="cuda").repeat(B)
        q, out = (torch.zeros(B * n, hq * D, dtype=torch.float16, device="cuda") for _ in range(2))
        ko, vo = (torch.zeros(B * n, hkv * D, dtype=torch.float16, device="cuda") for _ in range(2))
        K.rope_kv_append_q4(_cu(qkv), pos, inv, q, c.k, c.v, c.bt.repeat_interleave(n, 0).contiguous(), page, hq, hkv,
                            D, k_out=ko, v_out=vo, error=err)
        for b in range(B):
            for half, x in zip(held[b], (ko, vo)):
                half[at:at + n] = x.view(B, n, hkv, D)[b].cpu().numpy()
        K.prefill_attention_q4(q, c.k, c.v, c.bt, out, B, n, page, hq, hkv, D, c.max_seq_len,
                               starts=torch.full((B,), at, dtype=torch.int32, device="cuda"), error=err)
        qn, got = q.cpu().numpy().reshape(B, n, hq, D), out.cpu().numpy().reshape(B, n, hq, D)
        for b in range(B):
            for i in range(0, n, 4):
                R.close(got[b, i], *R.attend(qn[b, i], *held[b], at + i + 1), f"chunk at {at}, query {i}")
        at += n
    for _ in range(3):
        qkv = rng.normal(0, 1, (B, hq + 2 * hkv, D)).astype(np.float16)
        pos = torch.full((B,), at, dtype=torch.int32, device="cuda")
        out = torch.zeros(B, hq * D, dtype=torch.float16, device="cuda")
        K.gqa_decode_attention_rope_q4(_cu(qkv.reshape(B, -1)), pos, inv, c.k, c.v, c.bt, pos + 1, out, None, page, hq,
                                       hkv, D, c.max_seq_len, 1, error=err)
        rot = R.rotate(qkv[:, :hq + hkv], [at] * B, _inv(), 0)
        for b in range(B):
            for half, x in zip(held[b], (rot[b, hq:], qkv[b, hq + hkv:])):
                half[at] = R.values(*R.quantise(x))
            R.close(out[b].cpu().numpy().reshape(hq, D), *R.attend(rot[b, :hq], *held[b], at + 1), f"step at {at}")
        at += 1
    assert err.item() == 0
