"""The tight tolerance of tests/_kv_q4_tight.py on the CPU: restatements of the decode attention's arithmetic in
32 and 16 bits stay inside it or leave it as they should, and mistakes planted in the oracle leave it."""
import numpy as np
import pytest

from tests import _kv_q4 as R
from tests import _kv_q4_tight as T

D = 128


def _values(x):
    """What the cache holds of fp16 rows [T, hkv, 128], and the scale of each element's group."""
    codes, scales = R.quantise(x.reshape(-1, D))
    return R.values(codes, scales).reshape(x.shape), np.repeat(scales, 32, axis=1).reshape(x.shape)


def _decode(q, k, v, vs, warps, exact_v):
    """One head over its positions as the decode kernel goes about it: warp w takes every `warps`-th step of 32
    positions with its running maximum; P as fp16 times 2^15 over exact V, or (not exact_v) P times V's scales as
    fp16 over codes."""
    f32, f16 = np.float32, np.float16
    n, states = len(k), []
    s = (k @ q * T.SCALE * 1.4426950408889634).astype(f32)
    bias = f32(15.0 if exact_v else 0.0)
    for w in range(warps):
        m, l, o = f32(-np.inf), f32(0), np.zeros(D, f32)
        for p in range(32 * w, n, 32 * warps):
            z = s[p:p + 32]
            new = max(m, z.max())
            o, l, m = o * np.exp2(m - new), l * np.exp2(m - new), new
            e = np.exp2(z - m + bias)
            l += e.sum(dtype=f32)
            if exact_v:
                o += (e.astype(f16).astype(f32)[:, None] * v[p:p + 32].astype(f32)).sum(0, dtype=f32)
            else:
                pv = (e[:, None] * vs[p:p + 32].astype(f32)).astype(f16).astype(f32)
                o += (pv * (v[p:p + 32] / vs[p:p + 32]).astype(f32)).sum(0, dtype=f32)
        states.append((m, l, o))
    M = max(m for m, _, _ in states)
    f = [np.exp2(m - M) for m, _, _ in states]
    return (sum(o * x for (_, _, o), x in zip(states, f)) / sum(l * x for (_, l, _), x in zip(states, f))).astype(f16)


@pytest.mark.parametrize("n,warps,gain", [(131, 8, 1.0), (131, 8, 0.001), (2048, 8, 0.02), (8000, 4, 1.0),
                                          (8000, 4, 0.1), (8000, 4, 0.01)])
def test_weights_survive_small_values(n, warps, gain):
    """Behind a strong first position P over exact V is inside the tolerance whatever V's size; P times V's scale
    as fp16 loses most of the others' share where V is small."""
    q, k, v = T.with_sink(np.random.default_rng(n), n, 1, 1, 0.98, gain)
    (k, _), (v, vs) = _values(k), _values(v)
    want, tol = T.attend(q, k, v, n)
    got = [_decode(q[0].astype(np.float64), k[:, 0], v[:, 0], vs[:, 0], warps, x) for x in (True, False)]
    assert not T.outside(got[0], want, tol)
    if gain <= 0.02:
        assert T.outside(got[1], want, tol)


@pytest.mark.parametrize("n", [300, 2000, 20000])
def test_lost_and_doubled_steps_stand_out(n):
    """A step of 32 positions left out, counted twice, or read from its neighbour, anywhere in a row, leaves the
    tolerance; so does one position too many or too few in a short row."""
    rng = np.random.default_rng(n)
    q = rng.normal(0, 1, (2, D)).astype(np.float16)
    k, v = (_values(rng.normal(0, 1, (n + 32, 1, D)).astype(np.float16))[0] for _ in range(2))
    want, tol = T.attend(q, k, v, n)
    every = np.arange(n)
    for p in (0, 32, n // 2 // 32 * 32, (n - 1) // 32 * 32 - 32, n - 32):
        lost, doubled = np.delete(every, every[p:p + 32]), np.append(every, every[p:p + 32])
        swapped = every.copy()
        swapped[p:p + 32] += 32 if p + 64 <= n else -32
        for rows in (lost, doubled, swapped):
            assert T.outside(R.attend(q, k[rows], v[rows], len(rows))[0], want, tol), p
    if n == 300:
        for m in (n - 1, n + 1):
            assert T.outside(R.attend(q, k, v, m)[0], want, tol)
