"""A tolerance for the 4-bit cache's attention that follows the size of V and
shrinks with the number of positions, so that a lost or doubled step of a long
row, and weights lost where V is small, stand out of it."""
import numpy as np

D, SCALE = 128, 0.088388
H = 7.0  # an element is outside the sign bound below with a chance of 2 exp(-H^2 / 2) = 5e-11


def attend(q, k, v, n, floor=2.0 ** -40, chain=64):
    """One query row [hq, 128] over the first n positions of k, v fp64 [T, hkv, 128].
    Returns (out [hq, 128], tolerance [hq, 128]).  V's signs have to be random
    and independent of q and K.

    w = softmax weights, l = their sum before normalising, in units of the largest (>= 1).
      * Numerator.  Weight i enters as w_i (1 + a_i): 2^-11 for P as fp16 (half a
        step), dz for its score.  Given q and K the a_i are fixed numbers, so
        their effect sum_i a_i w_i v_i is a sum of fixed magnitudes under random
        signs: at most H (2^-11 + dz) sqrt(sum w_i^2 v_i^2) (Hoeffding).  P below
        fp16's normal numbers is off by at most `floor` of the largest weight:
        2^-25 under the scale that it is held at (times 2^15 in decode, 2^7 in
        prefill): floor sum |v_i| / l.
      * Denominator: dz, and fp32 sums of at most n / 8 + 64 terms: 2^-24 each.
      * O: fp32 sums of 16 products at a time whose adder may truncate: a chain of
        n / `chain` + 64 steps (decode: at least four warps to a row, prefill
        one accumulator: 16), 2^-22 each of what has been summed, whose size is
        |out| and the sign bound of a prefix.
      * dz, a score's error: 128 products and their group scales summed in fp32 by
        an adder that may truncate, 132 steps of 2^-23 of sum |q||k| 0.088388;
        2^-21 (|z| + 1) for the base-2 scale, the difference to the maximum and
        the exponential.
      * The result as fp16: 2^-11 of it, or 2^-25."""
    hq, hkv = q.shape[0], k.shape[1]
    out, tol = np.zeros((hq, D)), np.zeros((hq, D))
    if n == 0:
        return out, tol
    q = np.asarray(q, np.float16).astype(np.float64)
    for h in range(hq):
        kk, vv = k[:n, h // (hq // hkv)], v[:n, h // (hq // hkv)]
        z = kk @ q[h] * SCALE
        e = np.exp(z - z.max())
        l = e.sum()
        w = e / l
        out[h] = w @ vv
        dz = (np.abs(kk) @ np.abs(q[h])).max() * SCALE * 132 * 2.0 ** -23 + (np.abs(z).max() + 1) * 2.0 ** -21
        signs = np.sqrt((w * w) @ (vv * vv))
        size = np.abs(out[h])
        tol[h] = H * (2.0 ** -11 + dz) * signs * 1.01 + floor * np.abs(vv).sum(0) / l \
            + (dz + (n / 8 + 64) * 2.0 ** -24 + 2.0 ** -11) * size + 2.0 ** -25 \
            + (n / chain + 64) * 2.0 ** -22 * (size + H * signs)
    return out, tol


def outside(got, want, tol):
    """Whether some element is outside the tolerance (or not finite)."""
    got = np.asarray(got, np.float64).reshape(want.shape)
    return bool(not np.isfinite(got).all() or (np.abs(got - want) > tol).any())


def close(got, want, tol, what):
    got = np.asarray(got, np.float64).reshape(want.shape)
    assert np.isfinite(got).all(), f"{what}: not finite"
    off = np.abs(got - want)
    assert (off <= tol).all(), (f"{what}: off by up to {(off / tol).max():.2f} tolerances; relative to the norm "
                                f"{np.linalg.norm(got - want) / np.linalg.norm(want):.2e}")


def with_sink(rng, T, hq, hkv, weight, gain, sink_gain=0.02):
    """q [hq, 128] and fp16 k, v [T, hkv, 128]: position 0 takes about `weight` of every head's softmax and has a
    small V of its own (a first token, as models use it); the others have V of size `gain`."""
    G = hq // hkv
    u = rng.normal(0, 1, (hkv, D))
    q = (np.repeat(u, G, axis=0) + rng.normal(0, 0.1, (hq, D))).astype(np.float16)
    k = rng.normal(0, 1, (T, hkv, D))
    # the others' scores are N(0, 1): their exponentials sum to T e^0.5
    k[0] = u * (np.log(weight / (1 - weight) * T) + 0.5) / (np.square(u).sum(-1, keepdims=True) * SCALE)
    v = rng.normal(0, gain, (T, hkv, D))
    v[0] *= sink_gain
    return q, k.astype(np.float16), v.astype(np.float16)
