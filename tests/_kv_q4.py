"""The 4-bit KV cache restated in 64 bits for the tests: row format, quantiser,
rotation and attention, straight from their definitions (loops over groups,
sequences and heads; nothing shared with the package)."""
import numpy as np
import torch

D, ROW = 128, 72


def round_up_8_bits(v):
    """Smallest number >= v with 8 significant bits that is a multiple of 2^-24 (fp64 array, v >= 0)."""
    v = np.asarray(v, np.float64)
    m, e = np.frexp(v)
    s = np.ldexp(np.ceil(m * 256.0), e - 8)
    return np.where(s < 2.0 ** -16, np.ceil(s * 2.0 ** 24) * 2.0 ** -24, s)


def quantise(rows):
    """fp16 [n, 128] -> (codes int [n, 128], scales fp64 [n, 4]); NaN scales for a row that is not finite."""
    x = np.asarray(rows, np.float16).astype(np.float64).reshape(-1, 4, 32)
    bad = ~np.isfinite(x).all(axis=(1, 2))
    x = np.where(bad[:, None, None], 0.0, x)
    a = np.abs(x).max(axis=2)
    s = np.minimum(round_up_8_bits(a / 7.0), 9344.0)
    s = np.where(a == 0, 1.0, s)
    codes = np.clip(np.rint(x / s[..., None]), -7, 7).astype(np.int64).reshape(-1, D)
    return codes, np.where(bad[:, None], np.nan, s)


def row_bytes(codes, scales):
    """(code bytes [n, 64], scale bytes [n, 8])."""
    n = (codes + 8).astype(np.uint8)
    return n[:, 0::2] | (n[:, 1::2] << 4), scales.astype(np.float16).view(np.uint8).reshape(-1, 8)


def values(codes, scales):
    return codes * np.repeat(scales, 32, axis=1)


def rotate_exact(x, pos, inv_freq, style):
    """fp16 [n, heads, 128] at positions pos [n]: the rotation in 64 bits, and |x1| + |x2| of each element's pair."""
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(inv_freq, np.float32).astype(np.float64)
    c, s = np.cos(a), np.sin(a)
    x = np.asarray(x, np.float16).astype(np.float64)
    out, size = np.empty_like(x), np.empty_like(x)
    i1, i2 = (np.arange(0, D, 2), np.arange(1, D, 2)) if style == 0 else (np.arange(64), np.arange(64, D))
    out[..., i1] = x[..., i1] * c - x[..., i2] * s
    out[..., i2] = x[..., i1] * s + x[..., i2] * c
    size[..., i1] = size[..., i2] = np.abs(x[..., i1]) + np.abs(x[..., i2])
    return out, size


def rotate(x, pos, inv_freq, style):
    """The rotation rounded to fp16 (through fp32, as K is before it is quantised)."""
    return rotate_exact(x, pos, inv_freq, style)[0].astype(np.float32).astype(np.float16)


class Cache:
    """One layer's pools on the GPU with permuted pages, every block filled with
    random bytes that would show if they were read (NaN scales)."""

    def __init__(self, rng, lens, hkv, page, spare_pages=3, max_len=None, gain=1.0):
        self.hkv, self.page = hkv, page
        self.B = len(lens)
        self.pages = -(-max(max_len or max(max(lens), 1), 1) // page)
        self.max_seq_len = self.pages * page
        n = self.B * self.pages + spare_pages
        order = rng.permutation(n)[:self.B * self.pages]
        self.bt_np = order.reshape(self.B, self.pages).astype(np.int32)
        blocks = rng.integers(0, 256, (n, hkv, page * ROW), dtype=np.uint8)
        blocks[..., page * 64:] = 0xFF  # scales 0xFFFF: NaN
        self.rows = []  # per sequence (k, v) fp64 [T, hkv, 128]: the cached values
        for b, T in enumerate(lens):
            kv = []
            for half in range(2):
                kv.append((rng.normal(0, gain, (T, hkv, D)) *
                           np.exp(rng.normal(0, 0.5, (1, hkv, D)))).astype(np.float16))
            self.rows.append(kv)
        self.k_np, self.v_np = blocks, blocks.copy()
        out = []
        for b, T in enumerate(lens):
            out.append(tuple(self._write(pool, b, 0, x) for pool, x in zip((self.k_np, self.v_np), self.rows[b])))
        self.rows = out
        self.k, self.v = torch.from_numpy(self.k_np).cuda(), torch.from_numpy(self.v_np).cuda()
        self.bt = torch.from_numpy(self.bt_np).cuda()

    def _write(self, pool, b, start, x):
        """Quantises rows x [T, hkv, 128] into positions start.. of sequence b; returns their values."""
        T = x.shape[0]
        vals = np.zeros((T, self.hkv, D))
        if T == 0:
            return vals
        p = np.arange(start, start + T)
        pages, off = self.bt_np[b, p // self.page], p % self.page
        for h in range(self.hkv):
            codes, scales = quantise(x[:, h])
            vals[:, h] = values(codes, scales)
            cb, sb = row_bytes(codes, scales)
            for i in range(T):
                blk = pool[pages[i], h]
                blk[off[i] * 64:off[i] * 64 + 64] = cb[i]
                at = self.page * 64 + off[i] * 8
                blk[at:at + 8] = sb[i]
        return vals


SCALE = 0.088388


def attend(q, k, v, n, extra=()):
    """One query row [hq, 128] over the first n positions of k, v fp64 [T, hkv, 128].
    Returns (out [hq, 128], tolerance [hq, 128]).

    The tolerance, from the kernels' roundings (half a step each):
      * P times a V scale (or P) as fp16: 2^-11 of each term, and 2^-25 * 8 where
        it is subnormal (the largest P is 1, so the sum it is divided by is >= 1);
      * the result as fp16: 2^-11 of it, or 2^-25;
      * a score: 128 products and their group scales summed in fp32 by a tensor
        core that may truncate: 132 steps of 2^-23 of sum |q||k| 0.088388, on top
        of 2^-21 for the exponential and the base-2 scale; a score error moves
        numerator and denominator, so it counts twice."""
    hq, hkv = q.shape[0], k.shape[1]
    out, tol = np.zeros((hq, D)), np.zeros((hq, D))
    if n == 0:
        return out, tol
    q = np.asarray(q, np.float16).astype(np.float64)
    for h in range(hq):
        kk, vv = k[:n, h // (hq // hkv)], v[:n, h // (hq // hkv)]
        z = kk @ q[h] * SCALE
        p = np.exp(z - z.max())
        p /= p.sum()
        out[h] = p @ vv
        spread = p @ np.abs(vv)
        mag = (np.abs(kk) @ np.abs(q[h])).max() * SCALE
        dz = mag * 132 * 2.0 ** -23 + (np.abs(z).max() + 1) * 2.0 ** -21
        tol[h] = spread * (2.0 ** -11 + 2 * dz) * 1.01 + np.abs(out[h]) * 2.0 ** -11 + 2.0 ** -25 \
            + n * 8 * 2.0 ** -25
    return out, tol


def close(got, want, tol, what):
    got = np.asarray(got, np.float64).reshape(want.shape)
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - tol
    assert (over <= 0).all(), f"{what}: off by {np.abs(got - want).max():.3e}, {over.max():.3e} above the tolerance"
