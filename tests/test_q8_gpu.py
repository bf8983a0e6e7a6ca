"""The 8-bit linear layers' operators against their formulas in 64 bits."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from llamamps_b200 import kernels as K
from tests import _q8 as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(m, k, seed, spread=20.0):
    """Rows with a few far larger channels, a zero row and sizes from small to large."""
    g = _gen(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= 1.0 + spread * (torch.rand(k, generator=g, device="cuda") < 0.02).float()
    x *= torch.exp2(torch.randint(-6, 7, (m, 1), generator=g, device="cuda").float())
    if m > 2:
        x[m // 2] = 0
    return x.half()


SHAPES = [(1, 1), (1, 7), (3, 8), (1, 1536), (2, 31), (64, 1536), (257, 1536), (5, 768), (700, 64), (300, 1200),
          (2, 8960), (300, 8960), (1, 4480), (9, 1535), (600, 1535), (4, 333), (300, 2048), (300, 2056), (3, 16384),
          (2, 16392), (1, 40001), (5000, 8), (300, 512), (300, 256), (17, 264)]


# -- quantiser and norm -----------------------------------------------------------
@pytest.mark.parametrize("m,k", SHAPES)
def test_quantise_rows(cuda, m, k):
    x = _rows(m, k, m * 31 + k)
    values = torch.full((m, k), -3.0, dtype=torch.float16, device="cuda")
    codes, scales = K.quantise_rows_q8(x, values=values)
    assert codes.shape == (m, k) and codes.dtype == torch.int8 and (m == 1 or codes.stride(0) % 16 == 0)
    R.check_rows(x.double(), codes, scales, values, k)
    again, s2 = K.quantise_rows_q8(x)
    assert torch.equal(again, codes) and torch.equal(s2, scales)


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(cuda, m, k, residual):
    x, g = _rows(m, k, m * 17 + k), _gen(k)
    gamma = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).half()
    values = torch.empty(m, k, dtype=torch.float16, device="cuda")
    if residual:
        r = _rows(m, k, m + 5 * k, spread=3.0)
        if m > 4:
            r[4] = 0
        codes, scales, s = K.rms_norm_q8(x, gamma, EPS, residual=r, values=values)
        assert torch.equal(s, (r.float() + x.float()).half())
    else:
        s = x
        codes, scales = K.rms_norm_q8(x, gamma, EPS, values=values)
    # an element's square goes through at most k / 32 additions in its thread and 13 between threads
    R.check_rows(R.norm(s, gamma, EPS), codes, scales, values, k, additions=k / 32 + 13)


@pytest.mark.parametrize("m,k", [(7200, 776), (7200, 1024), (7200, 1536), (3600, 2048), (3600, 2312), (1800, 3584), (1800, 4096),
                                 (1800, 5120), (1800, 6152), (1800, 8960), (1800, 9216), (1800, 9224), (600, 1536), (300, 1032)])
@pytest.mark.parametrize("form", ["quantise", "values", "norm", "residual", "norm values", "residual values"])
def test_many_rows(cuda, m, k, form):
    """Rows enough to fill the device: more pieces a thread, by what a thread has to hold; each form against 64 bits."""
    x, gamma = _rows(m, k, m + k), 1 + _rows(1, k, 5)[0] / 4
    res = _rows(m, k, 7) if "residual" in form else None
    values = torch.empty(m, k, dtype=torch.float16, device="cuda") if "values" in form else None
    if "norm" in form or "residual" in form:
        out = K.rms_norm_q8(x, gamma, EPS, residual=res, values=values)
        s = x if res is None else out[2]
        assert res is None or torch.equal(s, x + res)
        # (two running sums a thread of four pairs a piece, at most six pieces; 13 additions between threads)
        R.check_rows(R.norm(s, gamma, EPS), out[0], out[1], values, k, additions=4 * 6 + 1 + 13)
    else:
        R.check_rows(x.double(), *K.quantise_rows_q8(x, values=values), values, k)


@pytest.mark.parametrize("m,k", [(1, 1536), (64, 1536), (300, 1536), (300, 1535), (5, 8960), (3, 20000), (300, 100)])
def test_strides_and_what_lies_between_rows(cuda, m, k):
    """Rows of larger buffers, odd strides and starts, sums in place; nothing outside the rows is written."""
    g = _gen(3)
    for off, more in ((0, 24), (1, 3), (8, 8)):
        def buffer(dtype, fill):
            return torch.full((m, k + off + more), fill, dtype=dtype, device="cuda")

        def rows(t):
            return t[:, off:off + k]
        bx, br, bv, bc = buffer(torch.float16, 7), buffer(torch.float16, 9), buffer(torch.float16, 5), buffer(torch.int8, 77)
        x, r, v, c = rows(bx), rows(br), rows(bv), rows(bc)
        x.copy_(_rows(m, k, 11 + off))
        r.copy_(_rows(m, k, 12 + off))
        gamma = torch.randn(k + 1, generator=g, device="cuda").half()[1:].clone()
        want = (r.float() + x.float()).half()
        sc = torch.full((m + 2,), -1.0, device="cuda")
        K.rms_norm_q8(x, gamma, EPS, residual=r, sum_out=r, codes=c, scales=sc[1:1 + m], values=v)
        assert torch.equal(r, want)
        R.check_rows(R.norm(want, gamma, EPS), c, sc[1:1 + m], v, k, additions=k / 32 + 13)
        x2 = x.clone()
        K.rms_norm_q8(x, gamma, EPS, residual=r, sum_out=x, codes=c, scales=sc[1:1 + m], values=v)
        assert torch.equal(x, (r.float() + x2.float()).half())
        K.quantise_rows_q8(r, c, sc[1:1 + m], values=v)
        R.check_rows(want.double(), c, sc[1:1 + m], v, k)
        assert float(sc[0]) == -1 == float(sc[-1])
        for t, fill in ((bx, 7), (br, 9), (bv, 5), (bc, 77)):
            assert bool((t[:, :off] == fill).all()) and bool((t[:, off + k:] == fill).all())


@pytest.mark.parametrize("m,k", [(6, 1536), (400, 1536), (6, 8960), (6, 1535), (400, 40)])
def test_rows_that_are_not_finite_and_extremes(cuda, m, k):
    x = _rows(m, k, 5)
    x[0, k // 2], x[1, 0], x[2, k - 1] = float("nan"), float("inf"), -float("inf")
    x[3] = 65504.0
    x[4] = 2.0 ** -24
    x[5] = 0
    x[5, k // 3] = -65504.0
    gamma = torch.full((k,), 2.0, dtype=torch.float16, device="cuda")
    for codes, scales, y in (
            (*K.quantise_rows_q8(x), x.double()),
            (*K.rms_norm_q8(x, gamma, EPS), torch.where(torch.isfinite(x).all(dim=1)[:, None], R.norm(x, gamma, EPS),
                                                        torch.nan))):
        R.check_rows(y, codes, scales, None, k, additions=k / 32 + 13)
        assert bool(torch.isnan(scales[:3]).all()) and not bool(codes[:3].any())
        assert bool((codes[3:5] == 127).all()) and int(codes[5, k // 3]) == -127
    r = x.clone()
    r[3] = 65504.0  # the sum is infinite in fp16
    codes, scales, s = K.rms_norm_q8(x, gamma, EPS, residual=r)
    assert torch.equal(s[3:], (r.float() + x.float()).half()[3:]) and bool(torch.isnan(scales[:4]).all())
    zero = torch.zeros(2, k, dtype=torch.float16, device="cuda")
    codes, scales = K.rms_norm_q8(zero, gamma, 0.0)  # (eps 0: the norm itself is 0 / 0)
    assert not bool(codes.any()) and not bool(scales.any())
    gamma[7] = float("nan")
    assert bool(torch.isnan(K.rms_norm_q8(x, gamma, EPS)[1]).all())


@pytest.mark.parametrize("k", [1536, 1535, 8960, 77])
@pytest.mark.parametrize("norm", [False, True])
def test_ties_and_their_neighbours(cuda, k, norm):
    """Rows of elements at the ties h m / 127 and next to them: every code is the formula's, half to even (127 v and
    h m have 31 bits at most, so their comparison in 64 bits is exact)."""
    g, m = _gen(k), 64
    gamma = (torch.rand(k, generator=g, device="cuda") + 0.5).half() if norm else torch.ones(k, device="cuda").half()
    gamma[0] = 1.0
    top = (torch.rand(m, 1, generator=g, device="cuda") * 3 + 0.5).half()
    top[::4] = 254.0 * 2.0 ** torch.arange(-8, 8, device="cuda")[:m // 4, None].half()  # (odd multiples are ties)
    h = torch.randint(-127, 127, (m, k), generator=g, device="cuda").double() + 0.5
    s = (h * top.double() / 127 / gamma.double()).half()
    s = (s.view(torch.int16) + torch.randint(-1, 2, (m, k), generator=g, device="cuda").short()).view(torch.float16)
    s[:, :1] = top
    v = s.double() * gamma.double()
    most = v.abs().amax(dim=1, keepdim=True)
    c = torch.floor(127 * v / most)
    c = torch.where(127 * v - c * most < 0, c - 1, c)
    c = torch.where(127 * v - (c + 1) * most >= 0, c + 1, c)
    above = 127 * v - (c + 0.5) * most  # 0: a tie between c and c + 1
    want = torch.where(above == 0, c + c.remainder(2), c + (above > 0))
    assert norm or int((above == 0).sum()) > k // 4  # (few v = s gamma of 22 bits are ties)
    got = K.rms_norm_q8(s, gamma)[0] if norm else K.quantise_rows_q8(s)[0]
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("k", [1536, 2048, 8960, 1535])
def test_rows_of_calls_of_any_size(cuda, k):
    """Codes, the quantiser's scales and the sums are the same bits for 1 to 16384 rows.  The norm's scales are not:
    two orders of the additions in a sum of squares are each off by a rounding for each addition that an element goes
    through (k / 32 in a thread, 13 between threads), the scale by half of that and its other roundings."""
    m = 16384
    x, r, gamma = _rows(m, k, 3), _rows(m, k, 4), 1 + _rows(1, k, 5)[0] / 4
    codes, scales = K.quantise_rows_q8(x)
    ncodes, nscales, total = K.rms_norm_q8(x, gamma, EPS, residual=r)
    rel = 2 * ((k / 32 + 13) / 2 + 6) * 2.0 ** -24
    for a, b in ((0, 1), (5, 69), (100, 700), (7, 2007), (0, 5000), (m - 3, m)):
        c, s = K.quantise_rows_q8(x[a:b])
        assert torch.equal(c, codes[a:b]) and torch.equal(s, scales[a:b])
        c, s, t = K.rms_norm_q8(x[a:b], gamma, EPS, residual=r[a:b])
        assert torch.equal(c, ncodes[a:b]) and torch.equal(t, total[a:b])
        want = nscales[a:b].double()
        assert bool(((s.double() - want).abs() <= rel * want).all())


def test_vectors_and_no_rows(cuda):
    x = _rows(1, 1536, 1)[0]
    c, s = K.quantise_rows_q8(x)
    assert c.shape == (1536,) and s.shape == (1,)
    R.check_rows(x[None].double(), c[None], s, None, 1536)
    gamma = torch.ones(1536, dtype=torch.float16, device="cuda")
    c, s, total = K.rms_norm_q8(x, gamma, residual=x)
    assert total.shape == (1536,) and torch.equal(total, x + x)
    c, s = K.quantise_rows_q8(torch.empty(0, 1536, dtype=torch.float16, device="cuda"))
    assert c.shape == (0, 1536) and s.shape == (0,)
    w = R.rand_codes(48, 1536, _gen(1), "cuda")
    assert K.w8a8_gemm(c, s, w, torch.ones(48, device="cuda")).shape == (0, 48)


# -- the product -----------------------------------------------------------------
MS = [1, 2, 3, 4, 5, 8, 16, 17, 31, 33, 48, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 385, 513, 1000, 2100]
NK = [(1, 1), (7, 16), (64, 15), (128, 128), (129, 272), (200, 100), (257, 1000), (1536, 1536), (333, 1201),
      (1000, 257), (136, 4480)]


def _operands(m, n, k, seed, extra=0):
    g = _gen(seed)
    x, w = R.rand_codes(m, k, g, "cuda", extra=extra), R.rand_codes(n, k, g, "cuda", extra=2 * extra)
    xs = torch.exp(torch.randn(m, generator=g, device="cuda")) * 0.01
    ws = torch.exp(0.3 * torch.randn(n, generator=g, device="cuda")) * (0.02 / k ** 0.5)
    return g, x, xs, w, ws


@pytest.mark.parametrize("m", MS)
def test_gemm(cuda, m):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i, (n, k) in enumerate(NK):
        g, x, xs, w, ws = _operands(m, n, k, m + i, extra=i % 2)
        bias = torch.randn(n, generator=g, device="cuda").half() if i % 4 in (1, 3) else None
        res = torch.randn(m, n, generator=g, device="cuda").half() if i % 4 in (2, 3) else None
        y = K.w8a8_gemm(x, xs, w, ws, bias=bias, residual=res, error=err)
        R.check_linear(y, x, xs, w, ws, bias, res)
    assert int(err) == 0


@pytest.mark.parametrize("m", MS)
def test_gated(cuda, m):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i, (n, k) in enumerate(NK):
        _, x, xs, w, ws = _operands(m, 2 * n, k, m + 50 + i, extra=i % 2)
        y = K.w8a8_gemm(x, xs, w, ws * 5, swiglu=True, error=err)
        R.check_gated(y, x, xs, w, ws * 5)
    assert int(err) == 0


@pytest.mark.parametrize("m,n,k,gated", [(1, 2048, 1536, 0), (64, 1536, 8960, 0), (16, 8960, 1536, 1),
                                         (1024, 2048, 1536, 0), (700, 8960, 1536, 1), (2048, 1536, 8960, 0),
                                         (96, 17920, 1536, 0), (4100, 1537, 1000, 1), (9, 151936, 1536, 0)])
def test_model_shapes(cuda, m, n, k, gated):
    g, x, xs, w, ws = _operands(m, 2 * n if gated else n, k, 9)
    if gated:
        R.check_gated(K.w8a8_gemm(x, xs, w, ws, swiglu=True), x, xs, w, ws)
        return
    bias, res = (torch.randn(s, generator=g, device="cuda").half() for s in ((n,), (m, n)))
    R.check_linear(K.w8a8_gemm(x, xs, w, ws, bias=bias, residual=res), x, xs, w, ws, bias, res)


@pytest.mark.parametrize("m,n,k", [(129, 64, 8000), (200, 1536, 8960), (300, 128, 3200), (300, 131, 3101), (512, 1536, 4480),
                                   (600, 300, 1537), (700, 1000, 1601), (1000, 333, 2999), (2000, 256, 4000)])
@pytest.mark.parametrize("form", ["none", "both"])
def test_few_tiles_share_k_out(cuda, m, n, k, form):
    """Long K behind few tiles: shares of one step more or less, ragged last steps, with and without bias and residual."""
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g, x, xs, w, ws = _operands(m, n, k, m + k)
    bias, res = (torch.randn(s, generator=g, device="cuda").half() if form == "both" else None for s in ((n,), (m, n)))
    for _ in range(3):
        y = K.w8a8_gemm(x, xs, w, ws, bias=bias, residual=res, error=err)
        R.check_linear(y, x, xs, w, ws, bias, res)
    assert int(err) == 0


@pytest.mark.parametrize("m", [512, 768, 1024, 1100, 1280, 2048, 2100, 2560])
def test_as_many_tiles_as_clusters_fit(cuda, m):
    """K shared out by four pairs, by two, by none: the numbers of tiles around what a device holds at once."""
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g, x, xs, w, ws = _operands(m, 512, 3200, m)
    res = torch.randn(m, 512, generator=g, device="cuda").half()
    R.check_linear(K.w8a8_gemm(x, xs, w, ws, residual=res, error=err), x, xs, w, ws, None, res)
    assert int(err) == 0


FIRST_IN_A_GRAPH = """
import torch
from llamamps_b200 import kernels as K
from tests import _q8 as R
x, w = (R.padded(n, 3200, torch.int8, "cuda") for n in (300, 500))
x.random_(-127, 128), w.random_(-127, 128)
xs, ws = (torch.rand(n, device="cuda") * 2 ** -10 for n in (300, 500))
y, err = torch.zeros(300, 500, dtype=torch.float16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    K.w8a8_gemm(x, xs, w, ws, out=y, error=err)
for _ in range(2):
    y.zero_()
    graph.replay()
    R.check_linear(y, x, xs, w, ws)
assert int(err) == 0
"""


def test_the_first_call_of_a_process_may_be_captured(cuda):
    """What a call asks of the device once is asked inside a capture, too."""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("m,n,k,gated", [(5, 4000, 1000, 0), (14, 2500, 777, 1), (14, 300, 4000, 0), (30, 600, 500, 1),
                                         (30, 2500, 1600, 0), (8, 9000, 300, 1), (16, 1000, 256, 1)])
def test_few_tokens(cuda, m, n, k, gated):
    """The forms for few tokens, by weight rows and K: 8, 16 and 32 warps a tile."""
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g, x, xs, w, ws = _operands(m, 2 * n if gated else n, k, 3, extra=1)
    if gated:
        R.check_gated(K.w8a8_gemm(x, xs, w, ws, swiglu=True, error=err), x, xs, w, ws)
    else:
        R.check_linear(K.w8a8_gemm(x, xs, w, ws, error=err), x, xs, w, ws)
    assert int(err) == 0


@pytest.mark.parametrize("m", [33, 47, 64, 65, 99, 128])
@pytest.mark.parametrize("n,k,gated", [(9504, 333, 0), (9500, 333, 0), (9473, 1536, 0), (4737, 700, 1), (20000, 128, 0), (10000, 1000, 1)])
def test_wide_outputs(cuda, m, n, k, gated):
    """Wide outputs of a batch: whole tiles and ragged ones, one CTA an SM and more, with and without bias."""
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bias in (False, True)[:1 if gated else 2]:
        g, x, xs, w, ws = _operands(m, 2 * n if gated else n, k, m)
        off = 8 if m in (47, 99) else 3  # (rows at 16 bytes, or not)
        buf = torch.full((m, -(-n // 8) * 8 + 16), 3.0, dtype=torch.float16, device="cuda")
        y, b = buf[:, off:off + n], torch.randn(n, generator=g, device="cuda").half() if bias else None
        K.w8a8_gemm(x, xs, w, ws, bias=b, swiglu=bool(gated), out=y, error=err)
        z = K.w8a8_gemm(x, xs, w, ws, bias=b, swiglu=bool(gated), error=err)
        assert torch.equal(y, z) and bool((buf[:, :off] == 3).all()) and bool((buf[:, off + n:] == 3).all())
        if gated:
            R.check_gated(y, x, xs, w, ws)
        else:
            R.check_linear(y, x, xs, w, ws, b)
        assert torch.equal(K.w8a8_gemm(x[5:12], xs[5:12], w, ws, bias=b, swiglu=bool(gated), error=err), z[5:12])
    assert int(err) == 0


def test_two_streams_at_once(cuda):
    """Calls of every kind on two streams that overlap, each with its own operands, again and again."""
    shapes = [(3, 500, 640, False), (64, 640, 2048, False), (100, 512, 1024, True), (300, 512, 4096, False),
              (600, 700, 512, True), (1500, 1024, 768, False)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    ops, want, got = {}, {}, {}
    err = torch.zeros(2, dtype=torch.int32, device="cuda")
    for s in range(2):
        for i, (m, n, k, gated) in enumerate(shapes):
            _, x, xs, w, ws = ops[s, i] = _operands(m, 2 * n if gated else n, k, 100 * s + i)
            want[s, i] = K.w8a8_gemm(x, xs, w, ws, swiglu=gated)
            got[s, i] = [torch.empty_like(want[s, i]) for _ in range(4)]
    torch.cuda.synchronize()
    for rep in range(4):
        for i, (m, n, k, gated) in enumerate(shapes):
            for s in range(2):
                with torch.cuda.stream(sides[s]):
                    _, x, xs, w, ws = ops[s, (i + 3 * s) % len(shapes)]
                    j = (i + 3 * s) % len(shapes)
                    K.w8a8_gemm(x, xs, w, ws, swiglu=shapes[j][3], out=got[s, j][rep], error=err[s:s + 1])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[key]) for key in got for g in got[key]) and not bool(err.any())


def test_two_streams_of_wide_outputs_and_few_tokens(cuda):
    """Two streams that overlap, with the calls whose tokens are the tensor core's rows and those of few tokens in two
    and four tiles, pairs that share K out between them."""
    shapes = [(48, 9504, 512, False), (12, 2000, 768, False), (64, 4800, 512, True), (24, 1000, 768, True),
              (300, 512, 4096, False), (24, 2000, 333, False), (12, 1000, 512, True), (33, 9504, 3000, False)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    ops, want, got = {}, {}, {}
    err = torch.zeros(2, dtype=torch.int32, device="cuda")
    for s in range(2):
        for i, (m, n, k, gated) in enumerate(shapes):
            _, x, xs, w, ws = ops[s, i] = _operands(m, 2 * n if gated else n, k, 100 * s + i)
            want[s, i] = K.w8a8_gemm(x, xs, w, ws, swiglu=gated)
            (R.check_gated if gated else R.check_linear)(want[s, i], x, xs, w, ws)
            got[s, i] = [torch.full_like(want[s, i], 7.0) for _ in range(4)]
    torch.cuda.synchronize()
    for rep in range(4):
        for i in range(len(shapes)):
            for s in range(2):
                j = (i + 3 * s) % len(shapes)
                with torch.cuda.stream(sides[s]):
                    _, x, xs, w, ws = ops[s, j]
                    K.w8a8_gemm(x, xs, w, ws, swiglu=shapes[j][3], out=got[s, j][rep], error=err[s:s + 1])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[key]) for key in got for g in got[key]) and not bool(err.any())


@pytest.mark.parametrize("m", [1, 7, 40, 130, 300])
def test_largest_sums_and_extreme_codes(cuda, m):
    """Sums at the edge of 32 bits (k = 131071, all codes -128), and codes of one sign."""
    k = 131071
    x, w = R.padded(m, k, torch.int8, "cuda"), R.padded(40, k, torch.int8, "cuda")
    x.fill_(-128)
    w.fill_(-128)
    w[1::2] = 127
    xs, ws = torch.full((m,), 2.0 ** -14, device="cuda"), torch.full((40,), 2.0 ** -10, device="cuda")
    R.check_linear(K.w8a8_gemm(x, xs, w, ws), x, xs, w, ws)
    R.check_gated(K.w8a8_gemm(x, xs, w, ws * 2.0 ** -4, swiglu=True), x, xs, w, ws * 2.0 ** -4)


@pytest.mark.parametrize("m", [1, 40, 130, 300, 600])
@pytest.mark.parametrize("n", [200, 131])
def test_output_strides_in_place_and_overflow(cuda, m, n):
    """Rows of y in a larger buffer, y and residual the same, results past fp16, NaN rows of x."""
    k = 320
    g, x, xs, w, ws = _operands(m, n, k, m)
    for off, more in ((0, 8), (1, 2), (8, 16)):
        buf = torch.full((m, n + off + more), 3.0, dtype=torch.float16, device="cuda")
        y = buf[:, off:off + n]
        r = torch.randn(m, n, generator=g, device="cuda").half()
        y.copy_(r)
        assert K.w8a8_gemm(x, xs, w, ws, residual=y, out=y) is y
        R.check_linear(y, x, xs, w, ws, None, r)
        assert bool((buf[:, :off] == 3).all()) and bool((buf[:, off + n:] == 3).all())
    xs[m // 2] = float("nan")
    xs[0] = 1e6 if m > 1 else xs[0]
    y = K.w8a8_gemm(x, xs, w, ws)
    R.check_linear(y, x, xs, w, ws)
    assert bool(torch.isnan(y[m // 2]).all())


@pytest.mark.parametrize("m,n", [(128, 256), (129, 256), (300, 257), (40, 200), (3, 64)])
def test_gate_values_of_any_size(cuda, m, n):
    """Gates from -200 to 200: the exponential overflows on one side and vanishes on the other."""
    k = 64
    g, x, xs, w, ws = _operands(m, 2 * n, k, 77)
    xs.fill_(1.0)
    ws[:n] = 200.0 / (64 * 127 * 127)
    ws[n:] = 1e-4
    R.check_gated(K.w8a8_gemm(x, xs, w, ws, swiglu=True), x, xs, w, ws)


@pytest.mark.parametrize("n,k,form", [(320, 1536, "both"), (200, 4480, "bias"), (131, 257, "residual"), (192, 640, "gated"),
                                      (1500, 768, "none")])
def test_a_token_does_not_depend_on_its_call(cuda, n, k, form):
    """Bit for bit: the rows of a call of 700 tokens, of calls of the first few, and each alone."""
    m, gated = 700, form == "gated"
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g, x, xs, w, ws = _operands(m, 2 * n if gated else n, k, 5)
    bias = torch.randn(n, generator=g, device="cuda").half() if form in ("bias", "both") else None
    res = torch.randn(m, n, generator=g, device="cuda").half() if form in ("residual", "both") else None
    y = K.w8a8_gemm(x, xs, w, ws, bias=bias, residual=res, swiglu=gated, error=err)
    for a, b in ((0, 1), (3, 11), (5, 20), (0, 32), (7, 71), (100, 200), (0, 257), (699, 700)):
        part = K.w8a8_gemm(x[a:b], xs[a:b], w, ws, bias=bias, residual=None if res is None else res[a:b], swiglu=gated,
                           error=err)
        assert torch.equal(part, y[a:b]), (a, b)
    assert int(err) == 0


@pytest.mark.parametrize("n,k,form", [(200, 256, "gated"), (131, 77, "gated"), (4800, 96, "gated"), (200, 256, "none"),
                                      (131, 77, "bias"), (9504, 96, "none"), (200, 256, "residual")])
def test_the_sign_of_a_zero_does_not_depend_on_the_call(cuda, n, k, form):
    """Gate sums of zero and far below zero against up values of both signs, zero sums and negative ones that vanish in
    fp16: the bits of the rows of a call of 700 tokens, of few and of middling calls, and the formula's sign."""
    m, gated = 700, form == "gated"
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g, x, xs, w, ws = _operands(m, 2 * n if gated else n, k, 6)
    xs.fill_(1.0)
    w[:n:3] = 0
    if gated:
        ws[:n] = 1000.0 / (k ** 0.5 * 73 * 73)  # (gates of some 1000: half of them vanish)
        ws[n:] = 2.0 ** -10
        if n > 16:
            w[n:n + 16:2] = 0  # (up values of zero, both kinds of gates before them)
    else:
        ws.fill_(2.0 ** -46)
    zero = torch.zeros(n, dtype=torch.float16, device="cuda")
    bias = zero if form == "bias" else None
    res = torch.where(torch.arange(n, device="cuda") % 2 == 0, zero, -zero).repeat(m, 1) if form == "residual" else None
    y = K.w8a8_gemm(x, xs, w, ws, bias=bias, residual=res, swiglu=gated, error=err)
    v = R.linear(x, xs, w, ws)
    if gated:
        v = v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:]
    elif bias is not None:
        v = v + bias.double()
    if res is not None:
        v = v + res.double()
    assert int((y == 0).sum()) > m * n // 4 and int(torch.signbit(y[y == 0]).sum()) > m * n // 64
    # (a sum of zero times a scale is +0 here as there; an integer has no zero of its own sign)
    assert torch.equal(torch.signbit(y), torch.signbit(v))
    for a, b in ((0, 1), (3, 11), (5, 17), (5, 20), (0, 32), (7, 71), (100, 200), (0, 257)):
        part = K.w8a8_gemm(x[a:b], xs[a:b], w, ws, bias=bias, residual=None if res is None else res[a:b], swiglu=gated,
                           error=err)
        assert torch.equal(part.view(torch.int16), y[a:b].view(torch.int16)), (a, b)
    assert int(err) == 0


# -- as they are used ----------------------------------------------------------------
def _block(x, part, gamma, wq, err, out=None):
    """Residual and norm, the gated projections, the quantiser, the down projection onto the residual stream."""
    c, s, total = K.rms_norm_q8(part, gamma, EPS, residual=x, sum_out=x)
    act = K.w8a8_gemm(c, s, wq[0], wq[1], swiglu=True, error=err)
    c, s = K.quantise_rows_q8(act)
    return K.w8a8_gemm(c, s, wq[2], wq[3], residual=x, out=out if out is not None else x, error=err)


@pytest.mark.parametrize("m", [1, 3, 64, 333])
def test_a_feed_forward_block(cuda, m):
    """The operators together: each next one gets what the last wrote, eager, on another stream and replayed."""
    h, i = 1536, 2240
    g = _gen(m)
    gamma = (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).half()
    gu = (torch.randn(2 * i, h, generator=g, device="cuda") * h ** -0.5).half()
    down = (torch.randn(h, i, generator=g, device="cuda") * i ** -0.5).half()
    wq = [*K.quantise_rows_q8(gu), *K.quantise_rows_q8(down)]
    x0, part = _rows(m, h, 1, spread=2.0), _rows(m, h, 2, spread=2.0)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = x0.clone()
    y = _block(x, part, gamma, wq, err).clone()
    # the same from the formulas, each stage from the kernels' values before it
    total = (x0.float() + part.float()).half()
    c, s = K.rms_norm_q8(total, gamma, EPS)
    act = K.w8a8_gemm(c, s, wq[0], wq[1], swiglu=True, error=err)
    R.check_rows(R.norm(total, gamma, EPS), c, s, None, h, additions=h / 32 + 13)
    R.check_gated(act, c, s, wq[0], wq[1])
    ca, sa = K.quantise_rows_q8(act)
    R.check_linear(y, ca, sa, wq[2], wq[3], None, total)
    # 8 bits against the unquantised block: rows and weights at 1/127 of their largest element, some 3 to 4 rms
    n = R.norm(total, gamma, EPS)
    gate, up = n @ gu.double().t(), None
    gate, up = gate[:, :i], gate[:, i:]
    full = (gate * torch.sigmoid(gate) * up) @ down.double().t()
    live = total.abs().amax(dim=1) > 0
    off = ((y.double() - total.double()) - full)[live].norm() / full[live].norm()
    assert float(off) < 0.08
    # another stream, and a captured graph replayed on new inputs
    side = torch.cuda.Stream()
    x = x0.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = _block(x, part, gamma, wq, err)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, y)
    xg, pg, out = x0.clone(), part.clone(), torch.empty_like(x0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _block(xg, pg, gamma, wq, err, out=out)
    for k in range(3):
        xn, pn = _rows(m, h, 10 + k), _rows(m, h, 20 + k)
        xg.copy_(xn)
        pg.copy_(pn)
        graph.replay()
        assert torch.equal(out, _block(xn, pn, gamma, wq, err)), k
    assert int(err) == 0


def test_products_right_behind_what_writes_their_operands(cuda):
    """Weights and rows that the kernel before has only just written, over and over (launches overlap)."""
    g = _gen(4)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for m in (1, 40, 130, 600):
        ws_ = [(torch.randn(640, 512, generator=g, device="cuda") * (1 + j)).half() for j in range(4)]
        xs_ = [torch.randn(m, 512, generator=g, device="cuda").half() for _ in range(4)]
        wc, wsc = K.quantise_rows_q8(ws_[0])
        xc, xsc = K.quantise_rows_q8(xs_[0])
        outs = [torch.empty(m, 640, dtype=torch.float16, device="cuda") for _ in range(40)]
        for j in range(40):
            K.quantise_rows_q8(xs_[j % 4], xc, xsc)
            K.quantise_rows_q8(ws_[(j // 2) % 4], wc, wsc)
            K.w8a8_gemm(xc, xsc, wc, wsc, out=outs[j], error=err)
        for j in range(40):
            a, b = K.quantise_rows_q8(xs_[j % 4]), K.quantise_rows_q8(ws_[(j // 2) % 4])
            R.check_linear(outs[j], a[0], a[1], b[0], b[1])
    assert int(err) == 0


@pytest.mark.parametrize("m,n,k,gated", [(48, 9504, 512, False), (64, 4800, 512, True), (12, 640, 512, False),
                                         (24, 640, 512, True), (300, 512, 4096, False), (600, 384, 1600, False)])
def test_every_product_right_behind_what_writes_its_operands(cuda, m, n, k, gated):
    """The same for wide outputs, few tokens in several tiles, and pairs that share K out: each starts while the kernel
    that writes its weights or rows still runs, and touches the weights before it may read them."""
    g, rows = _gen(m + n), 2 * n if gated else n
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    wide = [(torch.randn(rows, k, generator=g, device="cuda") * (1 + j) / k ** 0.5).half() for j in range(3)]
    toks = [torch.randn(m, k, generator=g, device="cuda").half() for _ in range(4)]
    wc, wsc = K.quantise_rows_q8(wide[0])
    xc, xsc = K.quantise_rows_q8(toks[0])
    outs = [torch.full((m, n), 7.0, dtype=torch.float16, device="cuda") for _ in range(24)]
    torch.cuda.synchronize()
    for j in range(24):
        if j % 2:  # the weights last, or the rows
            K.quantise_rows_q8(toks[j % 4], xc, xsc)
            K.quantise_rows_q8(wide[j % 3], wc, wsc)
        else:
            K.quantise_rows_q8(wide[j % 3], wc, wsc)
            K.quantise_rows_q8(toks[j % 4], xc, xsc)
        K.w8a8_gemm(xc, xsc, wc, wsc, swiglu=gated, out=outs[j], error=err)
    for j in range(24):
        a, b = K.quantise_rows_q8(toks[j % 4]), K.quantise_rows_q8(wide[j % 3])
        (R.check_gated if gated else R.check_linear)(outs[j], a[0], a[1], b[0], b[1])
    assert int(err) == 0


@pytest.mark.parametrize("m,apart", [(3, 1 << 30), (40, 1 << 26), (140, 1 << 25)])
@pytest.mark.parametrize("k,n", [(256, 192), (131, 77)])
def test_rows_far_apart(cuda, m, apart, k, n):
    """Rows whose offsets pass 32 bits: x, codes, residual, y and weights; the results of rows side by side."""
    def far(rows, cols, dtype):
        return torch.empty((rows - 1) * apart + cols, dtype=dtype, device="cuda").as_strided((rows, cols), (apart, 1))

    h = torch.float16
    x, w, gamma = _rows(m, k, 1), _rows(n, k, 2), _rows(1, k, 3)[0]
    want, wq = K.rms_norm_q8(x, gamma, residual=x), K.quantise_rows_q8(w)
    xf, codes, total = far(m, k, h).copy_(x), far(m, k, torch.int8), far(m, k, h)
    _, scales, _ = K.rms_norm_q8(xf, gamma, residual=xf, sum_out=total, codes=codes)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(total, want[2])
    del xf, total
    res = _rows(m, n, 4)
    gu = wq[0][:n // 2 * 2], wq[1][:n // 2 * 2]
    plain, gated = K.w8a8_gemm(*want[:2], *wq, residual=res), K.w8a8_gemm(*want[:2], *gu, swiglu=True)
    y = far(m, n, h).copy_(res)
    assert torch.equal(K.w8a8_gemm(codes, scales, *wq, residual=y, out=y), plain)
    few = min(n // 2 * 2, 4 if apart > 1 << 29 else 128)
    wf = far(few, k, torch.int8).copy_(wq[0][:few])
    near = K.w8a8_gemm(*want[:2], wq[0][:few], wq[1][:few])
    assert torch.equal(K.w8a8_gemm(codes, scales, wf, wq[1][:few], out=y[:, :few]), near)
    assert torch.equal(K.w8a8_gemm(codes, scales, *gu, swiglu=True, out=y[:, :n // 2]), gated)


def test_strides_past_32_bits_are_refused(cuda):
    """A distance of rows that does not fit the entry points' 32 bits must not arrive there as another one."""
    apart, err = (1 << 32) + 64, torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.zeros(apart + 64, dtype=torch.int8, device="cuda").as_strided((2, 64), (apart, 1))
    s, w = torch.ones(2, device="cuda"), torch.zeros(2, 64, dtype=torch.int8, device="cuda")
    y = torch.zeros(2, 2, dtype=torch.float16, device="cuda")
    for a, b in ((x, w), (w, x)):
        with pytest.raises(ValueError, match="32 bits"):
            K.w8a8_gemm(a, s, b, s, out=y, error=err)
    with pytest.raises(ValueError, match="codes.*32 bits"):
        K.quantise_rows_q8(torch.zeros(2, 64, dtype=torch.float16, device="cuda"), codes=x, scales=s)


def test_argument_mistakes(cuda):
    g, x, xs, w, ws = _operands(4, 48, 64, 1)
    h = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    gamma = torch.ones(64, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError, match="codes"):
        K.w8a8_gemm(h, xs, w, ws)
    with pytest.raises(TypeError, match="w_scales"):
        K.w8a8_gemm(x, xs, w, ws.double())
    with pytest.raises(ValueError, match="scales"):
        K.w8a8_gemm(x, xs[:3], w, ws)
    with pytest.raises(ValueError, match="w_codes"):
        K.w8a8_gemm(x, xs, R.rand_codes(48, 63, g, "cuda"), ws)
    with pytest.raises(ValueError, match="bias"):
        K.w8a8_gemm(x, xs, w, ws, bias=gamma)
    with pytest.raises(ValueError, match="out"):
        K.w8a8_gemm(x, xs, w, ws, out=h)
    with pytest.raises(ValueError, match="no bias or residual"):
        K.w8a8_gemm(x, xs, w, ws, bias=gamma[:24], swiglu=True)
    with pytest.raises(ValueError, match="as many gate rows"):
        K.w8a8_gemm(x, xs, w[:47], ws[:47], swiglu=True)
    with pytest.raises(ValueError, match="multiples of 16"):
        K.w8a8_gemm(x[:, 1:], xs, w[:, 1:], ws)
    with pytest.raises(ValueError, match="multiples of 16"):
        K.w8a8_gemm(x[:, :40].contiguous(), xs, w[:, :40], ws)
    with pytest.raises(ValueError, match="side by side"):
        K.w8a8_gemm(x, xs, w.t().contiguous().t(), ws)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.w8a8_gemm(x, xs, w, ws.cpu())
    big = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="lmps_w8a8_gemm"):
        K.w8a8_gemm(big, xs[:1], big, ws[:1])
    with pytest.raises(TypeError, match="x"):
        K.quantise_rows_q8(h.float())
    with pytest.raises(ValueError, match="overlap"):
        K.quantise_rows_q8(h[:1].expand(4, 64))
    with pytest.raises(ValueError, match="codes"):
        K.quantise_rows_q8(h, codes=torch.zeros(4, 63, dtype=torch.int8, device="cuda"))
    with pytest.raises(ValueError, match="gamma"):
        K.rms_norm_q8(h, gamma[:63])
    with pytest.raises(ValueError, match="sum_out"):
        K.rms_norm_q8(h, gamma, sum_out=h)
    with pytest.raises(ValueError, match="x"):
        K.rms_norm_q8(h[None], gamma)
    with pytest.raises(RuntimeError, match="lmps_rms_norm_q8"):
        K.rms_norm_q8(h, gamma, -1.0)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="captured"):
        with torch.cuda.graph(graph):
            K.w8a8_gemm(x, xs, w, ws, out=torch.empty(4, 48, dtype=torch.float16, device="cuda"))
