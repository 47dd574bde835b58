"""8-bit rows and their product (cl-inference_b200/int8.py) against 64-bit forms; needs a B200.

Tolerances, with u = 2^-24 (half a step of f32, relative):

codes   before its rounding to a whole number a code is v * inv: v carries at most two
        roundings (residual sum, norm weight), peak / 127 and 1 / step one each, and the peak
        the two of its own v, the product one: 8 u relative of at most 127, so it is within
        127 * 8 u < 6.1e-5 of the exact quotient, and the code within 0.5 + 6.1e-5.
        silu(g) * u comes from an exponential of 2^-22 (4 u), its argument's correction, 1 + e, a
        reciprocal of 2^-23 (2 u) and two products (4 u): 10 u for v and 10 u for the peak, beside
        the two of the step: 127 * 22 u < 1.7e-4.
scales  peak / 127 and its product with s one rounding each beside the peak's own; the sum of k
        squares in some order of f32 additions in which no value passes more than k / 32 + 24
        of them, halved by the square root, which with the mean, the addition of eps, the square
        root and the quotient adds 4: (k / 64 + 20) u is above all of them.
product acc -> f32, times two scales: 3 u of the product; the residual one more, of the sum;
        a 16-bit output one half step of its own (2^-8, 2^-11, or its smallest step).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["float32", "bfloat16", "float16"]
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}


def rand(torch, *shape, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=gen) * scale


def codes_of(torch, rows, k, seed, pitch=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pitch = (k + 15) // 16 * 16 if pitch is None else pitch
    c = torch.randint(-128, 128, (rows, pitch), device="cuda", generator=gen, dtype=torch.int32).to(torch.int8)
    return c[:, :k], (torch.rand(rows, device="cuda", generator=gen) + 0.5) / 512


def check_rows(torch, q, v, s=None, slack=6.1e-5):
    """q against the 64-bit rows V (and norm factors S)."""
    k = v.shape[1]
    peak = v.abs().amax(1)
    assert (peak > 0).all() and q.codes.dtype == torch.int8
    ideal = v * (127 / peak)[:, None]
    assert (q.codes.double() - ideal).abs().max().item() <= 0.5 + slack
    assert q.codes.abs().amax().item() <= 127
    want = peak / 127 * (1 if s is None else s)
    assert ((q.scales.double() - want).abs() / want).max().item() <= (k / 64 + 20) * U


SHAPES = [(1, 1), (3, 7), (2, 16), (1, 33), (5, 255), (9, 512), (4, 1000), (3, 2048), (2, 4096), (1, 5001), (2, 8192),
          (2, 14336), (1, 28672), (2, 40000), (300, 64)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("xtype", TYPES)
def test_quantize_rows(cuda, clq, m, k, xtype):
    torch = cuda
    x = rand(torch, m, k, seed=m + k).to(getattr(torch, xtype))
    x[:, 0] += 0.25  # no row of zeros
    check_rows(torch, clq.quantize_rows(x), x.double())


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("xtype,rtype", [(a, b) for a in TYPES for b in sorted({a, "float32"})] + [("float32", None),
                                                                                                  ("bfloat16", None)])
def test_norm_quantize(cuda, clq, m, k, xtype, rtype):
    torch = cuda
    x = rand(torch, m, k, seed=1).to(getattr(torch, xtype))
    g = rand(torch, k, seed=2, scale=0.3) + 1
    h = x.double()
    if rtype:
        r = rand(torch, m, k, seed=3, scale=3.0).to(getattr(torch, rtype))
        h = h + r.double()
    got = clq.norm_quantize(x, g, 1e-5, **({"residual": r} if rtype else {}))
    if rtype:
        got, total = got
        assert total.dtype == r.dtype
        far = (total.double() - h).abs()
        assert (far <= HALF_STEP[rtype] * 1.001 * h.abs() + U * h.abs() + TINY[rtype]).all()
    s = 1 / torch.sqrt((h * h).mean(1) + 1e-5)
    check_rows(torch, got, h * g.double(), s)


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("xtype", TYPES)
def test_swiglu_quantize(cuda, clq, m, k, xtype):
    torch = cuda
    both = rand(torch, m, 2 * k, seed=5, scale=2.0).to(getattr(torch, xtype))
    both[:, 0] = both[:, k] = 1.5  # no row of zeros
    gate, up = both[:, :k], both[:, k:]
    g = gate.double()
    check_rows(torch, clq.swiglu_quantize(gate, up), g * torch.sigmoid(g) * up.double(), slack=1.7e-4)


def test_swiglu_of_far_gates(cuda, clq):
    """Gates past the exponential's range: silu(-200) is 0 and silu(200) is 200."""
    torch = cuda
    gate = torch.tensor([[-200.0, 200.0, 0.0, -88.0]], device="cuda")
    up = torch.tensor([[3.0, 1.0, 5.0, 1.0]], device="cuda")
    q = clq.swiglu_quantize(gate, up)
    assert q.codes.tolist() == [[0, 127, 0, 0]]
    assert abs(q.scales.item() * 127 / 200 - 1) < 8 * U


@pytest.mark.parametrize("xtype", TYPES)
@pytest.mark.parametrize("offset,pitch", [(0, 96), (1, 97), (3, 101), (8, 96), (4, 128)])
def test_strided_and_unaligned_rows(cuda, clq, xtype, offset, pitch):
    """Rows inside a wider buffer at any element offset; what lies around the outputs stays."""
    torch = cuda
    m, k = 5, 80
    dtype = getattr(torch, xtype)
    buf = rand(torch, 3, m * pitch + offset + 16, seed=7).to(dtype)
    x, r, out = (b[offset:offset + m * pitch].view(m, pitch)[:, :k] for b in buf)
    g = rand(torch, k + 1, seed=8)[1:]  # off the 16-byte grid
    before, h = buf.clone(), x.double() + r.double()
    q, total = clq.norm_quantize(x, g, 1e-6, residual=r, residual_out=out)
    assert total is out
    check_rows(torch, q, h * g.double(), 1 / torch.sqrt((h * h).mean(1) + 1e-6))
    assert torch.equal(out, (x.float() + r.float()).to(dtype))
    out.copy_(before[2, offset:offset + m * pitch].view(m, pitch)[:, :k])
    assert torch.equal(buf, before)
    check_rows(torch, clq.swiglu_quantize(x, r), x.double() * torch.sigmoid(x.double()) * r.double(), slack=1.7e-4)
    # a transposed view has no unit last stride and is copied
    assert torch.equal(clq.quantize_rows(x.t()).codes, clq.quantize_rows(x.t().contiguous()).codes)
    # one row read for every token
    assert torch.equal(clq.quantize_rows(x[:1].expand(4, k)).codes, clq.quantize_rows(x[:1]).codes.expand(4, k))


@pytest.mark.parametrize("m,k", [(700, 513), (3, 1500), (900, 1501), (5, 5001), (650, 5001), (2, 20001), (160, 20001),
                                 (2, 33001)])
@pytest.mark.parametrize("xtype,rtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_rows_off_the_grid_at_length(cuda, clq, m, k, xtype, rtype):
    """Rows whose starts take every distance from the 16-byte grid in turn (the row stride is odd),
    one after another in their buffers, with the outputs' surroundings left as they were."""
    torch = cuda
    x = rand(torch, m * k + 8, seed=1).to(getattr(torch, xtype))[3:3 + m * k].view(m, k)
    r = rand(torch, m * (k + 2) + 8, seed=2).to(getattr(torch, rtype))[5:5 + m * (k + 2)].view(m, k + 2)[:, :k]
    buf = torch.full((m * (k + 4) + 8,), 7.0, dtype=r.dtype, device="cuda")
    out = buf[1:1 + m * (k + 4)].view(m, k + 4)[:, :k]
    g = rand(torch, k, seed=3, scale=0.3) + 1
    h = x.double() + r.double()
    q, total = clq.norm_quantize(x, g, 1e-5, residual=r, residual_out=out)
    check_rows(torch, q, h * g.double(), 1 / torch.sqrt((h * h).mean(1) + 1e-5))
    assert torch.equal(total, (x.float() + r.float()).to(r.dtype))
    out.fill_(7.0)
    assert (buf == 7).all()
    check_rows(torch, clq.quantize_rows(x), x.double())
    gate = x.flip(0).contiguous()
    check_rows(torch, clq.swiglu_quantize(gate, x), gate.double() * torch.sigmoid(gate.double()) * x.double(), slack=1.7e-4)
    assert status(clq) == 0


@pytest.mark.parametrize("m,k", [(3, 1023), (3, 1025), (148, 4095), (3, 4099), (3, 8191), (3, 8193), (4, 16383), (4, 16385),
                                 (149, 4095), (300, 777), (300, 2047), (300, 2049), (300, 4097), (300, 6143), (300, 6145),
                                 (300, 8191), (300, 8193), (200, 14337)])
@pytest.mark.parametrize("xtype,rtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_rows_off_the_grid_at_the_edges_of_each_split(cuda, clq, m, k, xtype, rtype):
    test_rows_off_the_grid_at_length(cuda, clq, m, k, xtype, rtype)
    # a norm without a residual
    torch = cuda
    x = rand(torch, m, k, seed=4).to(getattr(torch, xtype))
    g = rand(torch, k, seed=5, scale=0.3) + 1
    h = x.double()
    check_rows(torch, clq.norm_quantize(x, g, 1e-5), h * g.double(), 1 / torch.sqrt((h * h).mean(1) + 1e-5))


@pytest.mark.parametrize("m", [600, 1000])
@pytest.mark.parametrize("k", [1024, 4096, 14336])
def test_many_rows(cuda, clq, m, k):
    """Enough rows for the kernel that streams them, each against the same row among few."""
    torch = cuda
    for xtype, rtype in (("bfloat16", "float32"), ("float16", "float16"), ("float32", "float32")):
        x = rand(torch, m, k, seed=1).to(getattr(torch, xtype))
        r = rand(torch, m, k, seed=2).to(getattr(torch, rtype))
        g = rand(torch, k, seed=3)
        x[5, 7], x[m - 1, k - 1] = float("nan"), float("inf")
        for call in (lambda a, b: clq.norm_quantize(a, g, residual=b), lambda a, b: clq.norm_quantize(a, None, residual=b),
                     lambda a, b: (clq.quantize_rows(a), a), lambda a, b: (clq.swiglu_quantize(a, b.to(a.dtype)), a)):
            q, t = call(x, r)
            for at in (0, 100, m - 100):
                few, ft = call(x[at:at + 100], r[at:at + 100])
                assert torch.equal(q.codes[at:at + 100], few.codes)
                far = (q.scales[at:at + 100] - few.scales).abs() / few.scales
                assert (far.nan_to_num(0) <= (k / 64 + 20) * U).all()
                assert torch.equal(torch.isnan(q.scales[at:at + 100]), torch.isnan(few.scales))
                assert torch.equal(t[at:at + 100].nan_to_num(1), ft.nan_to_num(1))
            assert torch.isnan(q.scales[[5, m - 1]]).all() and int(torch.isnan(q.scales).sum()) == 2


@pytest.mark.parametrize("k", [40, 4096, 40000])
@pytest.mark.parametrize("rtype", TYPES)
def test_residual_in_place(cuda, clq, k, rtype):
    torch = cuda
    x = rand(torch, 4, k, seed=11).to(getattr(torch, rtype))
    r = rand(torch, 4, k, seed=12).to(getattr(torch, rtype))
    g = rand(torch, k, seed=13)
    q, total = clq.norm_quantize(x, g, residual=r)
    x2, r2 = x.clone(), r.clone()
    q2, t2 = clq.norm_quantize(x2, g, residual=r2, residual_out=r2)
    assert t2 is r2 and torch.equal(total, r2)
    assert torch.equal(q.codes, q2.codes) and torch.equal(q.scales, q2.scales)
    q3, t3 = clq.norm_quantize(x2, g, residual=r, residual_out=x2)  # onto the input rows
    assert torch.equal(total, x2) and torch.equal(q.codes, q3.codes)
    q4, t4 = clq.norm_quantize(x, None, residual=r)  # the sum alone, without a norm
    check_rows(torch, q4, x.double() + r.double())
    assert torch.equal(total, t4)
    with pytest.raises(ValueError):
        clq.norm_quantize(x[:3], g, residual=r[:3], residual_out=r[1:])


@pytest.mark.parametrize("k", [24, 1000, 4096, 36000])
def test_rows_with_nothing_or_nothing_finite(cuda, clq, k):
    torch = cuda
    inf, nan = float("inf"), float("nan")
    x = rand(torch, 8, k, seed=21)
    x[0] = 0
    x[1, k - 1] = nan
    x[2, 0] = inf
    x[3, k // 2] = -inf
    x[4] = 0
    x[4, k - 1] = 1e-44         # below FLT_MIN: the step stays FLT_MIN
    x[5] *= 1e30                # the squares leave f32
    x[6] = 0
    x[6, 1] = -3.4e38
    q = clq.quantize_rows(x)
    assert not q.codes[0].any() and q.scales[0].item() == 1.0
    for row in (1, 2, 3):
        assert not q.codes[row].any() and torch.isnan(q.scales[row])
    assert not q.codes[4].any() and q.scales[4].item() == 2.0 ** -126
    check_rows(torch, clq.Int8Rows(q.codes[5:8], q.scales[5:8]), x[5:8].double())
    assert q.codes[6, 1].item() == -127
    n = clq.norm_quantize(x, torch.ones(k, device="cuda"), 1e-5)
    assert not n.codes[0].any() and n.scales[0].item() == 1.0
    for row in (1, 2, 3, 5, 6):
        assert not n.codes[row].any() and torch.isnan(n.scales[row])
    assert torch.isfinite(n.scales[7])
    # a weight of infinity, at a place where the row is zero as well
    g = torch.ones(k, device="cuda")
    g[0] = inf
    assert torch.isnan(clq.norm_quantize(x, g).scales[[0, 7]]).all()
    y = clq.linear_int8(n, clq.quantize_rows(rand(torch, 20, k, seed=22)))
    assert torch.isnan(y[[1, 2, 3, 5, 6]]).all() and torch.isfinite(y[[0, 4, 7]]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 17), (5, 4096), (2, 5001), (70000, 3), (9, 700)])
def test_dequantize(cuda, clq, dtype, m, k):
    torch = cuda
    c, s = codes_of(torch, m, k, seed=31)
    q = clq.Int8Rows(c, s)
    want = c.float() * s[:, None]
    assert torch.equal(q.dequantize(getattr(torch, dtype)), want.to(getattr(torch, dtype)))
    wide = torch.full((m, k + 5), 7.0, dtype=getattr(torch, dtype), device="cuda")
    assert q.dequantize(out=wide[:, 3:3 + k]).data_ptr() == wide[:, 3:].data_ptr()
    assert torch.equal(wide[:, 3:3 + k], want.to(wide.dtype))
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + k:] == 7).all()


def test_no_rows_and_no_columns(cuda, clq):
    torch = cuda
    assert clq.quantize_rows(torch.empty(0, 9, device="cuda")).shape == (0, 9)
    q = clq.quantize_rows(torch.empty(4, 0, device="cuda"))
    assert q.shape == (4, 0) and (q.scales == 1).all()
    w = clq.quantize_rows(torch.empty(3, 0, device="cuda"))
    assert torch.equal(clq.linear_int8(q, w), torch.zeros(4, 3, device="cuda"))
    res = rand(torch, 4, 3, seed=1)
    assert torch.equal(clq.linear_int8(q, w, residual=res), res)
    c, s = codes_of(torch, 5, 32, seed=2)
    some = clq.Int8Rows(c, s)
    assert clq.linear_int8(some[:0], some).shape == (0, 5) and clq.linear_int8(some, some[:0]).shape == (5, 0)


# ---- the product -----------------------------------------------------------

def check_product(torch, got, x, w, residual=None):
    acc = x.codes.double() @ w.codes.double().t()
    p = acc * w.scales.double() * x.scales.double()[:, None]
    want, room = p, 3.01 * U * p.abs()
    if residual is not None:
        want = p + residual.double()
        room = room + 1.01 * U * want.abs()
    name = str(got.dtype).replace("torch.", "")
    if name != "float32":
        room = room + HALF_STEP[name] * 1.001 * want.abs() + TINY[name]
    fine = want.abs() < 65000 if name == "float16" else torch.ones_like(want, dtype=torch.bool)
    assert ((got.double() - want).abs() <= room + 1e-300)[fine].all()


M = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 192, 255, 256, 257, 385, 512]
NK = [(1, 1), (8, 16), (5, 33), (16, 64), (127, 100), (128, 128), (130, 131), (257, 256), (300, 1000), (512, 2048),
      (1000, 4096)]


@pytest.mark.parametrize("n,k", NK)
def test_linear_over_token_counts(cuda, clq, n, k):
    torch = cuda
    w = clq.Int8Rows(*codes_of(torch, n, k, seed=n + k))
    for m in M:
        x = clq.Int8Rows(*codes_of(torch, m, k, seed=m))
        check_product(torch, clq.linear_int8(x, w), x, w)


@pytest.mark.parametrize("m", [1, 5, 16, 24, 40, 64, 96, 160, 300, 700, 2100])
@pytest.mark.parametrize("n,k", [(4096, 512), (5003, 2051), (1024, 8192), (64, 14336), (2304, 96)])
def test_linear_over_weights(cuda, clq, m, n, k):
    torch = cuda
    w = clq.Int8Rows(*codes_of(torch, n, k, seed=n + k))
    x = clq.Int8Rows(*codes_of(torch, m, k, seed=m))
    res = rand(torch, m, n, seed=3)
    for dtype in TYPES:
        check_product(torch, clq.linear_int8(x, w, dtype=getattr(torch, dtype)), x, w)
        check_product(torch, clq.linear_int8(x, w, dtype=getattr(torch, dtype), residual=res), x, w, res)


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 4096), (1, 28672, 4096), (16, 4096, 14336), (1500, 3000, 700),
                                   (4096, 1024, 512), (8, 128256, 256), (250, 19200, 4096), (300, 4864, 2048),
                                   (1111, 9472, 1024), (77, 512, 40000)])
def test_linear_at_size(cuda, clq, m, n, k):
    torch = cuda
    w = clq.Int8Rows(*codes_of(torch, n, k, seed=n + k))
    x = clq.Int8Rows(*codes_of(torch, m, k, seed=m))
    got = clq.linear_int8(x, w)
    check_product(torch, got, x, w)
    assert torch.equal(got, clq.linear_int8(x, w))
    assert status(clq) == 0


@pytest.mark.parametrize("m", [1, 16, 40, 200])
@pytest.mark.parametrize("k", [131071, 131056])
def test_longest_rows_of_the_largest_codes(cuda, clq, m, k):
    """-128 * -128 * k is the largest sum: it fits 32 bits and is exact."""
    torch = cuda
    x = clq.Int8Rows(torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :k], torch.ones(m, device="cuda"))
    w = clq.Int8Rows(torch.full((20, 131072), -128, dtype=torch.int8, device="cuda")[:, :k],
                     torch.ones(20, device="cuda"))
    assert (clq.linear_int8(x, w) == float(np.float32(16384 * k))).all()
    with pytest.raises(clq.ClqError):
        long = torch.zeros((1, 131072), dtype=torch.int8, device="cuda")
        clq.linear_int8(clq.Int8Rows(long, x.scales[:1]), clq.Int8Rows(long, x.scales[:1]))


@pytest.mark.parametrize("m", [1, 11, 33, 130, 260])
def test_linear_of_small_sums_is_exact(cuda, clq, m):
    torch = cuda
    (xc, _), (wc, _) = codes_of(torch, m, 300, seed=m), codes_of(torch, 77, 300, seed=1)
    x, w = clq.Int8Rows(xc, torch.ones(m, device="cuda")), clq.Int8Rows(wc, torch.ones(77, device="cuda"))
    assert torch.equal(clq.linear_int8(x, w).double(), xc.double() @ wc.double().t())


@pytest.mark.parametrize("m", [1, 4, 16, 33, 100, 260])
@pytest.mark.parametrize("what", ["x off", "w off", "x pitch", "w pitch", "both"])
def test_linear_of_unaligned_rows(cuda, clq, m, what):
    torch = cuda
    k, n = 200, 150

    def rows(count, off, pitch, seed):
        c, s = codes_of(torch, 1, count * pitch + off, seed)
        return clq.Int8Rows(c[0, off:off + count * pitch].view(count, pitch)[:, :k], s.expand(count).contiguous())
    x = rows(m, 3 if what in ("x off", "both") else 0, 203 if what in ("x pitch", "both") else 208, 1)
    w = rows(n, 1 if what in ("w off", "both") else 0, 201 if what in ("w pitch", "both") else 256, 2)
    check_product(torch, clq.linear_int8(x, w), x, w)


@pytest.mark.parametrize("m", [1, 7, 8, 9, 16, 17, 64, 65, 200])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 15), (9, 16), (64, 17), (65, 31), (33, 47), (20, 63), (150, 79), (16, 80), (31, 95),
                                 (130, 127), (70, 143), (64, 145), (2500, 500), (1000, 1100), (300, 2051)])
@pytest.mark.parametrize("xoff,woff", [(1, 2), (15, 0), (4, 11)])
def test_linear_of_rows_that_end_beside_others(cuda, clq, m, n, k, xoff, woff):
    """Every distance from the 16-byte grid (odd strides), the neighbours' codes not taken in, the
    first row at its buffer's start and the last at its end."""
    torch = cuda

    def rows(count, off, seed):
        c, s = codes_of(torch, 1, count * k + off, seed, pitch=count * k + off)
        return clq.Int8Rows(c[0, off:].view(count, k), s.expand(count).contiguous())
    x, w = rows(m, xoff, 1), rows(n, woff, 2)
    res = rand(torch, m, n, seed=3)
    check_product(torch, clq.linear_int8(x, w, dtype=torch.bfloat16, residual=res), x, w, res)
    exact = x.codes.double() @ w.codes.double().t()
    ones = [clq.Int8Rows(q.codes, torch.ones_like(q.scales)) for q in (x, w)]
    assert torch.equal(clq.linear_int8(*ones).double(), exact.float().double())


@pytest.mark.parametrize("m", [1, 6, 16, 40, 130, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_into_a_wider_buffer_and_onto_its_residual(cuda, clq, m, dtype):
    """Columns 3.. of a wider output; what lies around them stays.  The rows past
    K of both operands hold other codes, which no sum may touch."""
    torch = cuda
    n, k = 131, 170
    w = clq.Int8Rows(*codes_of(torch, n, k, 1, pitch=192))
    x = clq.Int8Rows(*codes_of(torch, m, k, 2, pitch=256))
    wide = torch.full((m + 2, n + 9), 5.0, dtype=getattr(torch, dtype), device="cuda")
    out = wide[1:-1, 3:3 + n]
    assert clq.linear_int8(x, w, out=out) is out
    check_product(torch, out, x, w)
    assert (wide[0] == 5).all() and (wide[-1] == 5).all() and (wide[:, :3] == 5).all() and (wide[:, 3 + n:] == 5).all()
    if dtype == "float32":
        stream = rand(torch, m, n + 4, seed=3)[:, :n]
        want = clq.linear_int8(x, w, residual=stream)
        clq.linear_int8(x, w, out=stream, residual=stream)
        assert torch.equal(stream, want)
        with pytest.raises(ValueError):
            big = torch.zeros(m, n + 1, device="cuda")
            clq.linear_int8(x, w, out=big[:, 1:], residual=big[:, :n])


def test_row_ranges_of_a_weight(cuda, clq):
    torch = cuda
    w = clq.Int8Rows(*codes_of(torch, 500, 320, 1))
    for m in (1, 20, 140):
        x = clq.Int8Rows(*codes_of(torch, m, 320, 2))
        whole = clq.linear_int8(x, w)
        assert torch.equal(clq.linear_int8(x, w[37:411]), whole[:, 37:411])
        assert torch.equal(clq.linear_int8(x[m // 2:], w), whole[m // 2:])


def test_refusals(cuda, clq):
    torch = cuda
    x = rand(torch, 4, 64, seed=1)
    q = clq.quantize_rows(x)
    for call in (
        lambda: clq.quantize_rows(x.double()), lambda: clq.quantize_rows(x[0]), lambda: clq.quantize_rows(x.cpu()),
        lambda: clq.norm_quantize(x, torch.ones(63, device="cuda")),
        lambda: clq.norm_quantize(x, torch.ones(64, device="cuda", dtype=torch.bfloat16)),
        lambda: clq.norm_quantize(x, residual=x[:3]), lambda: clq.norm_quantize(x, residual=x.bfloat16()),
        lambda: clq.norm_quantize(x, residual_out=x),
        lambda: clq.norm_quantize(x, residual=x, residual_out=torch.empty(4, 65, device="cuda")),
        lambda: clq.swiglu_quantize(x, x.half()), lambda: clq.swiglu_quantize(x, x[:, :60]),
        lambda: clq.Int8Rows(x, q.scales), lambda: clq.Int8Rows(q.codes, q.scales[:3]),
        lambda: clq.linear_int8(x, q), lambda: clq.linear_int8(q, clq.quantize_rows(x[:, :32])),
        lambda: clq.linear_int8(q, q, dtype=torch.int32), lambda: clq.linear_int8(q, q, residual=rand(torch, 4, 5, seed=1)),
        lambda: clq.linear_int8(q, q, residual=rand(torch, 4, 4, seed=1).half()),
        lambda: clq.linear_int8(q, q, out=torch.empty(4, 8, device="cuda")[:, ::2]),
        lambda: clq.linear_int8(q, q, out=torch.empty(1, 4, device="cuda").expand(4, 4)),
        lambda: q.dequantize(torch.int8),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        q[::2]
    with pytest.raises(clq.ClqError):
        clq.norm_quantize(x, torch.ones(64, device="cuda"), -1.0)


# ---- together, as a layer uses them ----------------------------------------

class Layer:
    """The feed-forward half of a decoder layer in 8-bit activations."""

    def __init__(self, clq, torch, hidden, ffn, seed=0):
        self.clq, self.torch, self.ffn = clq, torch, ffn
        self.norm = rand(torch, hidden, seed=seed, scale=0.2) + 1
        self.gate_up = clq.quantize_rows(rand(torch, 2 * ffn, hidden, seed=seed + 1, scale=hidden ** -0.5))
        self.down = clq.quantize_rows(rand(torch, hidden, ffn, seed=seed + 2, scale=ffn ** -0.5))

    def __call__(self, y, stream):
        clq, f = self.clq, self.ffn
        q, h = clq.norm_quantize(y, self.norm, 1e-5, residual=stream)
        gu = clq.linear_int8(q, self.gate_up, dtype=y.dtype)
        a = clq.swiglu_quantize(gu[:, :f], gu[:, f:])
        return clq.linear_int8(a, self.down, residual=h), (q, h, gu, a)


@pytest.mark.parametrize("m", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_feed_forward(cuda, clq, m, dtype):
    """Each step of a run against the 64-bit form of what the step before it gave."""
    torch = cuda
    hidden, ffn = 512, 1376
    layer = Layer(clq, torch, hidden, ffn)
    y = rand(torch, m, hidden, seed=5).to(getattr(torch, dtype))
    stream = rand(torch, m, hidden, seed=6)
    out, (q, h, gu, a) = layer(y, stream)
    sums = y.double() + stream.double()
    s = 1 / torch.sqrt((sums * sums).mean(1) + 1e-5)
    check_rows(torch, q, sums * layer.norm.double(), s)
    check_product(torch, gu, q, layer.gate_up)
    g = gu[:, :ffn].double()
    check_rows(torch, a, g * torch.sigmoid(g) * gu[:, ffn:].double(), slack=1.7e-4)
    check_product(torch, out, a, layer.down, h)


def test_captured_layers_share_nothing(cuda, clq):
    """Two captured graphs of one layer on their own buffers, replayed at once on two
    streams, and an eager run on a third, all give what the eager run gave."""
    torch = cuda
    layer = Layer(clq, torch, 1024, 2048)
    for m in (1, 24, 200):
        ys = [rand(torch, m, 1024, seed=i) for i in range(3)]
        hs = [rand(torch, m, 1024, seed=10 + i) for i in range(3)]
        want = [layer(y, h)[0].clone() for y, h in zip(ys, hs)]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(layer(ys[i], hs[i])[0])
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in range(3)]
        for _ in range(3):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            with torch.cuda.stream(streams[2]):
                eager = layer(ys[2], hs[2])[0]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs + [eager], want))
        # new inputs in the captured buffers
        ys[0].copy_(ys[2])
        hs[0].copy_(hs[2])
        graphs[0].replay()
        assert torch.equal(outs[0], want[2])
    assert status(clq) == 0


def test_a_stream_by_handle(cuda, clq):
    torch = cuda
    side = torch.cuda.Stream()
    x = rand(torch, 40, 4096, seed=1)
    w = clq.quantize_rows(rand(torch, 256, 4096, seed=2))
    want = clq.linear_int8(clq.quantize_rows(x), w)
    torch.cuda.synchronize()
    default = torch.cuda.default_stream().cuda_stream
    assert torch.equal(clq.linear_int8(clq.quantize_rows(x, stream=default), w, stream=default), want)
    h = side.cuda_stream
    for _ in range(20):
        with torch.cuda.stream(side):
            busy = x @ x.t()  # the side stream is busy, the current one is not
        q = clq.quantize_rows(x, stream=h)
        y = clq.linear_int8(q, w, stream=h)
        v = q.dequantize(torch.float32, stream=h)
        side.synchronize()
        assert torch.equal(y, want) and torch.equal(v, q.codes.float() * q.scales[:, None])
    del busy


def test_a_packed_weight_in_8_bits(cuda, clq, synth):
    """A packed store requantized by row.  Against the unrounded operands each factor is off by
    half of its row's step: x by sx / 2 and w by sw / 2 (and 1e-4 of a step from the codes' own f32)."""
    torch = cuda
    n, k, m = 256, 1024, 5
    store = clq.Store("q8_0", n, k, synth.packed_blocks("q8_0", n, k, seed=1))
    wide = store.dequantize()
    w = clq.quantize_rows(wide)
    x = rand(torch, m, k, seed=2)
    q = clq.quantize_rows(x)
    got = clq.linear_int8(q, w)
    check_product(torch, got, q, w)
    x, wide = x.double(), wide.double()
    dx, dw = 0.5001 * q.scales.double()[:, None], 0.5001 * w.scales.double()
    room = dx * wide.abs().sum(1) + dw * x.abs().sum(1, keepdim=True) + k * dx * dw
    assert ((got.double() - x @ wide.t()).abs() <= room * (1 + 1e-5)).all()
    store.close()


def status(clq):
    import ctypes
    s = ctypes.c_int(-1)
    assert clq._lib.lib.clq_device_status(ctypes.byref(s)) == 0, clq._lib.last_error()
    return s.value
