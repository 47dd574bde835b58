"""8-bit rows (cl-inference_b200/int8.py) at the borders of their rule and of f32; needs a B200.

U = 2^-24 is half a step of f32, relative.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLT_MIN = np.float32(2.0 ** -126)


def border_rows(m, k, seed):
    """Rows of f32 whose values lie on the border of two codes: v * inv, rounded to f32, falls
    on or to one side of a half where the exact product falls on the other (or on it)."""
    rng = np.random.default_rng(seed)
    found = np.zeros((0,), np.float32)
    while len(found) < 64:
        peak = np.float32(rng.uniform(1, 2))
        inv = np.float32(1) / (peak / np.float32(127))
        near = ((np.arange(-126, 126) + 0.5) / np.float64(inv)).astype(np.float32)
        v = np.concatenate([near, np.nextafter(near, np.float32(9)), np.nextafter(near, np.float32(-9))])
        found = v[np.rint(v * inv) != np.rint(v.astype(np.float64) * np.float64(inv))]
    x = rng.choice(found, (m, k))
    x[np.arange(m), rng.integers(0, k, m)] = peak
    return x


@pytest.mark.parametrize("m,k", [(5, 64), (3, 4096), (3, 4097), (200, 1001), (300, 5000), (200, 9001), (600, 2048), (2, 40000)])
def test_codes_follow_the_documented_product(cuda, clq, m, k):
    """code = round(v * (1 / step)), the product rounded to f32 before it is rounded to a code."""
    torch = cuda
    x = border_rows(m, k, seed=k)
    step = np.maximum(FLT_MIN, np.abs(x).max(1, keepdims=True) / np.float32(127))
    inv = np.float32(1) / step
    want = np.rint(x * inv)
    assert (want != np.rint(x.astype(np.float64) * inv)).sum() > m * k // 2  # one rounding fewer gives other codes
    d = torch.from_numpy(x).cuda()
    zero = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    for q in (clq.quantize_rows(d), clq.norm_quantize(zero, torch.ones(k, device="cuda"), residual=d)[0],
              clq.norm_quantize(zero, None, residual=d)[0]):
        assert np.array_equal(q.codes.cpu().numpy(), want.astype(np.int8))
    assert np.array_equal(clq.quantize_rows(d).scales.cpu().numpy(), step[:, 0])


def far_gates(torch, m, k, xtype):
    """(gate, up) whose rows lie, or mostly lie, where e^-gate leaves f32."""
    gen = torch.Generator(device="cuda").manual_seed(m + k)

    def uniform(low, high):
        return torch.rand(m, k, device="cuda", generator=gen, dtype=torch.float64) * (high - low) + low
    most = 4.0 if xtype == "float16" else 38.0  # decimal exponents of up
    gate, up = uniform(-220, -87), 10 ** uniform(-2, most) * torch.sign(uniform(-1, 1))
    few = torch.tensor([-88.0, -95.0, -120.0, -300.0], dtype=torch.float64, device="cuda")
    for r in range(m):
        kind = r % 6
        if kind == 1:  # the smallest value must not lead the row
            gate[r] = few.repeat(k // 4 + 1)[:k]
            up[r] = torch.arange(1.0, 5.0, device="cuda", dtype=torch.float64).repeat(k // 4 + 1)[:k]
        elif kind == 2:  # as far as the type goes, beside one value of the row's kind above
            gate[r] = -60000.0 if xtype == "float16" else torch.where(uniform(0, 1)[r] < 0.5, -1e30, -3e38)
            gate[r, k // 2] = -88.0
            up[r] = 10.0 ** most
        elif kind == 3:  # beside values of ordinary size
            gate[r, k // 3:] = uniform(-3, 3)[r, k // 3:]
            gate[r, :k // 3] = -60000.0 if xtype == "float16" else -1e38
            up[r] = uniform(-2, 2)[r]
            gate[r, k - 1], up[r, k - 1] = 1.5, 1.0
        elif kind == 4:  # both sides of where the formula changes
            gate[r], up[r] = uniform(-87.5, -86.5)[r], uniform(1, 2)[r]
        elif kind == 5:  # results about the smallest normal number and below it
            gate[r], up[r] = uniform(-200, -170)[r], 10.0 ** most
    dtype = getattr(torch, xtype)
    return gate.to(dtype), up.to(dtype)


@pytest.mark.parametrize("m,k", [(6, 4), (6, 96), (12, 1001), (6, 4096), (6, 4099), (160, 5003), (600, 2048), (600, 9000),
                                 (300, 9001), (6, 40000)])
@pytest.mark.parametrize("xtype", ["float32", "bfloat16", "float16"])
def test_swiglu_of_rows_of_far_gates(cuda, clq, m, k, xtype):
    """Gates below -87, where silu decays to 0 however large they are, lead or share a row.
    v is within 11 U and 2^-137 of the exact value (include/clq.h), the peak too, peak / 127,
    1 / step and the product round once each: a code is within 127 * 25 U of the quotient and, as a step
    has FLT_MIN at least, 2^-137 / 2^-126 twice more; the scale within 12 U and 2^-137 / 127, and the
    half of a smallest number where it is FLT_MIN or less."""
    torch = cuda
    gate, up = far_gates(torch, m, k, xtype)
    q = clq.swiglu_quantize(gate, up)
    g = gate.double()
    v = g * torch.sigmoid(g) * up.double()
    assert torch.isfinite(v).all()
    peak = v.abs().amax(1)
    assert (peak > 0).all()
    step = torch.clamp(peak / 127, min=2.0 ** -126)
    # a peak under the bound may come out as 0 or not: a row of zeros has scale 1, and codes 0 like the other
    nothing = (peak <= 2.0 ** -137) & (q.scales == 1)
    assert (((q.scales.double() - step).abs() <= 12 * U * step + 2.0 ** -137) | nothing).all()
    ideal = (v / step[:, None]).clamp(-127, 127)
    assert ((q.codes.double() - ideal).abs() <= 0.5 + 127 * 25 * U + 2 * 2.0 ** -11).all()


def test_gates_that_are_not_finite(cuda, clq):
    torch = cuda
    for k in (8, 4097, 40000):
        gate = torch.full((4, k), -90.0, device="cuda")
        up = torch.ones(4, k, device="cuda")
        gate[0, k - 1], gate[1, 0], gate[2, k // 2] = float("-inf"), float("nan"), float("inf")
        q = clq.swiglu_quantize(gate, up)
        assert torch.isnan(q.scales[:3]).all() and not q.codes[:3].any() and q.scales[3].item() == 2.0 ** -126


@pytest.mark.parametrize("k", [16, 100, 4096, 5001, 40000])
@pytest.mark.parametrize("rtype", ["float32", "bfloat16"])
def test_norm_of_small_rows_without_epsilon(cuda, clq, k, rtype):
    """Where the squares leave f32 downwards the scale is NaN as it is upwards, never infinite; above
    2^-125 it is right: the sum of squares within (k / 32 + 24) U as for any row and 2^-24 for what
    squares lost, halved by the root, and 20 U for the steps around it."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(k)
    sign = torch.sign(torch.randn(8, k, device="cuda", generator=gen))
    sizes = [2.0 ** -62, 2.0 ** -64, 1e-25, 1e-38, 2.0 ** -133, 1.0, 0.0, 2.0 ** -61.5]
    h = (sign * torch.tensor(sizes, device="cuda")[:, None]).to(getattr(torch, rtype))
    zero = torch.zeros(8, k, device="cuda", dtype=torch.bfloat16)
    g = torch.ones(k, device="cuda")
    for q in (clq.norm_quantize(h, g, 0.0), clq.norm_quantize(zero, g, 0.0, residual=h)[0], clq.norm_quantize(h, g, 1e-44)):
        for row in (1, 2, 3, 4):
            assert torch.isnan(q.scales[row]) and not q.codes[row].any(), row
        assert q.scales[6].item() == 1.0 and not q.codes[6].any()
        for row in (0, 5, 7):
            d = h[row].double()
            want = d.abs().max() / 127 / torch.sqrt((d * d).mean())
            assert abs(q.scales[row].double() / want - 1).item() <= (k / 64 + 33) * U
            assert torch.equal(q.codes[row].float(), 127 * sign[row])
    fine = clq.norm_quantize(h, g, 1e-5)
    assert torch.isfinite(fine.scales).all()
    # a weight of zeros leaves nothing to code: an all-zero row
    assert (clq.norm_quantize(h, 0 * g, 0.0).scales == 1).all()


def test_the_stride_of_a_single_row_does_not_choose_its_kernel(cuda, clq):
    """One row, one weight row or both with the base on the 16-byte grid and a stride off it: the same
    result as with a padded stride, and about its time (the kernels for rows off the grid take twice it)."""
    torch, lib = cuda, clq._lib.lib
    k, n = 5123, 4096
    gen = torch.Generator(device="cuda").manual_seed(1)
    pitch = (k + 15) // 16 * 16
    w = torch.randint(-128, 128, (n, pitch), device="cuda", generator=gen, dtype=torch.int16).to(torch.int8)
    x = torch.randint(-128, 128, (64, pitch), device="cuda", generator=gen, dtype=torch.int16).to(torch.int8)
    ones = torch.ones(n, device="cuda")

    def product(m, rows, ldx, ldw):
        out = torch.zeros(m, rows, device="cuda")

        def call():
            rc = lib.clq_linear_int8_device(x.data_ptr(), ldx, ones.data_ptr(), m, w.data_ptr(), ldw, ones.data_ptr(), rows, k, None,
                                            0, out.data_ptr(), 0, rows, torch.cuda.current_stream().cuda_stream)
            assert rc == 0, clq._lib.last_error()
        return out, call

    values = torch.randn(1, 16384, device="cuda", generator=gen)

    def rows(ldx, ldc):
        codes, scales = torch.zeros(16384, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")

        def call():
            assert lib.clq_quantize_rows_device(values.data_ptr(), 0, 1, 16384, ldx, codes.data_ptr(), ldc, scales.data_ptr(),
                                                torch.cuda.current_stream().cuda_stream) == 0
        return codes, call

    def micros(call, times=100):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(times):
                call()
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b) * 1e3 / times)
        return best

    for padded, tight in ((product(1, n, pitch, pitch), product(1, n, k, pitch)),
                          (product(64, 1, pitch, pitch), product(64, 1, pitch, k)),
                          (rows(16384, 16384), rows(16385, 16385))):
        fast, slow = micros(padded[1]), micros(tight[1])
        assert torch.equal(padded[0], tight[0]) and padded[0].any()
        assert slow < 1.4 * fast, (fast, slow)


def test_rows_that_share_memory_are_read(cuda, clq):
    """One row for every token, or overlapping windows of a buffer: codes, residuals, values."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    row = clq.quantize_rows(torch.randn(1, 160, device="cuda", generator=gen))
    w = clq.quantize_rows(torch.randn(48, 160, device="cuda", generator=gen))
    bias = torch.randn(48, device="cuda", generator=gen)
    for m in (2, 20, 150):
        x = clq.quantize_rows(torch.randn(m, 160, device="cuda", generator=gen))
        want = clq.linear_int8(x, w, residual=bias.expand(m, 48).contiguous())
        assert torch.equal(clq.linear_int8(x, w, residual=bias.expand(m, 48)), want)
        out = torch.empty(m, 48, device="cuda")
        assert torch.equal(clq.linear_int8(x, w, out=out, residual=bias.expand(m, 48)), want)
        same = clq.Int8Rows(row.codes.expand(m, 160), row.scales.expand(m))
        assert torch.equal(clq.linear_int8(same, w), clq.linear_int8(row, w).expand(m, 48))
        assert torch.equal(same.dequantize(), row.dequantize().expand(m, 160))
    line = torch.randn(500, device="cuda", generator=gen)
    windows = line.unfold(0, 100, 7)
    assert windows.stride(0) == 7
    assert torch.equal(clq.quantize_rows(windows).codes, clq.quantize_rows(windows.contiguous()).codes)
    codes = row.codes[0].unfold(0, 32, 16)
    wide = clq.Int8Rows(codes, torch.ones(len(codes), device="cuda"))
    assert torch.equal(clq.linear_int8(wide, wide).double(), codes.double() @ codes.double().t())


def test_refusals_are_value_errors_whatever_else_is_given(cuda, clq):
    torch = cuda
    x = torch.randn(4, 64, device="cuda")
    q = clq.quantize_rows(x)
    out, h = torch.empty(4, 4, device="cuda"), torch.cuda.current_stream().cuda_stream
    for call in (
        lambda: clq.linear_int8(q, q, out=out, residual="none"), lambda: clq.linear_int8(q, q, out=out, residual=out[0]),
        lambda: clq.linear_int8(q, q, out=out, residual=torch.zeros(4, 4)),
        lambda: clq.linear_int8(q, q, out=out, residual=out.t()), lambda: clq.linear_int8(q, q, out="out", stream=h),
        lambda: clq.linear_int8(q, q, residual=torch.zeros(4, 4), stream=h),
        lambda: clq.quantize_rows(x.cpu(), stream=h), lambda: clq.quantize_rows([1.0], stream=h),
        lambda: clq.norm_quantize(x, torch.ones(64), stream=h), lambda: clq.norm_quantize(x, residual=x.cpu(), stream=h),
        lambda: clq.swiglu_quantize(x, x.cpu(), stream=h), lambda: q.dequantize(out=torch.empty(4, 64), stream=h),
    ):
        with pytest.raises(ValueError):
            call()
