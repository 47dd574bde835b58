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
