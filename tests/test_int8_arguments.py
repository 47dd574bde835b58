"""Refusals of the 8-bit row calls (include/clq.h, "8-bit activations") that need no GPU."""
import importlib

import pytest

FAKE = 256  # a non-null address that the checks never reach


def c(clq, name, *args):
    return getattr(clq._lib.lib, name)(*args)


def test_row_quantizers_check_arguments_before_device_work(clq):
    q = "clq_quantize_rows_device"
    assert c(clq, q, FAKE, 7, 2, 8, 8, FAKE, 8, FAKE, None) == 1
    assert "unknown row type 7" in clq._lib.last_error()
    assert c(clq, q, FAKE, 0, -1, 8, 8, FAKE, 8, FAKE, None) == 2
    assert c(clq, q, FAKE, 0, 2, 8, -8, FAKE, 8, FAKE, None) == 2      # rows backwards
    assert c(clq, q, FAKE, 0, 2, 8, 8, FAKE, 7, FAKE, None) == 2       # code rows overlap
    assert c(clq, q, None, 0, 2, 8, 8, FAKE, 8, FAKE, None) == 1
    assert c(clq, q, FAKE, 0, 2, 8, 8, None, 8, FAKE, None) == 1
    assert c(clq, q, FAKE, 0, 2, 8, 8, FAKE, 8, None, None) == 1
    assert c(clq, q, None, 0, 0, 8, 8, None, 8, None, None) == 0       # no rows: nothing to do


def test_norm_quantizer_checks_its_residual(clq):
    def call(rtype=0, residual=FAKE, out=FAKE, ldro=8, eps=1e-5, xtype=1):
        return c(clq, "clq_norm_quantize_device", FAKE, xtype, 2, 8, 8, FAKE, eps, residual, rtype, 8, out, ldro, FAKE, 8,
                 FAKE, None)
    assert call(rtype=2) == 1                      # bf16 rows beside an f16 residual
    assert "residual type 2" in clq._lib.last_error()
    assert call(residual=None) == 1                # an output without a residual
    assert call(ldro=7) == 2
    assert call(eps=-1.0) == 1
    assert call(eps=float("nan")) == 1
    assert c(clq, "clq_norm_quantize_device", 512, 0, 2, 8, 8, None, 0.0, FAKE, 0, 16, FAKE, 8, FAKE, 8, FAKE, None) == 2
    assert "two row strides" in clq._lib.last_error()  # in place, but not on itself
    assert c(clq, "clq_norm_quantize_device", FAKE, 1, 2, 8, 8, None, 0.0, 512, 0, 8, FAKE, 8, FAKE, 8, FAKE, None) == 2


def test_swiglu_and_dequantize_check_arguments(clq):
    s = "clq_swiglu_quantize_device"
    assert c(clq, s, FAKE, 8, FAKE, 8, 9, 2, 8, FAKE, 8, FAKE, None) == 1
    assert c(clq, s, FAKE, -8, FAKE, 8, 0, 2, 8, FAKE, 8, FAKE, None) == 2
    assert c(clq, s, None, 8, FAKE, 8, 0, 2, 8, FAKE, 8, FAKE, None) == 1
    assert c(clq, s, FAKE, 8, None, 8, 0, 2, 8, FAKE, 8, FAKE, None) == 1
    d = "clq_dequantize_rows_device"
    assert c(clq, d, FAKE, 8, FAKE, 2, 8, FAKE, 5, 8, None) == 1
    assert c(clq, d, FAKE, 8, FAKE, 2, 8, FAKE, 0, 7, None) == 2
    assert c(clq, d, FAKE, 8, None, 2, 8, FAKE, 0, 8, None) == 1
    assert c(clq, d, None, 8, None, 0, 8, None, 0, 8, None) == 0


def test_product_checks_arguments(clq):
    def call(x=FAKE, ldx=64, xs=FAKE, m=2, w=FAKE, ldw=64, ws=FAKE, n=3, k=64, res=None, ldr=0, out=FAKE, otype=0, ldo=3):
        return c(clq, "clq_linear_int8_device", x, ldx, xs, m, w, ldw, ws, n, k, res, ldr, out, otype, ldo, None)
    assert call(otype=4) == 1
    assert call(k=-1) == 2
    assert call(ldx=63) == 2
    assert call(ldw=63) == 2
    assert call(ldo=2) == 2
    assert call(res=FAKE, ldr=2) == 2
    assert call(res=FAKE, ldr=4) == 2                         # onto the output, with another stride
    assert call(res=FAKE, ldr=3, otype=1) == 2                # or of another type
    assert call(k=131072, ldx=131072, ldw=131072) == 9        # 32-bit sums could wrap
    assert "131071" in clq._lib.last_error()
    for missing in ("x", "xs", "w", "ws", "out"):
        assert call(**{missing: None}) == 1, missing
    assert call(m=0, x=None, xs=None) == 0
    assert call(n=0, w=None, ws=None, ldo=0) == 0


def test_addresses_off_their_type_are_refused(clq):
    def norm(x=FAKE, xtype=1, w=FAKE, res=FAKE, rtype=0, out=FAKE + 256, codes=FAKE, scales=FAKE):
        return c(clq, "clq_norm_quantize_device", x, xtype, 2, 8, 8, w, 1e-5, res, rtype, 8, out, 8, codes, 8, scales, None)
    for bad in (dict(x=FAKE + 1), dict(w=FAKE + 2), dict(res=FAKE + 2), dict(out=FAKE + 258), dict(scales=FAKE + 2),
                dict(x=FAKE + 2, xtype=0)):
        assert norm(**bad) == 1, bad
        assert "alignment" in clq._lib.last_error()
    assert c(clq, "clq_swiglu_quantize_device", FAKE + 1, 8, FAKE, 8, 2, 2, 8, FAKE, 8, FAKE, None) == 1
    assert c(clq, "clq_swiglu_quantize_device", FAKE, 8, FAKE + 1, 8, 2, 2, 8, FAKE, 8, FAKE, None) == 1
    assert c(clq, "clq_dequantize_rows_device", FAKE, 8, FAKE + 2, 2, 8, FAKE, 1, 8, None) == 1
    assert c(clq, "clq_dequantize_rows_device", FAKE, 8, FAKE, 2, 8, FAKE + 1, 1, 8, None) == 1

    def product(xs=FAKE, ws=FAKE, res=None, out=FAKE, otype=1):
        return c(clq, "clq_linear_int8_device", FAKE, 64, xs, 2, FAKE, 64, ws, 3, 64, res, 3, out, otype, 3, None)
    for bad in (dict(xs=FAKE + 1), dict(ws=FAKE + 2), dict(res=FAKE + 2), dict(out=FAKE + 1), dict(out=FAKE + 2, otype=0)):
        assert product(**bad) == 1, bad
        assert "alignment" in clq._lib.last_error()


def test_valid_calls_need_a_device(clq):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert c(clq, "clq_quantize_rows_device", FAKE, 0, 2, 8, 8, FAKE, 8, FAKE, None) == 8
    assert c(clq, "clq_linear_int8_device", FAKE, 64, FAKE, 2, FAKE, 64, FAKE, 3, 64, None, 0, FAKE, 0, 3, None) == 8


def test_python_calls_refuse_host_tensors(clq):
    import torch
    x = torch.zeros(2, 8)
    for call in (lambda: clq.quantize_rows(x), lambda: clq.norm_quantize(x, torch.ones(8)),
                 lambda: clq.swiglu_quantize(x, x), lambda: clq.Int8Rows(x.to(torch.int8), torch.ones(2)),
                 lambda: clq.linear_int8(x, x)):
        with pytest.raises(ValueError):
            call()


def test_outputs_beside_inputs_in_one_buffer_are_told_from_overlapping_ones():
    import torch
    mod = importlib.import_module("cl-inference_b200.int8")
    both = torch.zeros(5, 24)
    left, right = both[:, :12], both[:, 12:]
    assert not mod._overlap(left, right) and not mod._overlap(right, left)
    assert mod._overlap(both[:, :13], right) and mod._overlap(right, both[:, 4:13])
    assert mod._overlap(both[:3], both[2:]) and not mod._overlap(both[:2], both[2:])
    mod._apart(left, both[:, :12], "out")  # the same view made twice
    with pytest.raises(ValueError):
        mod._apart(both[:, 1:13], left, "out")
