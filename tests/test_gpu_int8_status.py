"""8-bit kernels that run while the device status word is set (needs a B200).

Their waits then give up at once wherever what they wait for is not there yet.  A launch
has to end, with its copies landed; what it writes is right, and the rest stays as it was;
the status reads the code once, and the next launch is whole.  The word is set as in
test_gpu_status.py: by the bounded wait of an all-reduce whose other rank never runs.
"""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

TYPES = {"float32": 0, "bfloat16": 1, "float16": 2}


def status(clq):
    s = ctypes.c_int(-1)
    assert clq._lib.lib.clq_device_status(ctypes.byref(s)) == 0, clq._lib.last_error()
    return s.value


class AbsentRank:
    """expire() leaves CLQ_ERR_TIMEOUT in the status word."""

    def __init__(self, torch, clq, synth):
        self.clq, self.lib, self.bufs, self.handle = clq, clq._lib.lib, [], ctypes.c_void_p()
        world, cap = 2, 4096
        for _ in range(world):
            recv, flags = ctypes.c_void_p(), ctypes.c_void_p()
            clq._lib.check(self.lib.clq_tp_buffers(world, cap, ctypes.byref(recv), ctypes.byref(flags)))
            self.bufs.append((recv, flags))
        r, f = ((ctypes.c_void_p * world)(*[b[i].value for b in self.bufs]) for i in range(2))
        clq._lib.check(self.lib.clq_tp_create(0, world, cap, r, f, ctypes.byref(self.handle)))
        self.store = clq.Store("q4_k", 512, 1024, synth.packed_blocks("q4_k", 512, 1024, seed=77))
        self.x, self.out = torch.zeros(1, 1024, device="cuda"), torch.empty(1, 512, device="cuda")
        self.torch = torch

    def expire(self):
        assert self.lib.clq_linear_allreduce_device(self.store.handle, 0, 512, self.x.data_ptr(), 0, 1, self.out.data_ptr(), 512,
                                                    self.handle, None) == 0, self.clq._lib.last_error()
        self.torch.cuda.synchronize()

    def close(self):
        self.lib.clq_tp_free(self.handle)
        for recv, flags in self.bufs:
            self.lib.clq_tp_buffers_free(recv, flags)
        self.store.close()


@pytest.fixture
def absent(cuda, clq, synth, monkeypatch):
    monkeypatch.setenv("CLQ_TP_WAIT_POLLS", "20000")
    assert status(clq) == 0
    a = AbsentRank(cuda, clq, synth)
    yield a
    a.close()
    assert status(clq) == 0


def rand(torch, *shape, seed):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("m,k,xtype,kind", [(2000, 4096, "bfloat16", "norm"), (2000, 8192, "float16", "norm"),
                                            (1500, 14336, "bfloat16", "swiglu"), (600, 24000, "bfloat16", "swiglu"),
                                            (700, 9001, "float16", "norm"), (2000, 5003, "bfloat16", "rows"),
                                            (500, 20001, "bfloat16", "swiglu"), (300, 30001, "float16", "norm")])
def test_streamed_rows_stop_where_a_row_does_not_come(cuda, clq, absent, m, k, xtype, kind):
    torch, lib = cuda, clq._lib.lib
    dtype, t = getattr(torch, xtype), TYPES[xtype]
    x, other = rand(torch, m, k, seed=1).to(dtype), rand(torch, m, k, seed=2).to(dtype)
    g = rand(torch, k, seed=3)

    def call():
        pitch = (k + 15) // 16 * 16
        codes, scales = torch.full((m, pitch), 99, dtype=torch.int8, device="cuda"), torch.full((m,), -1.0, device="cuda")
        total = other.clone()
        torch.cuda.synchronize()
        if kind == "swiglu":
            rc = lib.clq_swiglu_quantize_device(other.data_ptr(), k, x.data_ptr(), k, t, m, k, codes.data_ptr(), pitch,
                                                scales.data_ptr(), None)
        elif kind == "rows":
            rc = lib.clq_quantize_rows_device(x.data_ptr(), t, m, k, k, codes.data_ptr(), pitch, scales.data_ptr(), None)
        else:  # onto its residual
            rc = lib.clq_norm_quantize_device(x.data_ptr(), t, m, k, k, g.data_ptr(), 1e-5, total.data_ptr(), t, k,
                                              total.data_ptr(), k, codes.data_ptr(), pitch, scales.data_ptr(), None)
        assert rc == 0, clq._lib.last_error()
        return codes[:, :k], scales, total

    want = call()
    assert status(clq) == 0 and (want[1] > 0).all()
    for _ in range(3):
        absent.expire()
        codes, scales, total = call()
        assert clq._lib.STATUS_NAMES[status(clq)] == "CLQ_ERR_TIMEOUT"
        done = scales != -1
        print(f"{int(done.sum())} of {m} rows written")
        assert torch.equal(scales[done], want[1][done]) and torch.equal(codes[done], want[0][done])
        assert (codes[~done] == 99).all()
        assert ((total == want[2]) | (total == other)).all()
    assert status(clq) == 0
    assert all(torch.equal(a, b) for a, b in zip(call(), want))


@pytest.mark.parametrize("m,n,k", [(24, 4096, 4096), (40, 1024, 16384), (128, 4096, 4096), (64, 512, 40000), (45, 5003, 2051),
                                   (256, 6144, 4096), (32, 28672, 4096), (512, 4096, 14336), (2048, 4096, 4096),
                                   (300, 19200, 9000)])
@pytest.mark.parametrize("onto", [False, True])
def test_products_write_whole_sums_or_nothing(cuda, clq, absent, m, n, k, onto):
    """Tiles of one CTA, tiles whose parts of K are a cluster, and SM pairs."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(m)

    def rows(count):
        c = torch.randint(-128, 128, (count, (k + 15) // 16 * 16), device="cuda", generator=gen, dtype=torch.int16).to(torch.int8)
        return clq.Int8Rows(c[:, :k], torch.rand(count, device="cuda", generator=gen) + 0.5)
    x, w, before = rows(m), rows(n), rand(torch, m, n, seed=5)

    def call():
        out = before.clone()
        torch.cuda.synchronize()
        return clq.linear_int8(x, w, out=out, residual=out if onto else None)
    want = call()
    assert status(clq) == 0
    for _ in range(5):
        absent.expire()
        got = call()
        assert clq._lib.STATUS_NAMES[status(clq)] == "CLQ_ERR_TIMEOUT"
        print(f"{(got == want).double().mean().item():.3f} written")
        assert ((got == want) | (got == before)).all()
    assert torch.equal(call(), want)
