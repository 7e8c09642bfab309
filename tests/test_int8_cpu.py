"""8-bit integer linear layers: what is refused, before any launch (no GPU)."""
import ctypes as C

import pytest
import torch


def _refused(lib, call, words):
    call()
    try:
        assert lib.b200_last_error() == 1
        assert words in lib.b200_last_error_string(), lib.b200_last_error_string()
    finally:
        lib.b200_clear_error()


# addresses that the checks look at and nothing reads: every call below is refused before a launch
A, ODD = 4096, 4104


@pytest.mark.parametrize("suffix", ["f16", "bf16"])
def test_rows_refuse(lib, suffix):
    eps = C.c_float(1e-5)
    f = lambda name: getattr(lib, f"b200_{name}_i8_{suffix}")           # noqa: E731
    for bad in range(4):
        p = [A, A, A, A]
        p[bad] = None
        _refused(lib, lambda: f("rmsnorm")(*p, 2, 64, eps, 0), b"rmsnorm_i8")
        p = [A, A, A, A, A]
        p[bad + 1] = None
        _refused(lib, lambda: f("add_rmsnorm")(*p, 2, 64, eps, 0), b"add_rmsnorm_i8")
    _refused(lib, lambda: f("rmsnorm")(A, A, A, A, 2, 0, eps, 0), b"rmsnorm_i8")
    _refused(lib, lambda: f("quant_rows")(A, A, A, 2, 0, 0), b"quant_rows_i8")
    _refused(lib, lambda: f("quant_rows")(A, A, A, 2, 2 ** 30 + 1, 0), b"quant_rows_i8")
    _refused(lib, lambda: f("quant_rows")(A, None, A, 2, 8, 0), b"quant_rows_i8")
    _refused(lib, lambda: f("quant_rows")(A, A, A, 2 ** 30 + 1, 8, 0), b"quant_rows_i8")
    _refused(lib, lambda: f("rmsnorm")(A, A, A, A, 2 ** 30 + 1, 64, eps, 0), b"rmsnorm_i8")
    _refused(lib, lambda: f("add_rmsnorm")(A, A, A, A, A, 2 ** 30 + 1, 64, eps, 0), b"add_rmsnorm_i8")
    f("quant_rows")(None, None, None, 0, 8, 0)                           # no rows: nothing to do, nothing to refuse
    assert lib.b200_last_error() == 0


@pytest.mark.parametrize("suffix", ["f16", "bf16", "f32"])
def test_gemm_refuses(lib, suffix):
    f = getattr(lib, f"b200_gemm_i8_{suffix}")
    for bad in (0, 1, 2, 3, 5):
        p = [A, A, A, A, None, A]
        p[bad] = None
        _refused(lib, lambda: f(*p, 4, 64, 64, 0, 0), b"gemm_i8: bad arguments")
    ok = [A, A, A, A, None, A]
    for m, n, k, epi, words in ((4, 0, 64, 0, b"bad arguments"), (4, 64, 0, 0, b"bad arguments"), (4, 64, 72, 0, b"multiple of 16"),
                                (4, 64, 131072, 0, b"at most 131056"),
                                (2 ** 30 + 1, 64, 64, 0, b"at most 2^30"), (4, 2 ** 30 + 1, 64, 0, b"at most 2^30"),
                                (4, 63, 64, 1, b"odd number"), (4, 64, 64, 2, b"unknown epilogue")):
        _refused(lib, lambda: f(*ok, m, n, k, epi, 0), words)
    _refused(lib, lambda: f(ODD, A, A, A, None, A, 4, 64, 64, 0, 0), b"16-byte aligned")
    _refused(lib, lambda: f(A, A, ODD, A, None, A, 4, 64, 64, 0, 0), b"16-byte aligned")
    f(None, None, None, None, None, None, 0, 64, 64, 0, 0)
    assert lib.b200_last_error() == 0


@pytest.fixture
def ops(lib, monkeypatch):
    """The wrappers with tensors of the host: their checks run, a call that gets past them fails the test."""
    from vllm_rs_b200 import ops as o
    def contiguous(*ts):
        if not all(t is None or t.is_contiguous() for t in ts):
            raise ValueError("not contiguous")

    def launched(*_):
        raise AssertionError("a call that should have been refused reached the library")

    monkeypatch.setattr(o, "_on_device", contiguous)
    monkeypatch.setattr(o._lib, "check", launched)
    return o


def test_wrappers_refuse_rows(ops):
    x, w = torch.zeros(3, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.float16)
    for call in (lambda: ops.rmsnorm_i8(x, w[:32], 1e-5), lambda: ops.rmsnorm_i8(x, w.float(), 1e-5),
                 lambda: ops.rmsnorm_i8(x[0], w, 1e-5), lambda: ops.rmsnorm_i8(x.t(), w, 1e-5),
                 lambda: ops.add_rmsnorm_i8(x[:2], x, w, 1e-5), lambda: ops.add_rmsnorm_i8(x.float(), x, w, 1e-5),
                 lambda: ops.quant_rows_i8(x, out=torch.zeros(3, 64)), lambda: ops.quant_rows_i8(x, out=torch.zeros(3, 32, dtype=torch.int8)),
                 lambda: ops.quant_rows_i8(x, scales=torch.zeros(4)), lambda: ops.quant_rows_i8(x, scales=torch.zeros(3, dtype=torch.float16))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.quant_rows_i8(x.float())


def test_wrappers_refuse_tensors_of_the_host(lib, monkeypatch):
    from vllm_rs_b200 import ops
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    x = torch.zeros(3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="current device"):
        ops.quant_rows_i8(x)


def test_wrappers_refuse_products(ops):
    q, w, s, t = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(10, 64, dtype=torch.int8), torch.zeros(3), torch.zeros(10)
    f16 = torch.float16
    for call in (lambda: ops.gemm_i8(q[:, :32].contiguous(), s, w, t), lambda: ops.gemm_i8(q.to(torch.uint8), s, w, t),
                 lambda: ops.gemm_i8(q, s[:2], w, t), lambda: ops.gemm_i8(q, s, w, t[:9]), lambda: ops.gemm_i8(q, s.half(), w, t),
                 lambda: ops.gemm_i8(q, s[:, None], w, t), lambda: ops.gemm_i8(q, s, w, t, bias=t),
                 lambda: ops.gemm_i8(q, s, w, t, bias=torch.zeros(9, dtype=f16)), lambda: ops.gemm_i8(q, s, w, t, epilogue=2),
                 lambda: ops.gemm_i8(q, s, w[:9], t[:9], epilogue=ops.EPI_SILU_MUL),
                 lambda: ops.gemm_i8(q, s, w, t, out=torch.zeros(3, 5, dtype=f16)),
                 lambda: ops.gemm_i8(q, s, w, t, out=torch.zeros(3, 10)), lambda: ops.gemm_i8(q, s, w.t(), t)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.gemm_i8(q, s, w, t, dtype=torch.float64)


@pytest.mark.parametrize("rows,width", [(2 ** 32 + 3, 1), (1, 2 ** 32 + 16), (2 ** 30 + 1, 16)])
def test_wrappers_refuse_what_32_bits_do_not_count(ops, rows, width):
    make = lambda *shape, dtype=torch.float16: torch.empty(shape, dtype=dtype, device="meta")        # noqa: E731
    x, w, q = make(rows, width), make(width), make(rows, width, dtype=torch.int8)
    one, s1, s = make(1, width, dtype=torch.int8), make(1, dtype=torch.float32), make(rows, dtype=torch.float32)
    for call in (lambda: ops.quant_rows_i8(x), lambda: ops.rmsnorm_i8(x, w, 1e-5), lambda: ops.add_rmsnorm_i8(x, x, w, 1e-5),
                 lambda: ops.gemm_i8(q, s, one, s1), lambda: ops.gemm_i8(one, s1, q, s)):
        with pytest.raises(ValueError, match="2\\^30"):
            call()
