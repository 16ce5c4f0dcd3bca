"""What the calls on 8-bit rows refuse, through the Python layer and at the C entry points: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

from tensor_parallel_amd import _native, int8

INVALID, UNSUPPORTED = -1, -2


def test_host_tensors():
    x, q, s = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    rows = int8.QuantizedRows(q, s, torch.float16)
    for call in (lambda: int8.quantize_activations(x), lambda: int8.rms_norm(x, x[0], 1e-5), lambda: int8.add_rms_norm(x, x, x[0], 1e-5), lambda: int8.linear(rows, q, s),
                 lambda: int8.swiglu_up(rows, q, s, q, s), rows.dequantize):
        with pytest.raises(_native.NativeLibraryError):
            call()


@pytest.fixture
def checks(monkeypatch):
    """The checks of arguments on host tensors; a call that got past them would fail at the library."""
    monkeypatch.setattr(_native, "require_device", lambda *_: None)
    monkeypatch.setattr(_native, "lib", lambda: pytest.fail("the call was not refused"))


F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: _native.quantize_rows(z(2, 8, dtype=torch.float32)), TypeError),
    (lambda: _native.quantize_rows(z(2, 8, dtype=torch.float64)), TypeError),
    (lambda: _native.quantize_rows(torch.tensor(1.0, dtype=F16)), ValueError),
    (lambda: _native.rms_norm_q8(z(2, 8), z(7), 1e-5), ValueError),
    (lambda: _native.rms_norm_q8(z(2, 8), z(8, dtype=BF16), 1e-5), ValueError),
    (lambda: _native.rms_norm_q8(z(2, 8), z(1, 8), 1e-5), ValueError),
    (lambda: _native.add_rms_norm_q8(z(2, 1), z(2, 8), z(8), 1e-5), ValueError),  # no broadcast residual
    (lambda: _native.add_rms_norm_q8(z(2, 8, dtype=BF16), z(2, 8), z(8), 1e-5), ValueError),
    (lambda: _native.dequantize_rows(z(2, 8), torch.zeros(2), F16), TypeError),
    (lambda: _native.dequantize_rows(z(2, 8, dtype=I8), torch.zeros(3), F16), ValueError),
    (lambda: _native.dequantize_rows(z(2, 8, dtype=I8), torch.zeros(2, 1), F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), dtype=F16), TypeError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2, dtype=F16), z(4, 8, dtype=I8), torch.zeros(4), dtype=F16), TypeError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), dtype=torch.float32), TypeError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 7, dtype=I8), torch.zeros(4), dtype=F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(5), dtype=F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(3), z(4, 8, dtype=I8), torch.zeros(4), dtype=F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), z(3), dtype=F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), z(4, dtype=BF16), dtype=F16), ValueError),
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), dtype=F16, addend=z(1, 4)), ValueError),  # no broadcast addend
    (lambda: _native.linear_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), dtype=F16, copy=z(2, 4)), ValueError),
    (lambda: _native.swiglu_up_a8(z(2, 8, dtype=I8), torch.zeros(2), z(4, 8, dtype=I8), torch.zeros(4), z(5, 8, dtype=I8), torch.zeros(5), F16), ValueError),
])
def test_operands_that_do_not_fit(checks, call, error):
    with pytest.raises(error):
        call()


P, NULL = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0)  # an address that is never read


def at(offset):
    return ctypes.c_void_p((1 << 20) + offset)


def test_entry_points_check_what_they_are_given():
    lib = _native.lib()
    quantize = lambda q=P, rows=2, d=8, ldx=8, ldq=8, dtype=1, x=P, s=P: lib.tpamd_quantize_rows(x, q, s, rows, d, ldx, ldq, dtype, NULL)  # noqa: E731
    assert quantize(rows=-1) == quantize(d=-1) == quantize(ldx=7) == quantize(ldq=7) == quantize(dtype=2) == quantize(dtype=9) == INVALID
    assert quantize(x=NULL) == quantize(q=NULL) == quantize(s=NULL) == quantize(x=at(1)) == quantize(s=at(2)) == quantize(rows=1 << 31) == INVALID
    assert quantize(rows=0) == 0
    norm = lambda w=P, ldx=8: lib.tpamd_rms_norm_q8(P, w, P, P, 2, 8, ldx, 8, 1e-5, 0, NULL)  # noqa: E731
    assert norm(w=NULL) == norm(ldx=7) == norm(w=at(1)) == INVALID
    add = lambda r=P, s=P, ldr=8, lds=8: lib.tpamd_add_rms_norm_q8(P, r, P, s, P, P, 2, 8, 8, ldr, lds, 8, 1e-5, 0, NULL)  # noqa: E731
    assert add(r=NULL) == add(s=NULL) == add(ldr=7) == add(lds=7) == add(r=at(1)) == add(s=at(1)) == INVALID
    back = lambda y=P, ldy=8, dtype=2, rows=2: lib.tpamd_dequantize_rows(P, P, y, rows, 8, 8, ldy, dtype, NULL)  # noqa: E731
    assert back(y=NULL) == back(ldy=7) == back(dtype=3) == back(y=at(2)) == back(rows=-1) == INVALID and back(rows=0) == 0

    def linear(x=P, sx=P, w=P, sw=P, bias=NULL, y=P, m=2, n=4, k=16, ldx=16, ldw=16, ldy=4, dtype=0, act=0):
        return lib.tpamd_linear_a8(x, sx, w, sw, bias, y, m, n, k, ldx, ldw, ldy, dtype, act, NULL)

    assert linear(m=-1) == linear(n=-1) == linear(k=-1) == linear(ldx=15) == linear(ldw=15) == linear(ldy=3) == linear(dtype=2) == linear(act=2) == INVALID
    assert linear(x=NULL) == linear(sx=NULL) == linear(w=NULL) == linear(sw=NULL) == linear(y=NULL) == linear(y=at(1)) == linear(sx=at(2)) == linear(bias=at(1)) == INVALID
    assert linear(k=131072, ldx=131072, ldw=131072) == UNSUPPORTED and b"131072" in lib.tpamd_last_error()
    assert linear(m=0) == linear(n=0) == 0
    add = lambda a=P, lda=4, c=NULL: lib.tpamd_linear_a8_add(P, P, P, P, NULL, a, P, c, 2, 4, 16, 16, 16, lda, 4, 0, 0, NULL)  # noqa: E731
    assert add(a=NULL) == add(lda=3) == add(a=at(1)) == add(c=P) == add(c=at(1)) == INVALID
    pair = lambda u=P, su=P, ldw=16, k=16: lib.tpamd_swiglu_up_a8(P, P, P, P, u, su, P, 2, 4, k, 16, ldw, 4, 1, NULL)  # noqa: E731
    assert pair(u=NULL) == pair(su=NULL) == pair(ldw=15) == INVALID and pair(k=1 << 20) == UNSUPPORTED


def test_sizes_that_indices_do_not_reach():
    lib, most = _native.lib(), 1 << 30
    for d in (most, (1 << 31) - 1, 1 << 31):
        assert lib.tpamd_quantize_rows(P, P, P, 2, d, d, d, 0, NULL) == INVALID
        assert lib.tpamd_rms_norm_q8(P, P, P, P, 2, d, d, d, 1e-5, 0, NULL) == INVALID
        assert lib.tpamd_add_rms_norm_q8(P, P, P, P, P, P, 2, d, d, d, d, d, 1e-5, 0, NULL) == INVALID
        assert lib.tpamd_dequantize_rows(P, P, P, 2, d, d, d, 0, NULL) == INVALID
        for m, n in ((d, 16), (16, d)):
            assert lib.tpamd_linear_a8(P, P, P, P, NULL, P, m, n, 16, 16, 16, n, 0, 0, NULL) == INVALID
            assert lib.tpamd_swiglu_up_a8(P, P, P, P, P, P, P, m, n, 16, 16, 16, n, 0, NULL) == INVALID
