"""Rows in 8 bits (`tpamd_quantize_rows`, `tpamd_rms_norm_q8`, `tpamd_add_rms_norm_q8`, `tpamd_dequantize_rows`) against their definition in 64 bits. Codes are compared bit for bit: the
quotient 127 p / a of 16-bit values (of their products, 22 bits in fp16) is not so near to a half without lying on it that 64 bits would not tell."""
import numpy as np
import pytest
import torch

from tensor_parallel_amd import _native, int8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
EPS = 1e-5
DTYPES = [torch.bfloat16, torch.float16]


def definition(t, w=None):
    """(codes, scale) of a 2-D host tensor in 64 bits; w: of its RMS norm's rows."""
    t = t.double().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        p = t if w is None else t * w.double().numpy()
        factor = np.ones(len(t)) if w is None else 1 / np.sqrt((t * t).mean(1) + np.float64(np.float32(EPS)))
        a = np.abs(p).max(1) if p.shape[1] else np.zeros(len(p))
        bad, empty = ~np.isfinite(p).all(1), a < 2.0**-100
        fine = np.where(bad | empty, 1, a)
        codes = np.where((bad | empty)[:, None], 0, np.rint(127 * p / fine[:, None]))
        scale = np.where(bad, np.nan, np.where(empty, 1, a * factor / 127))
    return torch.from_numpy(codes).to(torch.int8), torch.from_numpy(scale)


def check(codes, scale, want, rtol):
    assert torch.equal(codes.cpu(), want[0])
    torch.testing.assert_close(scale.cpu().double(), want[1], rtol=rtol, atol=0, equal_nan=True)


# a row's scale: a division and a product (2^-23 each at most) and, behind a norm, half the error of a sum of squares in fp32: of the elements that a thread adds up in a row (at
# most 160 here) and 12 steps more, 2^-24 each, and 2^-22 of the square root
SCALE_RTOL, NORM_RTOL = 2.0**-22, 90 * 2.0**-24 + 2.0**-21


def rows_of(rows, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=g) * torch.where(torch.rand(d, generator=g) < 0.01, 30.0, 1.0) * (torch.rand(rows, 1, generator=g) + 0.01)
    return x.to(dtype)


SIZES = [(1, 1), (3, 7), (2, 8), (5, 100), (4, 512), (3, 520), (2, 2048), (7, 2056), (2, 4096), (3, 5504), (2, 8192), (2, 8200), (3, 16384), (2, 16392), (1, 20001), (1000, 64), (2050, 520), (2048, 2056), (2049, 4104), (2100, 16384), (16200, 520), (4100, 2056)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", SIZES)
def test_sizes(rows, d, dtype):
    x, r, w = rows_of(rows, d, dtype, 1), rows_of(rows, d, dtype, 2), (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(3))).to(dtype)
    check(*_native.quantize_rows(x.to(DEV)), definition(x), SCALE_RTOL)
    check(*_native.rms_norm_q8(x.to(DEV), w.to(DEV), EPS), definition(x, w), NORM_RTOL)
    total, codes, scale = _native.add_rms_norm_q8(r.to(DEV), x.to(DEV), w.to(DEV), EPS)
    want = (r.float() + x.float()).to(dtype)
    assert torch.equal(total.cpu(), want)
    check(codes, scale, definition(want, w), NORM_RTOL)
    for out in (torch.float32, dtype):
        assert torch.equal(_native.dequantize_rows(codes, scale, out).cpu(), (codes.cpu().float() * scale.cpu()[:, None]).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quotients_on_and_next_to_a_half(dtype):
    """A largest value of 127 makes the other values their own quotients; then rows of few significant bits, where a half is common."""
    halves = torch.arange(-127, 127.5, 0.5)
    rows = [torch.cat([torch.tensor([127.0 * s]), halves * s, torch.zeros(1)]) for s in (1.0, 0.25, 2.0**-9)]
    g = torch.Generator().manual_seed(0)
    rows += [(torch.randint(-16, 17, (512,), generator=g) * 0.125) for _ in range(3)]
    rows.append(torch.cat([torch.tensor([1.0]), (halves[:511] / 127)]))  # as near to a half as the dtype comes
    for row in rows:
        x = row[None].to(dtype)
        check(*_native.quantize_rows(x.to(DEV)), definition(x), SCALE_RTOL)
        w = torch.full((x.shape[1],), 1.5, dtype=dtype)
        check(*_native.rms_norm_q8(x.to(DEV), w.to(DEV), EPS), definition(x, w), NORM_RTOL)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [512, 515])
def test_rows_without_a_scale(dtype, d):
    x = rows_of(9, d, dtype, 4)
    x[1], x[2] = 0, -0.0
    x[3, 5], x[4, d - 1], x[5, 0] = float("nan"), float("inf"), float("-inf")
    x[6, 7], x[6, 8] = float("nan"), float("inf")
    x[7] *= 0.0
    x[7, 3] = 2.0**-110 if dtype is torch.bfloat16 else 2.0**-24  # below what a row needs, and the smallest value of fp16
    x[8] = torch.finfo(dtype).max
    w = torch.ones(d, dtype=dtype)
    codes, scale = _native.quantize_rows(x.to(DEV))
    check(codes, scale, definition(x), SCALE_RTOL)
    assert scale[1] == 1 and scale[2] == 1 and bool(scale[3:7].isnan().all()) and (scale[7] == 1) == (dtype is torch.bfloat16) and bool((codes[8] == 127).all())
    x[8] = 3.0  # (the squares of the largest values do not fit fp32, and the norm is zero then, as the 16-bit one)
    codes, scale = _native.rms_norm_q8(x.to(DEV), w.to(DEV), EPS)
    check(codes, scale, definition(x, w), NORM_RTOL)
    y = _native.linear_a8(codes, scale, torch.ones(4, d, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV), dtype=dtype)
    assert y.isnan().all(1).tolist() == [False] * 3 + [True] * 4 + [False] * 2  # and the product says which rows had none


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 100])
def test_strides_and_what_lies_between_rows(dtype, d):
    wide, rwide = rows_of(6, 2 * d + 24, dtype, 5).to(DEV), rows_of(6, 2 * d + 24, dtype, 6).to(DEV)
    w = torch.ones(2 * d, dtype=dtype, device=DEV)[::2]
    for x, r in [(wide[:, 8:8 + d], rwide[:, 16:16 + d]), (wide[:, 1:1 + d], rwide[:, :d]), (wide[:, :2 * d:2], rwide[:, :d]), (wide[:1, :d].expand(6, d), rwide[:, :d]),
                 (wide[::2, :d], rwide[1::2, :d]), (wide[:, :d].reshape(2, 3, d).transpose(0, 1), rwide[:, :d].reshape(3, 2, d))]:
        flat = x.reshape(-1, d).cpu()
        codes, scale = _native.quantize_rows(x)
        assert codes.shape == x.shape and scale.shape == x.shape[:-1] and codes.is_contiguous()
        check(codes.reshape(-1, d), scale.flatten(), definition(flat), SCALE_RTOL)
        total, codes, scale = _native.add_rms_norm_q8(r, x, w, EPS)
        want = (r.float() + x.float()).to(dtype).cpu()
        assert torch.equal(total.cpu(), want)
        check(codes.reshape(-1, d), scale.flatten(), definition(want.reshape(-1, d), w.cpu()), NORM_RTOL)
    # through the C entry points: pitches of every operand, and what lies between rows stays
    q, s = torch.full((7, d + 16), 99, dtype=torch.int8, device=DEV), torch.full((7,), 99.0, device=DEV)
    total = torch.full((7, d + 8), 99.0, dtype=dtype, device=DEV)
    stream = torch.cuda.current_stream(DEV).cuda_stream
    assert _native.lib().tpamd_add_rms_norm_q8(wide.data_ptr(), rwide.data_ptr(), w.contiguous().data_ptr(), total.data_ptr(), q.data_ptr(), s.data_ptr(), 6, d, wide.stride(0),
                                               rwide.stride(0), d + 8, d + 16, EPS, _native.dtype_code(dtype), stream) == 0
    want = (rwide[:, :d].float() + wide[:, :d].float()).to(dtype).cpu()
    check(q[:6, :d], s[:6], definition(want, w.cpu()), NORM_RTOL)
    assert torch.equal(total[:6, :d].cpu(), want)
    assert bool((q[6] == 99).all() and (q[:, d:] == 99).all() and s[6] == 99 and (total[6] == 99).all() and (total[:, d:] == 99).all())
    y = torch.full((7, d + 4), 99.0, device=DEV)
    assert _native.lib().tpamd_dequantize_rows(q.data_ptr(), s.data_ptr(), y.data_ptr(), 6, d, d + 16, d + 4, _native.F32, stream) == 0
    assert torch.equal(y[:6, :d], q[:6, :d].float() * s[:6, None]) and bool((y[6] == 99).all() and (y[:, d:] == 99).all())


def test_more_rows_than_one_launch_takes():
    rows = (1 << 20) + 3
    x = (torch.arange(rows * 8, device=DEV) % 251 - 125).reshape(rows, 8).to(torch.float16)
    codes, scale = _native.quantize_rows(x)
    most = x.float().abs().amax(1)
    assert torch.equal(codes, (x.double() * 127 / most.double()[:, None]).round().to(torch.int8))
    torch.testing.assert_close(scale, most / 127, rtol=SCALE_RTOL, atol=0)
    assert torch.equal(_native.dequantize_rows(codes, scale, torch.float32), codes.float() * scale[:, None])


@pytest.mark.parametrize("shape", [(0, 16), (2, 0), (0, 0), (2, 0, 8), (3, 1, 0)])
def test_nothing_to_do(shape):
    x = torch.zeros(shape, dtype=torch.float16, device=DEV)
    rows = int8.quantize_activations(x)
    assert rows.codes.shape == shape and rows.scale.shape == shape[:-1] and rows.dequantize().shape == shape and bool((rows.scale == 1).all())
    total, rows = int8.add_rms_norm(x, x, torch.ones(shape[-1], dtype=torch.float16, device=DEV), EPS)
    assert total.shape == shape and rows.codes.shape == shape and bool((rows.scale == 1).all())


def test_streams_graphs_and_gradients():
    x, w = rows_of(5, 4096, torch.bfloat16, 7).to(DEV), torch.ones(4096, dtype=torch.bfloat16, device=DEV)
    want = _native.add_rms_norm_q8(x, x, w, EPS)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        got = _native.add_rms_norm_q8(x, x, w, EPS)
    torch.cuda.current_stream(DEV).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, still = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        captured = (*_native.add_rms_norm_q8(still, still, w, EPS), _native.dequantize_rows(*_native.quantize_rows(still), torch.float32))
    for seed in (8, 9, 10):
        fresh = rows_of(5, 4096, torch.bfloat16, seed).to(DEV)
        still.copy_(fresh)
        graph.replay()
        eager = (*_native.add_rms_norm_q8(fresh, fresh, w, EPS), _native.dequantize_rows(*_native.quantize_rows(fresh), torch.float32))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
    leaf = x.clone().requires_grad_()
    with pytest.raises(NotImplementedError):
        int8.quantize_activations(leaf).dequantize(torch.float32).sum().backward()
    total, _ = int8.add_rms_norm(x, leaf, w, EPS)
    with pytest.raises(NotImplementedError):
        total.sum().backward()
