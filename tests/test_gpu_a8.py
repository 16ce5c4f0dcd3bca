"""Linears and gated pairs of 8-bit rows (`tpamd_linear_a8`, `tpamd_linear_a8_add`, `tpamd_swiglu_up_a8`) against their definition in 64 bits, on random codes and the extreme ones."""
import ctypes

import pytest
import torch

from tensor_parallel_amd import _native, int8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def codes(g, rows, k, low=-127):
    return torch.randint(low, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g)


def operands(m, n, k, dtype, seed=0, low=-127):
    """x, its scales, two weights with theirs, a bias, an addend. Products have a spread of about 1 and both signs."""
    g = torch.Generator(device=DEV).manual_seed(seed + m + 7 * n + 31 * k)
    unit = 1 / (73.0 * 73.0 * max(k, 1) ** 0.5)
    scales = [(torch.rand(count, device=DEV, generator=g) + 0.2) * by for count, by in ((m, 1.0), (n, unit), (n, unit))]
    return (codes(g, m, k, low), scales[0], codes(g, n, k, low), scales[1], codes(g, n, k, low), scales[2], torch.randn(n, device=DEV, generator=g).to(dtype),
            torch.randn(m, n, device=DEV, generator=g).to(dtype))


def product(x, sx, w, sw):
    """In 64 bits: the sums are exact there."""
    return (x.double() @ w.double().t().contiguous()) * sx.double()[:, None] * sw.double()


def step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, bound, dtype):
    """|got - want| <= bound + half a step of the result (and of fp16's smallest)."""
    off = (got.double() - want).abs()
    most = bound + step(dtype) * (want.abs() + bound) + (2.0**-25 if dtype is torch.float16 else 0)
    assert got.dtype is dtype and bool((off <= most).all()), f"{(off / most).max().item()} of the bound"


# Behind the exact sum, in fp32: its conversion, two products and the bias, 2^-24 each of what they round; the error function within 4 steps of a value below 2 (x / 2 of it).
F32 = 2.0**-21


def check(m, n, k, dtype, seed=0, low=-127):
    x, sx, g, sg, u, su, bias, addend = operands(m, n, k, dtype, seed, low)
    a, b = product(x, sx, g, sg), product(x, sx, u, su)
    one = _native.linear_a8(x, sx, g, sg, None, dtype)
    within(one, a, F32 * a.abs(), dtype)
    biased = a + bias.double()
    size = a.abs() + bias.double().abs()
    within(_native.linear_a8(x, sx, g, sg, bias, dtype), biased, F32 * size, dtype)
    within(_native.linear_a8(x, sx, g, sg, bias, dtype, _native.ACT_GELU), torch.nn.functional.gelu(biased), F32 * size, dtype)
    # with an addend: the product's own rounding, then the sum's
    copy = torch.full((m, n), float("nan"), dtype=dtype, device=DEV)
    total = _native.linear_a8(x, sx, g, sg, bias, dtype, addend=addend, copy=copy)
    assert torch.equal(total, (_native.linear_a8(x, sx, g, sg, bias, dtype).float() + addend.float()).to(dtype)) and torch.equal(total, copy)
    # silu(g) u: the exponential's argument is off by 2^-23 of it, and each factor and product by a few steps of fp32
    want = torch.nn.functional.silu(a) * b
    within(_native.swiglu_up_a8(x, sx, g, sg, u, su, dtype), want, 2.0**-21 * (2 + a.abs()) * (want.abs() + (a * b).abs() * 2.0**-2), dtype)
    return one


ROWS = [1, 2, 3, 8, 16, 17, 33, 64, 65, 127, 130, 257]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(1, 16), (7, 128), (50, 272), (129, 1040), (516, 384), (1000, 2064)])
def test_sizes(m, n, k):
    check(m, n, k, torch.float16 if m % 2 else torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (2, 3, 7), (5, 8, 15), (70, 33, 100), (300, 70, 1001), (1, 4096, 5504), (16, 16384, 8192), (40, 11008, 4096), (645, 2048, 4096), (701, 2750, 2064), (2103, 512, 5504),
                                   (1030, 4100, 1392)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ragged_and_real_sizes(m, n, k, dtype):
    check(m, n, k, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_do_not_depend_on_the_batch_they_are_in(dtype):
    """Sums are exact, so every kernel gives a row the same bits."""
    x, sx, w, sw, u, su, bias, _ = operands(300, 640, 1040, dtype)
    calls = [lambda n: _native.linear_a8(x[:n], sx[:n], w, sw, None, dtype), lambda n: _native.linear_a8(x[:n], sx[:n], w, sw, bias, dtype, _native.ACT_GELU),
             lambda n: _native.swiglu_up_a8(x[:n], sx[:n], w, sw, u, su, dtype)]
    for call in calls:
        whole = call(300)
        for rows in (1, 2, 16, 33, 64, 65, 128, 200):
            assert torch.equal(call(rows), whole[:rows])


@pytest.mark.parametrize("m", [1, 5, 64, 129])
def test_largest_sums(m):
    """Every code the lowest one there is, K the longest that is taken; then K a multiple of what the matrix pipe takes."""
    for k in (131071, 131056, 130944):
        x, w = (torch.full((r, k), -128, dtype=torch.int8, device=DEV) for r in (m, 20))
        sx, sw = torch.ones(m, device=DEV), torch.full((20,), 2.0**-20, device=DEV)
        y = _native.linear_a8(x, sx, w, sw, dtype=torch.bfloat16)
        assert bool((y.double() - 16384 * k * 2.0**-20).abs().max() <= step(torch.bfloat16) * 2048)
        w[:, ::2] = 127
        within(_native.linear_a8(x, sx, w, sw, dtype=torch.bfloat16), product(x, sx, w, sw), F32 * 2048, torch.bfloat16)
    check(m, 64, 1024, torch.bfloat16, low=-128)


@pytest.mark.parametrize("m", [1, 9, 40, 64, 100, 300])
@pytest.mark.parametrize("n,k", [(36, 144), (516, 1040)])
def test_pitches_and_what_lies_between_rows(m, n, k):
    """Through the C entry points: rows of every operand apart, with other codes, NaN and values between and behind them that are not read or are left as they were."""
    dtype = torch.bfloat16
    x, sx, g, sg, u, su, bias, addend = operands(m, n, k, dtype)

    def apart(t, by, fill):
        wide = torch.full((t.shape[0] + 40, t.shape[1] + by), fill, dtype=t.dtype, device=DEV)
        wide[:t.shape[0], :t.shape[1]] = t
        return wide

    stream = ctypes.c_void_p(torch.cuda.current_stream(DEV).cuda_stream)
    for by_codes, by_values in ((16, 8), (112, 4), (1, 1)):  # (the last: rows off the boundaries)
        xw, gw, uw, aw = apart(x, by_codes, 127), apart(g, by_codes, 127), apart(u, by_codes, -128), apart(addend, by_values, float("nan"))
        sxw = torch.cat([sx, torch.full((40,), float("nan"), device=DEV)])
        y, c = apart(torch.zeros(m, n, dtype=dtype, device=DEV), by_values, 7.0), apart(torch.zeros(m, n, dtype=dtype, device=DEV), by_values, 7.0)
        ptr = [t.data_ptr() for t in (xw, sxw, gw, sg)]
        assert _native.lib().tpamd_linear_a8_add(*ptr, bias.data_ptr(), aw.data_ptr(), y.data_ptr(), c.data_ptr(), m, n, k, k + by_codes, k + by_codes, n + by_values, n + by_values, 0, 0,
                                                 stream) == 0
        want = _native.linear_a8(x, sx, g, sg, bias, dtype, addend=addend)
        for t in (y, c):
            assert torch.equal(t[:m, :n], want) and bool((t[m:] == 7).all() and (t[:, n:] == 7).all())
        h = apart(torch.zeros(m, n, dtype=dtype, device=DEV), by_values, 7.0)
        assert _native.lib().tpamd_swiglu_up_a8(*ptr, uw.data_ptr(), su.data_ptr(), h.data_ptr(), m, n, k, k + by_codes, k + by_codes, n + by_values, 0, stream) == 0
        assert torch.equal(h[:m, :n], _native.swiglu_up_a8(x, sx, g, sg, u, su, dtype)) and bool((h[m:] == 7).all() and (h[:, n:] == 7).all())
        # the sum in the place of the addend
        assert _native.lib().tpamd_linear_a8_add(*ptr, bias.data_ptr(), aw.data_ptr(), aw.data_ptr(), None, m, n, k, k + by_codes, k + by_codes, n + by_values, n + by_values, 0, 0, stream) == 0
        assert torch.equal(aw[:m, :n], want) and bool(aw[m:].isnan().all() and aw[:, n:].isnan().all())


def test_views_and_orders_of_python_tensors():
    x, sx, w, sw, u, su, bias, addend = operands(12, 96, 256, torch.float16)
    want, pair = _native.linear_a8(x, sx, w, sw, bias, torch.float16, addend=addend), _native.swiglu_up_a8(x, sx, w, sw, u, su, torch.float16)
    wide = torch.zeros(12, 300, dtype=torch.int8, device=DEV)
    for at in (0, 16, 1, 44):
        wide[:, at:at + 256] = x
        assert torch.equal(_native.linear_a8(wide[:, at:at + 256], sx, w, sw, bias, torch.float16, addend=addend), want)
        assert torch.equal(_native.swiglu_up_a8(wide[:, at:at + 256], sx, w, sw, u, su, torch.float16), pair)
    columns = x.t().contiguous().t()
    spaced = torch.stack([sw, sw], 1)[:, 0]
    assert torch.equal(_native.linear_a8(columns, sx, w.t().contiguous().t(), spaced, bias, torch.float16, addend=addend.t().contiguous().t()), want)
    both = torch.cat([w, u], 1)  # the weights of a pair in one matrix, side by side
    assert torch.equal(_native.swiglu_up_a8(x, sx, both[:, :256], sw, both[:, 256:], su, torch.float16), pair)
    assert torch.equal(_native.swiglu_up_a8(x, sx, both[:, :256], sw, u, su, torch.float16), pair)  # unlike pitches
    assert torch.equal(_native.linear_a8(x.reshape(3, 4, 256), sx.reshape(3, 4), w, sw, bias, torch.float16, addend=addend.reshape(3, 4, 96)), want.reshape(3, 4, 96))
    assert torch.equal(_native.linear_a8(x[:1].expand(12, 256), sx[:1].expand(12), w, sw, None, torch.float16), _native.linear_a8(x[:1], sx[:1], w, sw, None, torch.float16).expand(12, 96))


def test_nothing_to_do_and_nothing_to_sum():
    x, sx, w, sw, u, su, bias, addend = operands(4, 24, 32, torch.float16)
    assert _native.linear_a8(x[:0], sx[:0], w, sw, None, torch.float16).shape == (0, 24) and _native.linear_a8(x, sx, w[:0], sw[:0], None, torch.float16).shape == (4, 0)
    none = _native.linear_a8(x[:, :0], sx, w[:, :0], sw, bias, torch.float16, addend=addend)
    assert torch.equal(none, (bias.float() + addend.float()).to(torch.float16))
    assert bool((_native.swiglu_up_a8(x[:, :0], sx, w[:, :0], sw, u[:, :0], su, torch.float16) == 0).all())
    assert bool(_native.linear_a8(x, torch.full_like(sx, float("nan")), w, sw, None, torch.float16).isnan().all())


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (16, 4096, 2048), (100, 512, 4096), (300, 2048, 1024)])
def test_streams_graphs_and_gradients(m, n, k):
    dtype = torch.bfloat16
    x, sx, w, sw, u, su, bias, addend = operands(m, n, k, dtype)

    def calls(x, sx):
        return [_native.linear_a8(x, sx, w, sw, bias, dtype, addend=addend), _native.swiglu_up_a8(x, sx, w, sw, u, su, dtype)]

    want = calls(x, sx)
    side, other = torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream(DEV))
    got = []
    for _ in range(4):  # two streams at once
        for s in (side, other):
            with torch.cuda.stream(s):
                got.append(calls(x, sx))
    for s in (side, other):
        torch.cuda.current_stream(DEV).wait_stream(s)
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
    still, scales = x.clone(), sx.clone()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graphs.append((torch.cuda.CUDAGraph(), []))
        with torch.cuda.graph(graphs[-1][0]):
            graphs[-1][1].extend(calls(still, scales))
    for seed in (1, 2, 3):
        fresh, fresh_scale, *_ = operands(m, n, k, dtype, seed)
        still.copy_(fresh)
        scales.copy_(fresh_scale)
        eager = calls(fresh, fresh_scale)
        for graph, outs in graphs:
            graph.replay()
            eager_again = calls(fresh, fresh_scale)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(outs, eager, eager_again))
    rows = int8.QuantizedRows(x, sx, dtype)
    with pytest.raises(NotImplementedError):
        int8.linear(rows, w, sw, addend=addend.clone().requires_grad_()).sum().backward()


TILES = [64128, 128128, 128192, 192192, 192256, 256256]


@pytest.mark.parametrize("splits", [1, 3, 64])
@pytest.mark.parametrize("tile", TILES)
def test_every_tile(tile, splits, tune):
    """Tiles that reach over the ends of rows and columns, K that ends inside a stage (one piece of 16, seven of them, none), fewer K tiles than stages or ranges."""
    tune("TPAMD_A8_TILE", tile)
    tune("TPAMD_A8_SPLITS", splits)
    for m, n, k in [(1, 1, 16), (65, 50, 272), (130, 516, 384), (300, 1001, 1040), (515, 388, 2032), (256, 512, 4096)]:
        check(m, n, k, torch.float16 if k % 128 else torch.bfloat16, low=-128)


def test_a_tile_that_there_is_none_of(tune):
    tune("TPAMD_A8_TILE", 64064)
    x, sx, w, sw, *_ = operands(70, 64, 128, torch.float16)
    with pytest.raises(_native.Unsupported, match="tile"):
        _native.linear_a8(x, sx, w, sw, dtype=torch.float16)


@pytest.mark.parametrize("tile,splits", [(128128, 4), (256256, 2)])
def test_ranges_of_k_under_capture_and_without_scratch_memory(tile, splits, tune):
    """The ranges' sums lie in the stream's scratch buffer: a graph captured on a stream that has none takes the spare one, or all of K in a block; the same bits either way."""
    tune("TPAMD_A8_TILE", tile)
    x, sx, w, sw, u, su, *_ = operands(200, 640, 2048, torch.bfloat16)
    want = _native.linear_a8(x, sx, w, sw), _native.swiglu_up_a8(x, sx, w, sw, u, su)
    tune("TPAMD_A8_SPLITS", splits)
    graphs = []
    for _ in range(3):
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream(DEV)
        with torch.cuda.graph(graph, stream=stream):
            graphs.append((graph, (_native.linear_a8(x, sx, w, sw), _native.swiglu_up_a8(x, sx, w, sw, u, su)), stream))
    for _ in range(3):
        for graph, got, _ in graphs:
            graph.replay()
            assert torch.equal(_native.linear_a8(x, sx, w, sw), want[0])
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for *_, stream in graphs:
        _native.release_scratch(DEV, stream.cuda_stream)


def test_threads_on_streams_of_their_own(tune):
    """Four host threads, each with a stream, K in ranges and several tiles: each one's results are those of calls in turn."""
    import threading

    sizes = [(300, 512, 4096), (40, 1000, 2064), (130, 256, 8192), (700, 688, 1024)]
    work = [operands(m, n, k, torch.bfloat16, i) for i, (m, n, k) in enumerate(sizes)]
    tune("TPAMD_A8_SPLITS", 4)
    want = [(_native.linear_a8(x, sx, g, sg, bias, torch.bfloat16), _native.swiglu_up_a8(x, sx, g, sg, u, su, torch.bfloat16)) for x, sx, g, sg, u, su, bias, _ in work]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        x, sx, g, sg, u, su, bias, _ = work[i]
        stream = torch.cuda.Stream(DEV)
        with torch.cuda.stream(stream):
            for _ in range(20):
                one, pair = _native.linear_a8(x, sx, g, sg, bias, torch.bfloat16), _native.swiglu_up_a8(x, sx, g, sg, u, su, torch.bfloat16)
                if not (torch.equal(one, want[i][0]) and torch.equal(pair, want[i][1])):
                    wrong.append(i)
        stream.synchronize()
        _native.release_scratch(DEV, stream.cuda_stream)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
