"""Several ranks' rows in 8 bits and products of them in one launch (`tpamd_rows_q8_ranks`, `tpamd_linear_a8_ranks`, `tpamd_swiglu_up_a8_ranks`): bit for bit what each rank's own call gives."""
import ctypes

import pytest
import torch

import tensor_parallel_amd as tp
from tensor_parallel_amd import _native, together
from tensor_parallel_amd.int8 import quantize_linears_

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16]


def rank_operands(ranks, m, n, k, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def codes(rows):
        return torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g)

    def scales(rows):
        return torch.rand(rows, device=DEV, generator=g) * 0.01 + 0.001

    return [(codes(m), scales(m), codes(n), scales(n), codes(n), scales(n), torch.randn(n, device=DEV, generator=g).to(dtype)) for _ in range(ranks)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ranks", [1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(1, 2048, 512), (2, 16, 16), (8, 50, 272), (17, 5504, 1024), (33, 130, 2064), (64, 1000, 640), (65, 256, 512), (5, 24, 100), (3, 26000, 256), (0, 16, 32), (4, 7, 0)])
def test_products(dtype, ranks, m, n, k):
    operands = rank_operands(ranks, m, n, k, dtype)
    for act in (_native.ACT_NONE, _native.ACT_GELU):
        calls = [(x, sx, w, sw, bias, dtype, act) for x, sx, w, sw, _, _, bias in operands]
        for with_bias in (True, False):
            calls = [c if with_bias else (*c[:4], None, *c[5:]) for c in calls]
            for got, call in zip(_native.linear_a8_ranks(calls), calls):
                assert torch.equal(got, _native.linear_a8(*call))
    pairs = [(x, sx, w, sw, u, su, dtype) for x, sx, w, sw, u, su, _ in operands]
    for got, call in zip(_native.swiglu_up_a8_ranks(pairs), pairs):
        assert torch.equal(got, _native.swiglu_up_a8(*call))


def test_ranks_of_unlike_alignment_and_bias():
    """Operands that one launch does not take: a rank off 16-byte boundaries, a bias at one of them."""
    a, b = rank_operands(2, 9, 96, 256, torch.float16)
    off = torch.empty(96 * 256 + 1, dtype=torch.int8, device=DEV)[1:].view(96, 256)
    off.copy_(b[2])
    calls = [(a[0], a[1], a[2], a[3], a[6], torch.float16, 0), (b[0], b[1], off, b[3], None, torch.float16, 0)]
    for got, call in zip(_native.linear_a8_ranks(calls), calls):
        assert torch.equal(got, _native.linear_a8(*call))
    with pytest.raises(ValueError, match="different forms"):
        _native.linear_a8_ranks([calls[0], (b[0][:5], b[1][:5], *calls[1][2:])])
    with pytest.raises(ValueError, match="different forms"):
        _native.swiglu_up_a8_ranks([(*a[:6], torch.float16), (*b[:6], torch.bfloat16)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ranks", [1, 2, 3])
@pytest.mark.parametrize("rows,d", [(1, 4096), (2, 8), (5, 100), (7, 2056), (64, 688), (3, 16384), (2, 16392), (70, 1040), (2050, 4104), (0, 16), (2, 0)])
def test_rows(dtype, ranks, rows, d):
    g = torch.Generator(device=DEV).manual_seed(rows + d)
    xs, rs = ([torch.randn(rows, d, device=DEV, generator=g).to(dtype) for _ in range(ranks)] for _ in range(2))
    ws = [(1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(dtype) for _ in range(ranks)]
    for got, x in zip(_native.quantize_rows_ranks([(x,) for x in xs]), xs):
        assert all(torch.equal(a, b) for a, b in zip(got, _native.quantize_rows(x)))
    for got, x, w in zip(_native.rms_norm_q8_ranks([(x, w, 1e-5) for x, w in zip(xs, ws)]), xs, ws):
        assert all(torch.equal(a, b) for a, b in zip(got, _native.rms_norm_q8(x, w, 1e-5)))
    for got, r, x, w in zip(_native.add_rms_norm_q8_ranks([(r, x, w, 1e-5) for r, x, w in zip(rs, xs, ws)]), rs, xs, ws):
        assert all(torch.equal(a, b) for a, b in zip(got, _native.add_rms_norm_q8(r, x, w, 1e-5)))
    if ranks > 1 and rows:
        with pytest.raises(ValueError, match="different forms"):
            _native.quantize_rows_ranks([(xs[0],), (xs[1][:rows - 1],)])


def test_refusals_of_the_library():
    """Before anything is launched: nothing is read or written, so the addresses need not be any."""
    lib = _native.lib()
    rank = (_native.A8Rank * 2)()
    assert lib.tpamd_linear_a8_ranks(1, rank, 4, 16, 16, 16, 16, 16, _native.BF16, 0, None) == -1
    assert lib.tpamd_linear_a8_ranks(2, None, 4, 16, 16, 16, 16, 16, _native.BF16, 0, None) == -1
    assert lib.tpamd_linear_a8_ranks(1, rank, 4, 16, 131072, 131072, 131072, 16, _native.BF16, 0, None) == -2
    assert lib.tpamd_swiglu_up_a8_ranks(1, rank, 4, 16, 16, 16, 16, 16, 7, None) == -1
    assert lib.tpamd_linear_a8_ranks(0, None, 4, 16, 16, 16, 16, 16, _native.BF16, 0, None) == 0
    rows = (_native.Q8Rank * 2)()
    rows[1].w = 64
    assert lib.tpamd_rows_q8_ranks(2, rows, 4, 16, 16, 16, 16, 16, ctypes.c_float(1e-5), _native.BF16, None) == -1
    rows[1].w, rows[0].r, rows[1].r = None, 64, 64
    assert lib.tpamd_rows_q8_ranks(2, rows, 4, 16, 16, 16, 16, 16, ctypes.c_float(1e-5), _native.BF16, None) == -1
    assert lib.tpamd_rows_q8_ranks(1, rows, 4, 16, 16, 16, 16, 16, ctypes.c_float(1e-5), _native.F32, None) == -1


@pytest.mark.parametrize("rows", [3, 40])
def test_ranks_that_meet_give_what_they_give_alone(rows, monkeypatch):
    """Two rank shards of a Llama on a static cache, recorded and replayed too, with and without meeting."""
    from transformers import LlamaConfig, LlamaForCausalLM, StaticCache

    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=300, hidden_size=512, intermediate_size=1376, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, max_position_embeddings=128,
                         attn_implementation="sdpa")
    split = tp.tensor_parallel(LlamaForCausalLM(config).to(torch.bfloat16).eval(), [DEV, DEV])
    tp.attention.fuse_rotary_(split, assume_no_padding=True)
    quantize_linears_(split, skip=lambda name, m: "lm_head" in name, activations=True)
    ids = torch.randint(2, 300, (rows, 12), device=DEV)

    def run(record):
        cache = StaticCache(config=config, max_cache_len=16)
        outs = [split(input_ids=ids[:, :8], past_key_values=cache, use_cache=True).logits, split(input_ids=ids[:, 8:9], past_key_values=cache, use_cache=True).logits]
        step = tp.graphs.capture(split, input_ids=ids[:, 9:10].clone(), past_key_values=cache, use_cache=True) if record else split
        for at in range(9, 12):
            outs.append(step(input_ids=ids[:, at:at + 1], past_key_values=cache, use_cache=True).logits.clone())
            torch.cuda.synchronize()
        return outs

    with torch.no_grad():
        run(False)
        eager, replayed = run(False), run(True)
        monkeypatch.setattr(together, "MEET", False)
        alone = run(False)
    for a, b, c in zip(eager, replayed, alone):
        # (codes and sums are the same; attention, head and additions are other launches)
        for other in (b, c):
            torch.testing.assert_close(other.float(), a.float(), rtol=2e-2, atol=2e-2 * a.float().std().item())
