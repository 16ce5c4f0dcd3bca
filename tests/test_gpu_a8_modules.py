"""Linears of 8-bit rows as modules: `ShardLinearA8` and a run of the operators against their definition in 64 bits, a tensor-parallel Llama and a Falcon whose Linears were replaced by
`quantize_linears_(..., activations=True)`, and which of their forwards take rows from the norms' launches."""
import copy
import pickle

import pytest
import torch
from torch import nn

import tensor_parallel_amd as tp
from tensor_parallel_amd import _native, int8, shard_modules
from tensor_parallel_amd.int8 import QuantizedRows, ShardLinearA8, quantize_linears_, quantize_rows

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16]


def codes64(x):
    """The rows' values in 64 bits as their codes stand for them, by the definition."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    return torch.where(a > 0, (127 * x / a.clamp_min(1e-300)).round(), 0.0) * torch.where(a > 0, a / 127, 1.0)


def weights64(w):
    wq, scale, *_ = quantize_rows(w)
    return wq.double() * scale.double()[:, None]


def step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,bias", [(1, 64, 256, False), (7, 96, 500, True), (40, 256, 1024, True), (150, 130, 1040, False)])
def test_module_matches_the_definition(dtype, M, N, K, bias):
    torch.manual_seed(M)
    lin = nn.Linear(K, N, bias=bias).to(DEV, dtype)
    x = torch.randn(2, M, K, device=DEV).to(dtype)
    mod = ShardLinearA8.from_weight(lin.weight, lin.bias)
    want = codes64(x) @ weights64(lin.weight.detach()).t().contiguous() + (lin.bias.double() if bias else 0)
    got = mod(x)
    # exact codes and sums; scales, products and the bias in fp32 (2^-21 of what they round), and half a step of the result
    size = want.abs() + (lin.bias.double().abs() if bias else 0)
    assert got.dtype is dtype and bool(((got.double() - want).abs() <= 2.0**-21 * size + step(dtype) * want.abs() * 1.001 + 2.0**-25).all())
    assert torch.equal(mod(int8.quantize_activations(x)), got)
    with pytest.raises(TypeError, match="quantised for"):
        mod(x.float())
    with pytest.raises(NotImplementedError):
        mod(x.clone().requires_grad_()).sum().backward()


def test_rows_in_lines():
    """Rows of a multiple of 16 codes that is none of 128 begin on 128-byte boundaries, in modules and in the codes of many rows; what stands between them is nowhere in results or saved weights."""
    torch.manual_seed(3)
    weight, x = torch.randn(130, 1376, device=DEV).bfloat16(), torch.randn(3, 50, 1376, device=DEV).bfloat16()
    mod = ShardLinearA8.from_weight(weight)
    assert mod.wq.shape == (130, 1376) and mod.wq.stride() == (1408, 1) and mod.wq.data_ptr() % 128 == 0
    rows, few = int8.quantize_activations(x), int8.quantize_activations(x[0])
    assert rows.codes.shape == x.shape and rows.codes.stride() == (50 * 1408, 1408, 1) and few.codes.is_contiguous()
    want = mod(x)
    wq, scale, *_ = quantize_rows(weight)
    assert torch.equal(want, int8.linear(QuantizedRows(rows.codes.contiguous(), rows.scale, x.dtype), wq, scale))
    assert torch.equal(want[0], mod(few)) and torch.equal(rows.dequantize()[0], few.dequantize())
    saved = mod.state_dict()
    assert torch.equal(saved["wq"], wq) and all(t.is_contiguous() for t in saved.values())
    for other in (copy.deepcopy(mod), pickle.loads(pickle.dumps(mod))):
        assert other.wq.stride() == (1408, 1) and torch.equal(other(x), want)
    other = ShardLinearA8.from_weight(torch.randn_like(weight))
    other.load_state_dict(saved)
    assert other.wq.stride() == (1408, 1) and torch.equal(other(x), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 19, 70, 300])
def test_a_run_of_the_operators(dtype, M):
    """Residual and norm, gate and up, hidden rows, down with another rank's part: the second half of a decoder layer, each step against its definition on what the step before gave."""
    g = torch.Generator(device=DEV).manual_seed(M)
    d, ffn = 512, 688
    r, x, other = (torch.randn(M, d, device=DEV, generator=g).to(dtype) for _ in range(3))
    w = (1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(dtype)
    gate, up, down = (torch.randn(n, k, device=DEV, generator=g).to(dtype) * 0.05 for n, k in ((ffn, d), (ffn, d), (d, ffn)))
    (gq, gs), (uq, us), (dq, ds) = (quantize_rows(t)[:2] for t in (gate, up, down))
    total, rows = int8.add_rms_norm(r, x, w, 1e-5)
    assert torch.equal(total, (r.float() + x.float()).to(dtype))
    t = total.double()
    assert bool(((rows.dequantize(torch.float32).double() - codes64(t * w.double()) * (t.square().mean(1, keepdim=True) + 1e-5).rsqrt()).abs()
                 <= 2.0**-19 * rows.scale.double()[:, None] * 127).all())
    h = int8.swiglu_up(rows, gq, gs, uq, us)
    values = rows.codes.double() * rows.scale.double()[:, None]
    a, b = values @ weights64(gate).t().contiguous(), values @ weights64(up).t().contiguous()
    want = torch.nn.functional.silu(a) * b
    assert bool(((h.double() - want).abs() <= step(dtype) * want.abs() * 1.01 + 2.0**-21 * (2 + a.abs()) * (want.abs() + (a * b).abs() / 4) + 2.0**-25).all())
    hidden = int8.quantize_activations(h)
    out = int8.linear(hidden, dq, ds, addend=other)
    part = codes64(h) @ weights64(down).t().contiguous()
    want = part + other.double()
    assert bool(((out.double() - want).abs() <= 1.01 * step(dtype) * (part.abs() + want.abs()) + 2.0**-20 * part.abs() + 2.0**-24).all())


def _llama(attention="eager"):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=300, hidden_size=512, intermediate_size=768, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, max_position_embeddings=256,
                         attn_implementation="eager" if attention == "tpamd" else attention)
    model = LlamaForCausalLM(config).to(torch.bfloat16).eval()
    if attention == "tpamd":
        model.config._attn_implementation = tp.attention.register()
    return model


def not_the_head(name, module):
    return "lm_head" in name


def near(got, want):
    """The quantisation of eight Linears' weights and rows a layer, each about 1 % of a result (half a step of 127 to a largest value of 3.5 deviations) and the
    half of them in a row: 4 % of the logits' spread, and 4.5 deviations of that among some ten thousand."""
    off = got.float() - want.float()
    assert off.square().mean().sqrt() < 0.06 * want.float().std() and off.abs().max() < 0.3 * want.float().std()


def test_tensor_parallel_llama():
    model = _llama()
    ids = torch.randint(0, 300, (2, 24), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        tp_model = tp.tensor_parallel(model, [DEV, DEV])
        before = tp_model(input_ids=ids).logits
        with pytest.raises(ValueError, match="outlier"):
            quantize_linears_(tp_model, outlier_cols={}, activations=True)
        n = quantize_linears_(tp_model, skip=not_the_head, activations=True)
        assert n == 2 * 2 * 7 and sum(isinstance(m, ShardLinearA8) for m in tp_model.modules()) == n
        first, after, again = (tp_model(input_ids=ids).logits for _ in range(3))
        mlps = [m for m in tp_model.modules() if m._modules.get("down_proj") is not None]
        assert len(mlps) == 4 and all(m.forward.__func__ is shard_modules._gated_mlp_a8_forward for m in mlps)
    near(first, before)
    near(after, before)
    assert torch.equal(after, again)
    with pytest.raises(RuntimeError, match="int8"):
        with tp.save_tensor_parallel(tp_model):
            tp_model.state_dict()
    assert any(k.endswith(".wq") for k in tp_model.state_dict())


@pytest.mark.parametrize("ranks", [1, 2])
@pytest.mark.parametrize("static", [False, True])
def test_norms_hand_rows_to_attention_and_mlp(ranks, static, monkeypatch):
    """On a cache, with the fused attention: both norms of a layer in 8 bits, no other launch that quantises their rows; a hook on a norm or on the block behind it puts the 16-bit norm back."""
    from transformers import DynamicCache, StaticCache

    model = _llama("eager" if static else "tpamd")  # (the second gives attention modules no mask on a growing cache)
    split = tp.tensor_parallel(model, [DEV] * ranks) if ranks > 1 else model.to(DEV)
    if ranks == 1:
        shard_modules.install_shard_kernels(split)
    assert tp.attention.fuse_rotary_(split, assume_no_padding=static) == 2 * ranks
    quantize_linears_(split, skip=not_the_head, activations=True)
    ids = torch.randint(2, 300, (2, 40), device=DEV)

    def forward():
        cache = StaticCache(config=model.config, max_cache_len=64) if static else DynamicCache()
        return [split(input_ids=part, past_key_values=cache, use_cache=True).logits for part in (ids[:, :39], ids[:, 39:])]

    counts = {}
    for name in ("rms_norm_q8", "add_rms_norm_q8", "quantize_rows", "rms_norm", "rms_norm_ranks", "add_rms_norm", "add_rms_norm_ranks", "swiglu_up_a8"):
        inner = getattr(_native, name)
        monkeypatch.setattr(_native, name, lambda *a, _f=inner, _n=name, **k: counts.update({_n: counts.get(_n, 0) + 1}) or _f(*a, **k))
    for name in ("rms_norm_q8", "add_rms_norm_q8", "quantize_rows", "swiglu_up_a8"):  # two ranks' calls in one
        inner = getattr(_native, name + "_ranks")
        monkeypatch.setattr(_native, name + "_ranks", lambda calls, _f=inner, _n=name: counts.update({_n: counts.get(_n, 0) + len(calls), "met": counts.get("met", 0) + 1}) or _f(calls))
    with torch.no_grad():
        forward()
        counts.clear()
        want = forward()
        layers = 2 * ranks * 2  # over both calls
        assert counts["rms_norm_q8"] == counts["add_rms_norm_q8"] == counts["swiglu_up_a8"] == layers
        assert counts["quantize_rows"] == 2 * layers  # the attention's output and the hidden rows
        assert counts.get("met", 0) == (5 * 2 if ranks == 2 else 0)  # all of them in the step of one position, of each of the two layers
        seen = []
        handles = []
        for m in split.modules():
            if m._modules.get("post_attention_layernorm") is not None:
                handles.append(m.post_attention_layernorm.register_forward_hook(lambda mod, args, out: seen.append(out.dtype)))
                inner = m._modules["self_attn"]._modules.get("tp_wrapped_module", m._modules["self_attn"])
                handles.append(inner.register_forward_pre_hook(lambda mod, args, kwargs: seen.append(kwargs["hidden_states"].dtype), with_kwargs=True))
        counts.clear()
        got = forward()
        assert counts.get("rms_norm_q8", 0) == counts.get("add_rms_norm_q8", 0) == 0 and len(seen) == 2 * layers
        for h in handles:
            h.remove()
        again = forward()
    for a, b, c in zip(want, got, again):
        near(b, a)  # (norms rounded to 16 bits in between)
        assert torch.equal(a, c)


def test_recorded_decode_step():
    """A step on a static cache recorded as a HIP graph and replayed over new tokens, against eager steps."""
    from transformers import StaticCache

    model = _llama("sdpa")
    split = tp.tensor_parallel(model, [DEV, DEV])
    tp.attention.fuse_rotary_(split, assume_no_padding=True)
    quantize_linears_(split, skip=not_the_head, activations=True)
    ids = torch.randint(2, 300, (3, 30), device=DEV)
    with torch.no_grad():
        split(input_ids=ids)  # (a block's first call returns what its own forward gives, which rounds in between: a cache filled by it holds other values)
        caches = [StaticCache(config=model.config, max_cache_len=64) for _ in range(2)]
        for cache in caches:
            split(input_ids=ids[:, :20], past_key_values=cache, use_cache=True)
            split(input_ids=ids[:, 20:21], past_key_values=cache, use_cache=True)
        step = tp.graphs.capture(split, input_ids=ids[:, 21:22].clone(), past_key_values=caches[0], use_cache=True)
        for at in range(21, 30):
            eager = split(input_ids=ids[:, at:at + 1], past_key_values=caches[1], use_cache=True).logits.float()
            torch.cuda.synchronize()
            got = step(input_ids=ids[:, at:at + 1], past_key_values=caches[0], use_cache=True).logits.float()
            # (codes and their sums are the same; the head's and the attention's sums may be taken in another order)
            torch.testing.assert_close(got, eager, rtol=2e-2, atol=2e-2 * eager.std().item())


@pytest.mark.parametrize("M", [3, 70])
def test_falcon_mlp(M):
    from transformers import FalconConfig
    from transformers.models.falcon.modeling_falcon import FalconMLP

    torch.manual_seed(M)
    mlp = FalconMLP(FalconConfig(hidden_size=256, bias=False)).to(DEV, torch.float16)
    weight, second = mlp.dense_h_to_4h.weight.detach().clone(), mlp.dense_4h_to_h.weight.detach().clone()
    shard_modules.install_shard_kernels(mlp)
    assert quantize_linears_(mlp, activations=True) == 2
    x = torch.randn(M, 256, device=DEV).half()
    with torch.no_grad():
        got = mlp(x)
    h = torch.nn.functional.gelu(codes64(x) @ weights64(weight).t().contiguous()).half()
    want = codes64(h) @ weights64(second).t().contiguous()
    # the hidden rows may be rounded one step of fp16 apart, and their codes then one of 127 in a few places: a percent of the result's spread
    assert (got.double() - want).abs().max() < 0.02 * want.std() + 2 * step(torch.float16) * want.abs().max()


def test_layers_that_stay():
    """A Linear that is skipped keeps its block's own forward; a block whose forward is not the gated pattern keeps that too."""
    class Odd(nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj, self.down_proj, self.act_fn = nn.Linear(64, 96, bias=False), nn.Linear(64, 96, bias=False), nn.Linear(96, 64, bias=False), nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))  # the other way round

    torch.manual_seed(0)
    odd = Odd().to(DEV, torch.bfloat16)
    x = torch.randn(5, 64, device=DEV).bfloat16()
    with torch.no_grad():
        want = odd(x)
        assert quantize_linears_(odd, activations=True) == 3
        outs = [odd(x) for _ in range(2)]
    assert "forward" not in odd.__dict__ and torch.equal(*outs)
    near(outs[0], want)
    with pytest.raises(ValueError, match="32 bits"):
        ShardLinearA8.from_weight(torch.zeros(4, 131072, dtype=torch.float16, device=DEV))
    rows = QuantizedRows(torch.zeros(2, 3, 8, dtype=torch.int8, device=DEV), torch.ones(2, 3, device=DEV), torch.float16)
    assert rows.shape == (2, 3, 8) and rows.dim() == 3 and rows.device == DEV


def test_a_fused_block_whose_parts_change():
    """Once gate and up are one launch: a hook on one of them is told again, a Linear put in its place is called, and the launch comes back when both are as they were."""
    class Mlp(nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj, self.down_proj, self.act_fn = nn.Linear(64, 96, bias=False), nn.Linear(64, 96, bias=False), nn.Linear(96, 64, bias=False), nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))

    torch.manual_seed(0)
    mlp = Mlp().to(DEV, torch.bfloat16)
    x = torch.randn(5, 64, device=DEV).bfloat16()
    with torch.no_grad():
        quantize_linears_(mlp, activations=True)
        mlp(x)
        assert mlp.forward.__func__ is shard_modules._gated_mlp_a8_forward
        want, told = mlp(x), []
        handle = mlp.up_proj.register_forward_hook(lambda mod, args, out: told.append(out.shape))
        near(mlp(x), want)
        assert told == [(5, 96)]
        near(mlp(int8.quantize_activations(x)), want)
        handle.remove()
        kept, mlp.gate_proj = mlp.gate_proj, nn.Linear(64, 96, bias=False).to(DEV, torch.bfloat16)
        nn.init.zeros_(mlp.gate_proj.weight)
        assert bool((mlp(x) == 0).all())
        mlp.gate_proj = kept
        assert torch.equal(mlp(x), want)


@pytest.mark.parametrize("bias", [False, True])
def test_one_launch_for_q_k_and_v(bias, monkeypatch):
    """Their codes and scales are views of one matrix, which a fused attention multiplies at once; where one of them is something else since, they are three launches again."""
    from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=300, hidden_size=528, intermediate_size=768, num_hidden_layers=1, num_attention_heads=6, num_key_value_heads=2, head_dim=64, max_position_embeddings=256,
                         attention_bias=bias)
    model = LlamaForCausalLM(config).to(DEV, torch.bfloat16).eval()
    model.config._attn_implementation = tp.attention.register()
    shard_modules.install_shard_kernels(model)
    tp.attention.fuse_rotary_(model)
    attn = model.model.layers[0].self_attn
    if bias:
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            nn.init.normal_(attn._modules[name].bias)
    weights = {name: attn._modules[name].weight.detach().clone() for name in ("q_proj", "k_proj", "v_proj")}
    quantize_linears_(model, skip=not_the_head, activations=True)
    whole = attn.__dict__["_tp_qkv8"]
    assert whole[0].shape == (6 * 64 + 4 * 64, 528) and whole[0].stride() == (640, 1)
    for name, w in weights.items():
        wq, scale, *_ = quantize_rows(w)
        part = attn._modules[name]
        assert torch.equal(part.wq, wq) and torch.equal(part.scale, scale) and part.wq.untyped_storage().data_ptr() == whole[0].untyped_storage().data_ptr()
        assert all(t.is_contiguous() for t in part.state_dict().values())
    ids = torch.randint(2, 300, (2, 40), device=DEV)
    launches = []
    inner = _native.linear_a8
    monkeypatch.setattr(_native, "linear_a8", lambda *a, **k: launches.append(a[2].shape[0]) or inner(*a, **k))  # q, k, v (q_proj has 384 rows, the others 128), o_proj, down_proj

    def forward():
        cache, outs = DynamicCache(), []
        for part in (ids[:, :39], ids[:, 39:]):
            launches.clear()
            outs.append(model(input_ids=part, past_key_values=cache, use_cache=True).logits)
        return outs

    with torch.no_grad():
        forward()
        want = forward()
        assert launches == [640, 528, 528]
        told = []
        handle = attn.k_proj.register_forward_hook(lambda mod, args, out: told.append(out.shape[-1]))
        watched = forward()
        assert launches.count(128) == 2 and told == [128, 128]
        handle.remove()
        forward()
        assert launches == [640, 528, 528]
        copied = copy.deepcopy(model)
        attn.v_proj.scale = attn.v_proj.scale.clone()
        apart = forward()
        assert launches == [384, 128, 128, 528, 528] and "_tp_qkv8" not in attn.__dict__
        launches.clear()
        cache = DynamicCache()
        again = [copied(input_ids=part, past_key_values=cache, use_cache=True).logits for part in (ids[:, :39], ids[:, 39:])]
    # the same codes, scales and sums; the head and the attention are the same launches
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, apart, again))
    for a, b in zip(want, watched):
        near(b, a)
