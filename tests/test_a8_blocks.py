"""Gated MLPs and projections of 8-bit rows as modules: which calls their fused forwards make for the block's own and which they leave to it. The library's calls are stood in for by their definitions on
host tensors, so no GPU is needed."""
import copy
import types
import weakref

import pytest
import torch
from torch import nn

from tensor_parallel_amd import _native, attention, int8, shard_modules, together
from tensor_parallel_amd.collectives import SumContext
from tensor_parallel_amd.int8 import ShardLinearA8, quantize_linears_


def rows64(p):
    """(codes, scale) of the rows of p, by the definition."""
    p = p.double()
    a = p.abs().amax(-1)
    empty = a < 2.0**-100
    codes = torch.where(empty[..., None], 0.0, (127 * p / torch.where(empty, 1.0, a)[..., None]).round())
    return codes.to(torch.int8), torch.where(empty, 1.0, a / 127).float()


@pytest.fixture
def calls(monkeypatch):
    """The names of the library's calls that are made, which the definitions answer."""
    made = []

    def product(q, scale, wq, wscale):
        return (q.double() @ wq.double().t()) * scale.double()[..., None] * wscale.double()

    def quantize(x):
        made.append("quantize_rows")
        return rows64(x)

    def linear(q, scale, wq, wscale, bias=None, dtype=torch.bfloat16, act=0, addend=None, copy=None):
        made.append("linear_a8")
        y = product(q, scale, wq, wscale)
        return (y if bias is None else y + bias.double()).to(dtype)

    def pair(q, scale, gate, gscale, up, uscale, dtype=torch.bfloat16):
        made.append("swiglu_up_a8")
        return (nn.functional.silu(product(q, scale, gate, gscale)) * product(q, scale, up, uscale)).to(dtype)

    for name, call in (("quantize_rows", quantize), ("linear_a8", linear), ("swiglu_up_a8", pair), ("dequantize_rows", lambda q, s, dtype: (q.double() * s.double()[..., None]).to(dtype))):
        monkeypatch.setattr(_native, name, call)
    return made


class Mlp(nn.Module):
    def __init__(self, act=None):
        super().__init__()
        torch.manual_seed(0)
        for name, shape in (("gate_proj", (96, 64)), ("up_proj", (96, 64)), ("down_proj", (64, 96))):
            setattr(self, name, a8(*shape))
        self.act_fn = nn.SiLU() if act is None else act

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


def a8(n, k, bias=False):
    return ShardLinearA8(*rows64(torch.randn(n, k).bfloat16() * k**-0.5), torch.randn(n).bfloat16() if bias else None, torch.bfloat16)


def fused(block, x):
    """The block as its users have it: armed by quantize_linears_, and called."""
    quantize_linears_(block, activations=True)
    with torch.no_grad():
        block(x)
    assert block.forward.__func__ is shard_modules._gated_mlp_a8_forward
    return block


def inputs(rows=5):
    return torch.randn(rows, 64, generator=torch.Generator().manual_seed(1)).bfloat16()


@pytest.mark.parametrize("change", [
    lambda m: setattr(m, "gate_proj", a8(96, 64, bias=True)),
    lambda m: setattr(m, "up_proj", a8(96, 64, bias=True)),
    lambda m: setattr(m.gate_proj, "bias", torch.randn(96).bfloat16()),
    lambda m: setattr(m.gate_proj, "bias", nn.Parameter(torch.randn(96).bfloat16())),
    lambda m: setattr(m, "act_fn", nn.ReLU()),
    lambda m: setattr(m, "act_fn", nn.GELU()),
    lambda m: setattr(m.act_fn, "forward", torch.tanh),
    lambda m: m.act_fn.register_forward_hook(lambda mod, args, out: 2 * out),
], ids=["gate with a bias", "up with a bias", "a bias assigned", "a bias to be learned", "ReLU", "GELU", "a forward of the SiLU's own", "a hook on the SiLU"])
def test_a_part_that_is_something_else_since(calls, change):
    """What stands in gate's, up's or the activation's place is what the block computes with, whether a Linear or the layer around hands the input over."""
    x, block = inputs(), fused(Mlp(), inputs())
    change(block)
    assert not shard_modules.takes_rows(block)
    calls.clear()
    with torch.no_grad():
        got, want = block(x), type(block).forward(block, x)
    assert "swiglu_up_a8" not in calls and torch.equal(got, want)


def test_the_launch_comes_back(calls):
    x, block = inputs(), fused(Mlp(), inputs())
    with torch.no_grad():
        want = block(x)
        block.act_fn = nn.ReLU()
        assert not torch.equal(block(x), want)
        block.act_fn = nn.SiLU()
        calls.clear()
        assert torch.equal(block(x), want) and calls == ["quantize_rows", "swiglu_up_a8", "quantize_rows", "linear_a8"] and shard_modules.takes_rows(block)
        assert torch.equal(block(int8.quantize_activations(x)), want)


def test_who_is_said_to_return_the_down_projections_output(calls):
    """A Linear may hold other ranks' parts of a sum where the wrapped block is known to return its output as it is: the fused forward does, of the block's own forward nobody knows."""
    x, block = inputs(), fused(Mlp(), inputs())
    known = []
    for act in (nn.SiLU(), nn.Tanh()):
        block.act_fn = act
        ctx = SumContext(None, 0, nn.Module(), block)
        together.push_sum_context(ctx)
        try:
            with torch.inference_mode():
                block(x)
        finally:
            together.pop_sum_context()
        known.append(shard_modules.hands_through(ctx, block.down_proj))
    assert known == [True, False]


def test_every_call_gives_the_same(calls):
    """A block's first call as well, whose gate and up would be rounded to 16 bits by its own forward."""
    block, x = Mlp(), inputs(40)
    with torch.no_grad():
        own = block(x)
        quantize_linears_(block, activations=True)
        first, second = block(x), block(x)
    assert torch.equal(first, second) and not torch.equal(first, own)


class Exchanged(Mlp):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class Scaled(Mlp):
    def forward(self, x):
        return 1.02 * self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Shifted(Mlp):
    def forward(self, x):
        out = self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))
        out += 0.01
        return out


class Residual(Mlp):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)) + 0.01 * x


class OneOfTwo(Mlp):
    def forward(self, x):
        if x.shape[0] > 7:
            return self.up_proj(x)[:, :64]
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Squared(Mlp):
    def forward(self, x):
        g = self.act_fn(self.gate_proj(x))
        return self.down_proj(g * g)


class WithASetting(Mlp):
    def forward(self, x, scale=None):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


@pytest.mark.parametrize("cls", [Exchanged, Scaled, Shifted, Residual, OneOfTwo, Squared, WithASetting])
@pytest.mark.parametrize("first", ["zeros", "values"])
def test_blocks_of_another_formula(calls, cls, first):
    """They keep their own forward, whatever they are called with first."""
    block = cls()
    quantize_linears_(block, activations=True)
    with torch.no_grad():
        block(torch.zeros(5, 64).bfloat16() if first == "zeros" else inputs())
        calls.clear()
        for x in (inputs(), inputs(9)):
            assert torch.equal(block(x), cls.forward(block, x))
    assert "swiglu_up_a8" not in calls and not shard_modules.takes_rows(block)


class InSteps(Mlp):
    def forward(self, hidden):
        """The same formula."""
        up = self.up_proj(hidden)
        up *= self.act_fn(self.gate_proj(hidden))
        down = self.down_proj(up)
        return down


@pytest.mark.parametrize("cls", [Mlp, InSteps])
def test_blocks_of_this_formula(calls, cls):
    block = cls()
    quantize_linears_(block, activations=True)
    with torch.no_grad():
        assert not block(torch.zeros(5, 64).bfloat16()).any()
        assert calls == ["quantize_rows", "swiglu_up_a8", "quantize_rows", "linear_a8"]


def test_a_class_that_is_given_another_forward(calls):
    class Own(Mlp):
        forward = Mlp.forward

    block, x = fused(Own(), inputs()), inputs()
    Own.forward = Scaled.forward
    with torch.no_grad():
        assert torch.equal(block(x), Scaled.forward(block, x)) and not shard_modules.takes_rows(block)


def test_a_forward_that_keeps_something_is_not_called_ahead(calls):
    """quantize_linears_ calls no forward of a program's that could tell."""
    seen = []

    class Counting(Mlp):
        def forward(self, x):
            seen.append(type(x))
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))

    block = Counting()
    quantize_linears_(block, activations=True)
    with torch.no_grad():
        block(inputs())
    assert seen == [torch.Tensor]


def projections(whole, bias=False):
    attn = nn.Module()
    for i, name in enumerate(attention.QKV):
        setattr(attn, name, ShardLinearA8(*rows64(whole[64 * i:64 * i + 64]), torch.randn(64).bfloat16() if bias else None, torch.bfloat16))
    return attn


def test_linears_of_8_bits_put_in_one_by_one_end_the_16_bit_sharing(calls):
    """The matrix of 16-bit weights that fuse_rotary_ has laid out is given back once all three projections are of 8-bit rows."""
    whole = torch.randn(3 * 64, 64).bfloat16()
    attn = projections(whole)
    attn.__dict__["_tp_qkv"] = (whole, None)
    assert attention.share_qkv_a8(attn)
    x = inputs()[None]
    with torch.no_grad():
        got = attention._project_qkv(attn, x, 32)
    assert all(torch.equal(part.flatten(2), attn._modules[name](x)) for part, name in zip(got, attention.QKV))
    assert "_tp_qkv" not in attn.__dict__


def test_two_calls_that_find_the_sharing_ended(calls):
    """The second of two threads finds that the first has ended it already."""
    attn = projections(torch.randn(3 * 64, 64).bfloat16())
    attention.share_qkv_a8(attn)

    class Ended(list):
        def __iter__(self):
            attn.__dict__.pop("_tp_qkv8", None)
            return super().__iter__()

    attn.__dict__["_tp_qkv8"] = Ended(attn.__dict__["_tp_qkv8"])
    attn.v_proj.scale = attn.v_proj.scale.clone()
    x = inputs()[None]
    with torch.no_grad():
        got = attention._project_qkv(attn, x, 32)
        assert all(torch.equal(part.flatten(2), attn._modules[name](x)) for part, name in zip(got, attention.QKV))


def test_codes_stay_where_they_are_when_other_linears_are_quantised(calls):
    """A graph that was recorded before may read them."""
    model = nn.ModuleList([projections(torch.randn(3 * 64, 64).bfloat16())])
    assert attention.share_qkv_a8(model[0])
    at = [model[0]._modules[name].wq.data_ptr() for name in attention.QKV]
    quantize_linears_(model, activations=True)
    assert at == [model[0]._modules[name].wq.data_ptr() for name in attention.QKV]


def test_hooks_on_all_modules_are_told_of_every_linear(calls):
    x, block, attn = inputs(), fused(Mlp(), inputs()), projections(torch.randn(3 * 64, 64).bfloat16())
    attention.share_qkv_a8(attn)
    told = []
    for register in (nn.modules.module.register_module_forward_hook, nn.modules.module.register_module_forward_pre_hook):
        told.clear()
        handle = register(lambda mod, *rest: told.append(mod))
        try:
            with torch.no_grad():
                block(x)
                attention._project_qkv(attn, x[None], 32)
            assert not shard_modules.takes_rows(block)
        finally:
            handle.remove()
        assert {m for m in told if type(m) is ShardLinearA8} == {block.gate_proj, block.up_proj, block.down_proj, attn.q_proj, attn.k_proj, attn.v_proj}
    calls.clear()
    with torch.no_grad():
        block(x)
        attention._project_qkv(attn, x[None], 32)
    assert calls == ["quantize_rows", "swiglu_up_a8", "quantize_rows", "linear_a8", "quantize_rows", "linear_a8"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_model_that_is_told_its_dtype(calls, dtype):
    """Scales stay in 32 bits and the bias in what the Linear was quantised for: the other dtype is refused with the input, as before."""
    model = nn.ModuleList([a8(96, 64, bias=True), nn.Linear(4, 4)])
    with torch.no_grad():
        want = model[0](inputs())
        model.to(dtype)
        assert model[1].weight.dtype is dtype and model[0].scale.dtype is torch.float32 and model[0].bias.dtype is torch.bfloat16
        assert torch.equal(model[0](inputs()), want)
        if dtype is not torch.bfloat16:
            with pytest.raises(TypeError, match="quantised for"):
                model[0](inputs().to(dtype))


def moved(module):
    """The module after a move to another device and back: as torch copies a view, without the bytes between its rows."""
    return module._apply(lambda t: t.clone(memory_format=torch.contiguous_format))


@pytest.mark.parametrize("change", [moved, lambda m: m.load_state_dict(m.state_dict(), assign=True)], ids=["moved", "assigned"])
def test_rows_in_lines_again(calls, change):
    mod, whole = a8(96, 80), a8(96, 256)
    x = torch.randn(5, 80, generator=torch.Generator().manual_seed(1)).bfloat16()
    with torch.no_grad():
        want = mod(x)
        for m in (mod, whole):
            change(m)
        assert mod.wq.stride() == (128, 1) and whole.wq.stride() == (256, 1) and torch.equal(mod(x), want)


@pytest.mark.parametrize("bias", [False, True])
def test_projections_that_move(calls, bias):
    """They are three launches again, nothing keeps the matrix that they were laid out in, and fuse_rotary_ lays them out anew, where quantize_linears_ leaves what it does not replace."""
    attn = projections(torch.randn(3 * 64, 64).bfloat16(), bias)
    assert attention.share_qkv_a8(attn)
    kept = [weakref.ref(t) for t in attn.__dict__["_tp_qkv8"] if t is not None]
    with torch.no_grad():
        want = attention._project_qkv(attn, inputs()[None], 32)
        moved(attn)
        assert not any(ref() is not None for ref in kept)
        calls.clear()
        got = attention._project_qkv(attn, inputs()[None], 32)
        assert calls == ["quantize_rows"] + ["linear_a8"] * 3 and all(map(torch.equal, got, want))
        at = [attn._modules[name].wq.data_ptr() for name in attention.QKV]
        quantize_linears_(nn.ModuleList([attn]), activations=True)
        assert at == [attn._modules[name].wq.data_ptr() for name in attention.QKV]
        attn.forward = types.MethodType(attention._fused_rotary_forward, attn)
        attention.fuse_rotary_(nn.ModuleList([attn]))
        calls.clear()
        got = attention._project_qkv(attn, inputs()[None], 32)
        assert calls == ["quantize_rows", "linear_a8"] and all(map(torch.equal, got, want))
        copied = copy.deepcopy(attn)
        moved(attn)
        calls.clear()
        assert all(map(torch.equal, attention._project_qkv(copied, inputs()[None], 32), want)) and calls == ["quantize_rows", "linear_a8"]
