"""Gated MLPs and projections of 16-bit Linears whose parts change, or are watched, once gate and up, or q, k and v, are one launch. The launch is stood in for by torch on host tensors, so no GPU is
needed."""
import copy
import gc
import weakref

import pytest
import torch
from torch import nn

from tensor_parallel_amd import _native, attention, shard_modules, together
from tensor_parallel_amd.collectives import SumContext


class Mlp(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj, self.act_fn = nn.Linear(64, 96, bias=False), nn.Linear(64, 96, bias=False), nn.Linear(96, 64, bias=False), nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


@pytest.fixture
def calls(monkeypatch):
    made = []

    def pair(x, wg, wu):
        made.append("swiglu_up")
        return nn.functional.silu(x @ wg.t()) * (x @ wu.t())

    monkeypatch.setattr(_native, "swiglu_up", pair)
    monkeypatch.setattr(_native, "linear", lambda x, w, b=None, **more: nn.functional.linear(x, w, b))
    return made


def fused():
    torch.manual_seed(0)
    block = Mlp().bfloat16()
    shard_modules.install_shard_kernels(block)
    with torch.no_grad():
        block(inputs())
    assert block.forward.__func__ is shard_modules._gated_mlp_forward
    return block


def inputs():
    return torch.randn(5, 64, generator=torch.Generator().manual_seed(1)).bfloat16()


def with_bias():
    return nn.Linear(64, 96).bfloat16()


@pytest.mark.parametrize("change", [
    lambda m: setattr(m, "gate_proj", with_bias()),
    lambda m: setattr(m, "up_proj", with_bias()),
    lambda m: setattr(m.gate_proj, "bias", nn.Parameter(torch.randn(96).bfloat16())),
    lambda m: setattr(m, "act_fn", nn.ReLU()),
    lambda m: setattr(m.act_fn, "forward", torch.tanh),
    lambda m: m.act_fn.register_forward_hook(lambda mod, args, out: 2 * out),
    lambda m: m.up_proj.register_forward_hook(lambda mod, args, out: 2 * out),
], ids=["gate with a bias", "up with a bias", "a bias assigned", "ReLU", "a forward of the SiLU's own", "a hook on the SiLU", "a hook on up"])
def test_a_part_that_is_something_else_since(calls, change):
    x, block = inputs(), fused()
    with torch.no_grad():
        before = block(x)
        change(block)
        calls.clear()
        got, want = block(x), Mlp.forward(block, x)
    assert not calls and torch.equal(got, want) and not torch.equal(got, before)


def test_hooks_on_all_modules(calls):
    block, told = fused(), []
    handle = nn.modules.module.register_module_forward_hook(lambda mod, *rest: told.append(mod))
    try:
        with torch.no_grad():
            block(inputs())
    finally:
        handle.remove()
    assert block.gate_proj in told and block.up_proj in told and block.act_fn in told


def test_the_launch_comes_back_and_goes_with_a_copy(calls):
    x, block = inputs(), fused()
    with torch.no_grad():
        want, kept = block(x), block.act_fn
        block.act_fn = nn.ReLU()
        block(x)
        block.act_fn = kept
        calls.clear()
        assert torch.equal(block(x), want) and torch.equal(copy.deepcopy(block)(x), want) and calls == ["swiglu_up"] * 2


def test_a_linear_of_the_same_kind_in_gates_place(calls):
    """It is what the launch multiplies by, and nothing keeps the one before."""
    x, block = inputs(), fused()
    before = weakref.ref(block.gate_proj)
    new = nn.Linear(64, 96, bias=False).bfloat16()
    new.__class__ = shard_modules.ShardLinear
    block.gate_proj = new
    calls.clear()
    with torch.no_grad():
        assert torch.equal(block(x), Mlp.forward(block, x)) and calls == ["swiglu_up"]
    del new
    gc.collect()
    assert before() is None


def test_who_is_said_to_return_the_down_projections_output(calls):
    block, known = fused(), []
    for act in (block.act_fn, nn.Tanh()):
        block.act_fn = act
        ctx = SumContext(None, 0, nn.Module(), block)
        together.push_sum_context(ctx)
        try:
            with torch.inference_mode():
                block(inputs())
        finally:
            together.pop_sum_context()
        known.append(shard_modules.hands_through(ctx, block.down_proj))
    assert known == [True, False]


def projections(bias):
    """q, k and v as fuse_rotary_ lays them out."""
    torch.manual_seed(0)
    attn, whole, shift = nn.Module(), torch.randn(96, 64).bfloat16(), torch.randn(96).bfloat16()
    for name, rows in (("q_proj", (0, 64)), ("k_proj", (64, 80)), ("v_proj", (80, 96))):
        part = nn.Linear(64, rows[1] - rows[0], bias=bias)
        part.__class__, part.weight = shard_modules.ShardLinear, nn.Parameter(whole[slice(*rows)])
        if bias:
            part.bias = nn.Parameter(shift[slice(*rows)])
        setattr(attn, name, part)
    attn.__dict__["_tp_qkv"] = (whole, shift if bias else None)
    return attn


def test_projections_that_are_watched(calls, monkeypatch):
    """A hook on one of q, k and v or on all modules is told of their calls; without one they are one launch again."""
    inner, launches = _native.linear, []
    monkeypatch.setattr(_native, "linear", lambda x, w, b=None, **more: launches.append(w.shape[0]) or inner(x, w, b))
    attn = projections(False)
    x, told = inputs()[None], []

    def project():
        launches.clear()
        with torch.no_grad():
            return [part.flatten(2) for part in attention._project_qkv(attn, x, 16)]

    want = project()
    assert launches == [96]
    for register in (attn.k_proj.register_forward_hook, nn.modules.module.register_module_forward_hook):
        handle = register(lambda mod, args, out: told.append(mod))
        try:
            got = project()
        finally:
            handle.remove()
        assert launches == [64, 16, 16] and attn.k_proj in told
        for a, b in zip(got, want):
            torch.testing.assert_close(a.float(), b.float(), rtol=2.0**-7, atol=64 * 2.0**-24 * 64)  # (torch may add these up in another order: a step of bf16 each)
        told.clear()
    assert all(map(torch.equal, project(), want)) and launches == [96]


@pytest.mark.parametrize("change", ["another", "none", "one where there was none"])
def test_a_projection_with_another_bias(calls, change):
    attn, x = projections(change != "one where there was none"), inputs()[None]
    with torch.no_grad():
        attention._project_qkv(attn, x, 16)
        attn.k_proj.bias = None if change == "none" else nn.Parameter(torch.randn(16).bfloat16())
        got = attention._project_qkv(attn, x, 16)
        assert all(torch.equal(part.flatten(2), attn._modules[name](x)) for part, name in zip(got, attention.QKV))


class Exchanged(Mlp):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class Scaled(Mlp):
    def forward(self, x):
        return 1.01 * self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Steep(Mlp):
    class Swish(nn.Module):
        def forward(self, x):
            return x * torch.sigmoid(1.7 * x)

    def __init__(self):
        super().__init__()
        self.act_fn = self.Swish()


@pytest.mark.parametrize("cls", [Exchanged, Scaled, Steep])
@pytest.mark.parametrize("first", ["zeros", "values"])
def test_blocks_of_another_formula(calls, cls, first):
    """They keep their own forward, whatever they are called with first."""
    torch.manual_seed(0)
    block, x = cls().bfloat16(), inputs()
    shard_modules.install_shard_kernels(block)
    with torch.no_grad():
        block(torch.zeros_like(x) if first == "zeros" else x)
        assert torch.equal(block(x), cls.forward(block, x))


def test_a_class_that_is_given_another_forward(calls):
    class Own(Mlp):
        forward = Mlp.forward

    torch.manual_seed(0)
    block, x = Own().bfloat16(), inputs()
    shard_modules.install_shard_kernels(block)
    with torch.no_grad():
        block(x)
        assert block.forward.__func__ is shard_modules._gated_mlp_forward
        Own.forward = Scaled.forward
        assert torch.equal(block(x), Scaled.forward(block, x))
