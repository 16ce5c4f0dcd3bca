"""int8 shard Linears from the Python layer: weight-only with outlier columns kept in 16 bits, or of rows in 8 bits.

The reference has no int8 code of its own: its users quantise the wrapped model with a third-party library before or
after `tp.tensor_parallel` (README of the reference, LLM.int8 notebooks). This module is that step for the shards of this
package: `quantize_linears_` turns the 16-bit Linears of a module tree (the rank shards of a `tp.TensorParallel`, or any
module on a HIP device) into `ShardLinearW8`, whose forward is `tpamd_linear_w8`. The definition is closed form:

  O        = the outlier input columns of a Linear (chosen by the caller, sorted)
  scale[n] = max over k not in O of |W[n,k]| / 127            (1.0 where that max is 0)
  Wq[n,k]  = clamp(round_half_even(W[n,k] / scale[n]), -127, 127) for k not in O, 0 for k in O
  y        = x . (Wq * scale[:,None])^T  +  x[:, O] . W[:, O]^T  (+ bias)

The quantiser runs on the device with torch's elementwise ops (it runs once per weight); the Linear itself runs on the
library's kernels only.

With both operands in 8 bits (`QuantizedRows`, `quantize_activations`, `rms_norm`, `add_rms_norm`, `linear`, `swiglu_up`) the rows of an activation have a scale each too:

  a        = max |p| over the row, p = x, or w x of an RMS norm's input x (its factor f = rsqrt(mean(x^2) + eps) is in the scale alone; else f = 1)
  codes    = round_half_even(127 p / a) of the exact quotient          scale = a f / 127      (no |p| of 2^-100 or more: 1.0, an infinity or NaN: NaN, and codes of 0)
  linear   = act(scale[m] wscale[n] (codes . Wq^T) + bias), the product exact in 32-bit integers, rounded once (a partial sum of other ranks is added to the rounded value)

A quantised Linear no longer has a `weight`: `save_tensor_parallel`, which rebuilds the full
weights of the original model from the shards, refuses a model that holds one; its shards can be saved as they are.
"""
from __future__ import annotations

import functools
import types
from typing import Callable, Mapping, NamedTuple, Optional, Sequence, Tuple, Union

import torch
from torch import nn

from . import _native, together
from . import shard_modules
from .attention import QKV, share_qkv_a8
from .shard_modules import _guard, is_conv1d, product_in_context

OutlierChoice = Union[None, Mapping[str, Sequence[int]], Callable[[str, nn.Module], Optional[Sequence[int]]]]


def quantize_rows(w: torch.Tensor, outlier_cols: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """w [N, K] (bfloat16 / float16 / float32, on a HIP device) -> (wq int8 [N, K], scale float32 [N],
    outlier_idx int32 [n_out] sorted, w_out [N, n_out] in w's dtype) by the definition in the module docstring."""
    _native.require_device(w, "quantize_rows")
    if w.dim() != 2:
        raise ValueError(f"quantize_rows: expected a [N, K] weight, got {tuple(w.shape)}")
    N, K = w.shape
    if outlier_cols is None:
        cols = torch.empty(0, dtype=torch.int64, device=w.device)
    else:
        cols = torch.as_tensor(outlier_cols, dtype=torch.int64, device=w.device).flatten()
        if cols.numel() and (int(cols.min()) < 0 or int(cols.max()) >= K):
            raise ValueError(f"quantize_rows: outlier columns must lie in [0, {K})")
        cols = torch.unique(cols)  # sorted, no repeats
    keep = torch.ones(K, dtype=torch.bool, device=w.device)
    keep[cols] = False
    q = torch.empty((N, K), dtype=torch.int8, device=w.device)
    scale = torch.empty(N, dtype=torch.float32, device=w.device)
    # The definition's two divisions are float32 divisions rounded correctly. The device's float32 division is allowed an
    # error of a unit in the last place, which would move a quotient across a rounding boundary now and then: they are
    # done in float64 and rounded to float32 instead, which gives the correctly rounded float32 quotient. Blocks of rows
    # bound the temporaries.
    for r0 in range(0, N, 4096):
        wd = w.detach()[r0:r0 + 4096].double()
        absmax = wd.abs().masked_fill(~keep, 0.0).amax(dim=1) if K else wd.new_zeros(wd.shape[0])
        sc = (absmax / 127.0).float()
        sc = torch.where(sc == 0, torch.ones_like(sc), sc)
        quot = (wd / sc.double()[:, None]).float()
        q[r0:r0 + 4096] = torch.round(quot).clamp_(-127, 127).to(torch.int8)  # torch.round: ties to even
        scale[r0:r0 + 4096] = sc
    q[:, ~keep] = 0
    return q, scale, cols.to(torch.int32), w.detach()[:, cols].contiguous()


class QuantizedRows(NamedTuple):
    """Rows of an activation in 8 bits: `scale` * `codes` stand for rows of `dtype`, which is what Linears of them return."""

    codes: torch.Tensor  # int8 [..., K]; of many rows each begins on a 128-byte boundary, so there may be bytes between them
    scale: torch.Tensor  # float32 [...]
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dim(self) -> int:
        return self.codes.dim()

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """scale * codes, in `dtype` (the rows' own by default)."""
        return _guard(_native.dequantize_rows(self.codes, self.scale, self.dtype if dtype is None else dtype), self.scale)


def _calls():
    """The library's calls: made together with the other ranks where ranks take turns."""
    return _native if together.current_turn() is None else together


def quantize_activations(x: torch.Tensor) -> QuantizedRows:
    """The rows of x (bfloat16 or float16, on a HIP device) in 8 bits, by the definition in the module docstring. Inference only, as everything here: a
    backward pass through the rows' scales, or what Linears make of them, raises."""
    codes, scale = _calls().quantize_rows(x)
    return QuantizedRows(codes, _guard(scale, x), x.dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> QuantizedRows:
    """The RMS norm of x's rows in 8 bits, in one launch: weight * x * rsqrt(mean(x^2) + eps), not rounded in between."""
    codes, scale = _calls().rms_norm_q8(x, weight, eps)
    return QuantizedRows(codes, _guard(scale, x, weight), x.dtype)


def add_rms_norm(r: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float) -> Tuple[torch.Tensor, QuantizedRows]:
    """(r + x, the RMS norm of that sum in 8 bits), in one launch: a residual stream and the input of the Linears behind its norm."""
    total, codes, scale = _calls().add_rms_norm_q8(r, x, weight, eps)
    return _guard(total, r, x), QuantizedRows(codes, _guard(scale, r, x, weight), x.dtype)


def linear(rows: QuantizedRows, wq: torch.Tensor, wscale: torch.Tensor, bias: Optional[torch.Tensor] = None, *, gelu: bool = False,
           addend: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A Linear of 8-bit rows on int8 weights [N, K] with a float32 scale for each output (`quantize_rows` without outlier columns makes both), in the rows' dtype. `addend`: other ranks' partial
    sum, added to the rounded result. K is at most 131071 (the sum fits 32 bits)."""
    codes, scale, dtype = rows
    return _guard(_native.linear_a8(codes, scale, wq, wscale, bias, dtype, _native.ACT_GELU if gelu else _native.ACT_NONE, addend), scale, wscale, bias, addend)


def swiglu_up(rows: QuantizedRows, gate: torch.Tensor, gate_scale: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor) -> torch.Tensor:
    """silu(g) * u of the Linears g and u of 8-bit rows (as in `linear`, no bias), in one launch and rounded once."""
    codes, scale, dtype = rows
    return _guard(_calls().swiglu_up_a8(codes, scale, gate, gate_scale, up, up_scale, dtype), scale, gate_scale, up_scale)


# From 65 to this many rows a Linear neither meets its peer nor hands a sum over: the host sets the pace of an eager prompt there, and the reduction kernel's launch costs it
# less than keeping book of what a module returns (the Falcon-40B-shaped layer on 200 / 400 / 512 rows: 965 / 975 / 1012 us, 1000 / 1005 / 1047 with
# the sum in the Linears; on 600 / 850 / 1024 rows, where the device does, 1268 / 1457 / 1573 and 1261 / 1449 / 1562).
W8_ALONE_ROWS = 512


class ShardLinearW8(nn.Module):
    """A Linear whose weight is stored as int8 rows with one float32 scale each, plus the outlier input columns in the
    activation dtype; the forward is `tpamd_linear_w8`. Inference only."""

    def __init__(self, wq: torch.Tensor, scale: torch.Tensor, outlier_idx: torch.Tensor, w_out: torch.Tensor,
                 bias: Optional[torch.Tensor], dtype: torch.dtype):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"ShardLinearW8: activations must be bfloat16 or float16, got {dtype}")
        self.out_features, self.in_features = wq.shape
        self.dtype = dtype
        self.register_buffer("wq", wq.contiguous())
        self.register_buffer("scale", scale.contiguous())
        self.register_buffer("outlier_idx", outlier_idx.to(torch.int32).contiguous())
        self.register_buffer("w_out", w_out.to(dtype).contiguous())
        self.register_buffer("bias", None if bias is None else bias.detach().to(dtype).contiguous())

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    outlier_cols: Optional[Sequence[int]] = None) -> "ShardLinearW8":
        """Quantise a [out, in] weight that lives on a HIP device."""
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"ShardLinearW8: the weight must be bfloat16 or float16, got {weight.dtype}")
        wq, scale, idx, w_out = quantize_rows(weight, None if outlier_cols is None else torch.as_tensor(outlier_cols))
        return cls(wq, scale, idx, w_out, bias, weight.dtype)

    def forward(self, input: torch.Tensor) -> torch.Tensor:  # noqa: A002
        return self._product(input, _native.ACT_NONE)

    def _product(self, input: torch.Tensor, act: int) -> torch.Tensor:  # noqa: A002
        if input.dtype != self.dtype:
            raise TypeError(f"ShardLinearW8: the input is {input.dtype}, the Linear was quantised for {self.dtype}")
        idx = self.outlier_idx
        n_out = idx.numel()
        operands = (input.detach(), self.wq, self.scale, idx if n_out else None, self.w_out if n_out else None, self.bias)
        few = input.numel() <= together.W8_TOGETHER_ROWS * input.shape[-1]
        if not few and input.numel() <= W8_ALONE_ROWS * input.shape[-1]:
            return _guard(_native.linear_w8(*operands, act), input)
        alone = functools.partial(_native.linear_w8, *operands, act)
        return product_in_context(self, input, self.out_features, (input,), functools.partial(together.linear_w8, *operands, act) if few else alone, alone,
                                  (lambda rank, op: together.linear_w8_sum(*operands, rank, op)) if few and act == _native.ACT_NONE else None, learned=False)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"outlier_columns={self.outlier_idx.numel()}, dtype={self.dtype}")


def _in_lines(wq: torch.Tensor) -> torch.Tensor:
    """Codes [N, K] whose rows begin on 128-byte boundaries (K a multiple of 16; else as they are, one after another: the matrix pipe takes whole pieces of 16 codes, and such rows go to a kernel that
    takes any, 20 to 75 times slower). A row of K = 2752 that begins inside a line shares it with the next one, and products ask for such lines twice: 8 x 4096 x 2752 5.3 us, 4.9 with rows in
    lines; 16 x 4096 x 5520 9.7 and 7.6; the pair of 4096 x 5504 x 4112 198, 170 with the input's rows in lines as well."""
    K = wq.shape[1]
    if K % 128 == 0 or K % 16 != 0:
        return wq.contiguous()
    if wq.stride(1) == 1 and wq.stride(0) % 128 == 0 and wq.stride(0) >= K and wq.storage_offset() % 128 == 0:
        return wq  # they are
    lines = wq.new_zeros((wq.shape[0], (K + 127) // 128 * 128))
    lines[:, :K] = wq
    return lines[:, :K]


class ShardLinearA8(nn.Module):
    """A Linear of 8-bit rows: weights int8 with a float32 scale for each output, the input's rows quantised by the forward (`quantize_activations`) unless they come as
    `QuantizedRows`; the product is `tpamd_linear_a8`. Inference only."""

    def __init__(self, wq: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor], dtype: torch.dtype):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"ShardLinearA8: activations must be bfloat16 or float16, got {dtype}")
        self.out_features, self.in_features = wq.shape
        if self.in_features > MAX_A8_FEATURES:
            raise ValueError(f"ShardLinearA8: sums of {self.in_features} products of 8-bit codes may not fit 32 bits (at most {MAX_A8_FEATURES} do)")
        self.dtype = dtype
        self.register_buffer("wq", _in_lines(wq))
        self.register_buffer("scale", scale.contiguous())
        self.register_buffer("bias", None if bias is None else bias.detach().to(dtype).contiguous())

    def _apply(self, fn, recurse=True):
        """Moves with its module, and stays what it was quantised for: a model that is told its dtype once more (`.to(torch.bfloat16)`) would otherwise have 16-bit scales, which no product takes.
        Codes that have moved begin their rows on 128-byte boundaries again, and let go of the matrix that they were laid out in with others (attention.share_qkv_a8)."""
        scale, bias, codes = self.scale, self.bias, self.wq
        super()._apply(fn, recurse)
        if self.wq is not codes:
            self.wq = _in_lines(self.wq)
            self.__dict__.pop("_tp_rows_of", []).clear()
        if self.scale.dtype is not torch.float32:
            self.scale = scale.to(self.scale.device)
        if bias is not None and self.bias.dtype is not self.dtype:
            self.bias = bias.to(self.bias.device)
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self.wq = _in_lines(self.wq)  # (assign=True puts the saved tensor in)

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "wq"] = destination[prefix + "wq"].contiguous()  # without the bytes between its rows

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "ShardLinearA8":
        """Quantise a [out, in] weight that lives on a HIP device."""
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"ShardLinearA8: the weight must be bfloat16 or float16, got {weight.dtype}")
        if weight.dim() == 2 and weight.shape[1] > MAX_A8_FEATURES:
            raise ValueError(f"ShardLinearA8: sums of {weight.shape[1]} products of 8-bit codes may not fit 32 bits (at most {MAX_A8_FEATURES} do)")
        wq, scale, _, _ = quantize_rows(weight)
        return cls(wq, scale, bias, weight.dtype)

    def rows_of(self, input: Union[torch.Tensor, QuantizedRows]) -> QuantizedRows:  # noqa: A002
        if input.dtype != self.dtype:
            raise TypeError(f"ShardLinearA8: the input is {input.dtype}, the Linear was quantised for {self.dtype}")
        return input if type(input) is QuantizedRows else quantize_activations(input)

    def forward(self, input: Union[torch.Tensor, QuantizedRows]) -> torch.Tensor:  # noqa: A002
        return self._product(input, _native.ACT_NONE)

    def _product(self, input: Union[torch.Tensor, QuantizedRows], act: int) -> torch.Tensor:  # noqa: A002
        rows = self.rows_of(input)
        operands = (rows.codes, rows.scale, self.wq, self.scale, self.bias, self.dtype, act)
        return product_in_context(self, rows, self.out_features, (rows.scale,), functools.partial(together.linear_a8, *operands), functools.partial(_native.linear_a8, *operands),
                                  (lambda rank, op: together.linear_a8_sum(*operands, rank, op)) if rows.codes.numel() <= together.A8_TOGETHER_ROWS * self.in_features else None, learned=False)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, dtype={self.dtype}"


shard_modules.LINEAR_A8 = ShardLinearA8
MAX_A8_FEATURES = 131071  # 128 * 128 * in_features < 2^31


def _outliers_of(choice: OutlierChoice, name: str, module: nn.Module) -> Optional[Sequence[int]]:
    if choice is None:
        return None
    if callable(choice):
        return choice(name, module)
    return choice.get(name)


def quantize_linears_(module: nn.Module, outlier_cols: OutlierChoice = None,
                      skip: Callable[[str, nn.Module], bool] = lambda name, m: False, activations: bool = False) -> int:
    """Replace, in place, every 16-bit `nn.Linear` (and transformers `Conv1D`) under `module` whose weight lives on a HIP
    device by a `ShardLinearW8`. `outlier_cols`: the outlier input columns per Linear, as a mapping from the Linear's name
    under `module` (as in `module.named_modules()`) or as a function of (name, Linear); none by default. `skip(name,
    Linear)` keeps a Linear as it is (an output head, say). Returns how many were replaced.

    `activations=True`: both operands in 8 bits (`ShardLinearA8`; no outlier columns). A SiLU-gated MLP block, one whose forward is down_proj(act_fn(gate_proj(x)) * up_proj(x)) and nothing else, then
    quantises its input once for gate and up, which are one launch (`swiglu_up`), a fused attention of the Llama pattern its input once for q, k and v, which are one launch too, and a Llama decoder layer takes their inputs from the launches of its norms (`rms_norm`,
    `add_rms_norm`) where nothing watches the norms. Linears whose inputs are no multiple of 16 features are better left out (`skip`): the matrix pipe does not take them."""
    if activations and outlier_cols is not None:
        raise ValueError("quantize_linears_: with 8-bit activations there are no outlier columns")
    replaced = 0
    for parent_name, parent in list(module.named_modules()):
        projections = False  # whether one of q, k and v is replaced here
        for child_name, child in list(parent.named_children()):
            name = f"{parent_name}.{child_name}" if parent_name else child_name
            conv1d = is_conv1d(child)
            if not (isinstance(child, nn.Linear) or conv1d):
                continue
            w = child.weight
            if w.device.type != "cuda" or w.dtype not in (torch.bfloat16, torch.float16) or skip(name, child):
                continue
            weight = w.detach().t() if conv1d else w.detach()  # Conv1D keeps [in, out]
            if activations:
                new = ShardLinearA8.from_weight(weight, getattr(child, "bias", None))
            else:
                new = ShardLinearW8.from_weight(weight, getattr(child, "bias", None), _outliers_of(outlier_cols, name, child))
            setattr(parent, child_name, new)
            replaced += 1
            if child_name in QKV:  # their 16-bit weights laid out as one matrix (fuse_rotary_) have no reader any more
                parent.__dict__.pop("_tp_qkv", None)
                projections = True
            # a SiLU-gated MLP block whose fused forward reads gate_proj.weight / up_proj.weight goes back to its own forward
            fused = parent.__dict__.get("forward")
            if getattr(fused, "__func__", None) in (shard_modules._gated_mlp_forward, shard_modules._gated_mlp_first_forward):
                del parent.forward
        if activations and projections:  # (others' codes stay where they are: a recorded graph may read them)
            share_qkv_a8(parent)
        if activations and shard_modules.is_gated_silu_a8_mlp(parent):
            parent.forward = types.MethodType(shard_modules._gated_mlp_a8_forward, parent)
    return replaced
