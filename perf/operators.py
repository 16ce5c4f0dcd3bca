"""Linears with both operands in 8-bit integers and what stands around them, as measurable cases.

Every case is one call that a serving program makes of `tp.int8`: rows of activations become 8-bit codes with a scale each (`quantize_activations`, or in the launch of
an RMS norm with or without the residual's addition: `rms_norm`, `add_rms_norm`), and codes are multiplied by 8-bit weights with a scale for each channel (`linear`, and
`swiglu_up` for the gate/up pair of a gated MLP). Sizes are those of this repository's configurations: two rank shards of a Llama-2-7B-shaped decoder (d 4096, ffn 11008) and of a
Falcon-40B-shaped layer (d 8192), from one row to the 4096 of its prompts, and sizes that divide nothing.

kinds:
  norm      (q, s) = 8-bit rows of w * x / rms(x); `residual`: of x + r, and that sum itself. Codes are returned as the values they stand for
  quantize  (q, s) = 8-bit rows of x, returned as the values they stand for
  linear    act(s_x s_w (q_x . q_w^T) + bias), then, with `addend`, another rank's partial sum
  pair      silu(s_x s_g (q_x . q_g^T)) * (s_x s_u (q_x . q_u^T))
"""
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
MOST_PRODUCTS = 2 * 4096 * 5504 * 4096  # multiplications of the largest listed case
MOST_ELEMENTS = 4096 * 8192


def listed():
    return [
        # one user chatting: the norm behind the attention of a decode step, bound by the call
        {"name": "add+norm 1x4096", "kind": "norm", "rows": 1, "d": 4096, "residual": True, "dtype": "bf16"},
        # the first norm of a layer on three ragged prompts
        {"name": "norm 2103x4096", "kind": "norm", "rows": 2103, "d": 4096, "residual": False, "dtype": "f16"},
        # the second norm on long prompts of the wide model, the most memory that a norm moves
        {"name": "add+norm 4096x8192", "kind": "norm", "rows": 4096, "d": 8192, "residual": True, "dtype": "bf16"},
        # the hidden rows of a Falcon-shaped MLP shard in front of its second Linear, a small serving batch
        {"name": "quantize 16x16384", "kind": "quantize", "rows": 16, "d": 16384, "dtype": "f16"},
        # the hidden rows of a gated MLP shard on prompts
        {"name": "quantize 4096x5504", "kind": "quantize", "rows": 4096, "d": 5504, "dtype": "bf16"},
        # the down projection of one decode step, with the other rank's part
        {"name": "linear 1 4096x5504", "kind": "linear", "rows": 1, "n": 4096, "k": 5504, "bias": False, "gelu": False, "addend": True, "dtype": "bf16"},
        # batch 16 through the Falcon-shaped shard: bound by its 134 MB of weights
        {"name": "linear 16 16384x8192", "kind": "linear", "rows": 16, "n": 16384, "k": 8192, "bias": False, "gelu": True, "addend": False, "dtype": "f16"},
        # q/k/v of a few short sequences scored together: too few tiles for the device
        {"name": "linear 645 6144x4096", "kind": "linear", "rows": 645, "n": 6144, "k": 4096, "bias": True, "gelu": False, "addend": False, "dtype": "bf16"},
        # the down projection on long prompts
        {"name": "linear 4096 4096x5504", "kind": "linear", "rows": 4096, "n": 4096, "k": 5504, "bias": False, "gelu": False, "addend": True, "dtype": "bf16"},
        # the gated pair of a small serving batch
        {"name": "pair 8 5504x4096", "kind": "pair", "rows": 8, "n": 5504, "k": 4096, "dtype": "bf16"},
        # on ragged prompts, with a width that is no whole number of 128-byte lines
        {"name": "pair 701 2750x2064", "kind": "pair", "rows": 701, "n": 2750, "k": 2064, "dtype": "f16"},
        # on long prompts, the largest work here
        {"name": "pair 4096 5504x4096", "kind": "pair", "rows": 4096, "n": 5504, "k": 4096, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quantize", "linear", "linear", "linear", "pair", "pair"])
    dtype = rng.choice(["bf16", "f16"])
    if kind in ("norm", "quantize"):
        d = rng.choice([2048, 4096, 5504, 8192, 11008, 16384, _log(rng, 500, 16384)])
        case = {"kind": kind, "rows": _log(rng, 1, min(4096, MOST_ELEMENTS // d)), "d": d, "dtype": dtype}
        return {**case, "residual": rng.random() < 0.6} if kind == "norm" else case
    n = rng.choice([2048, 4096, 5504, 6144, 8192, 16384, _log(rng, 400, 16384)])
    k = rng.choice([2048, 4096, 5504, 8192, 16 * _log(rng, 40, 700)])
    rows = _log(rng, 1, 4096)
    case = {"kind": kind, "rows": max(1, min(rows, MOST_PRODUCTS // (n * k * (2 if kind == "pair" else 1)))), "n": n, "k": k, "dtype": dtype}
    if kind == "linear":
        case.update(bias=rng.random() < 0.4, gelu=rng.random() < 0.3, addend=rng.random() < 0.4)
    return case


# ---- preparation -------------------------------------------------------------------------------------------------------
def _activations(gen, rows, d, dtype):
    """Rows as decoders have them: of spread 1, a few channels far out (one in 500 times 20), some rows of a batch louder than others."""
    x = torch.randn(rows, d, device=DEV, generator=gen)
    x *= torch.where(torch.rand(d, device=DEV, generator=gen) < 0.002, 20.0, 1.0)
    x *= torch.rand(rows, 1, device=DEV, generator=gen) * 2 + 0.1
    return x.to(dtype)


def _codes(gen, rows, columns, spread):
    """Rows of normally distributed values in 8 bits, and their scales."""
    x = torch.randn(rows, columns, device=DEV, generator=gen) * spread
    scale = x.abs().amax(1, keepdim=True) / 127
    return (x / scale).round().to(torch.int8), scale.flatten()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, rows, kind = DTYPES[case["dtype"]], case["rows"], case["kind"]
    state = {"kind": kind, "dtype": dtype}
    if kind in ("norm", "quantize"):
        state["x"] = _activations(gen, rows, case["d"], dtype)
        if rows >= 8:
            state["x"][rows // 2] = 0  # a row of padding
        if kind == "norm":
            state["w"] = (1 + 0.2 * torch.randn(case["d"], device=DEV, generator=gen)).to(dtype)
            state["r"] = _activations(gen, rows, case["d"], dtype) if case["residual"] else None
            if rows >= 8 and case["residual"]:
                state["r"][rows // 2] = 0
        return state
    n, k = case["n"], case["k"]
    state["x"], state["xs"] = _codes(gen, rows, k, 1.0)
    state["w"], state["ws"] = _codes(gen, n, k, 0.02)
    if kind == "pair":
        state["u"], state["us"] = _codes(gen, n, k, 0.02)
        return state
    state["bias"] = torch.randn(n, device=DEV, generator=gen).to(dtype) if case["bias"] else None
    state["addend"] = torch.randn(rows, n, device=DEV, generator=gen).to(dtype) if case["addend"] else None
    state["gelu"] = case["gelu"]
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def _gelu(v):
    return 0.5 * v * (1 + torch.erf(v * 0.5**0.5))


def _plain_rows(p, factor):
    """8-bit rows of p (fp32) times factor [rows]: (values, scales). The quotient is rounded as it is, so in 64 bits: many lie next to a half."""
    most = p.abs().amax(1)
    empty = most == 0
    codes = (p.double() * 127 / torch.where(empty, 1.0, most).double()[:, None]).round().float()
    scale = torch.where(empty, 1.0, most * factor / 127)
    return codes * scale[:, None], scale


def _own_rows(rows):
    return {"values": rows.dequantize(torch.float32), "scale": rows.scale}


def run(state):
    kind, x, dtype = state["kind"], state["x"], state["dtype"]
    if own:
        from tensor_parallel_amd import int8

        if kind == "quantize":
            return _own_rows(int8.quantize_activations(x))
        if kind == "norm":
            if state["r"] is None:
                return _own_rows(int8.rms_norm(x, state["w"], EPS))
            total, rows = int8.add_rms_norm(state["r"], x, state["w"], EPS)
            return {"total": total, **_own_rows(rows)}
        rows = int8.QuantizedRows(x, state["xs"], dtype)
        if kind == "pair":
            return int8.swiglu_up(rows, state["w"], state["ws"], state["u"], state["us"])
        return int8.linear(rows, state["w"], state["ws"], state["bias"], gelu=state["gelu"], addend=state["addend"])
    if kind == "quantize":
        values, scale = _plain_rows(x.float(), 1.0)
        return {"values": values, "scale": scale}
    if kind == "norm":
        total = x if state["r"] is None else (state["r"].float() + x.float()).to(dtype)
        t = total.float()
        values, scale = _plain_rows(t * state["w"].float(), torch.rsqrt((t * t).mean(1) + EPS))
        out = {"values": values, "scale": scale}
        return out if state["r"] is None else {"total": total, **out}
    scale = state["xs"][:, None]
    y = (x.float() @ state["w"].float().t()) * scale * state["ws"]
    if kind == "pair":
        u = (x.float() @ state["u"].float().t()) * scale * state["us"]
        return (y / (1 + torch.exp(-y)) * u).to(dtype)
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if state["gelu"]:
        y = _gelu(y)
    y = y.to(dtype)
    return y if state["addend"] is None else (y.float() + state["addend"].float()).to(dtype)


def work(case):
    rows = case["rows"]
    if case["kind"] in ("norm", "quantize"):
        d = case["d"]
        read = 2 * rows * d + (2 * rows * d if case.get("residual") else 0) + (2 * d if case["kind"] == "norm" else 0)
        written = 4 * rows * d + 4 * rows + (2 * rows * d if case.get("residual") else 0)  # the values in 32 bits, as they are returned
        return {"bytes": read + written, "flops": 8 * rows * d}
    n, k, matrices = case["n"], case["k"], 2 if case["kind"] == "pair" else 1
    extra = (2 * n if case.get("bias") else 0) + (2 * rows * n if case.get("addend") else 0)
    return {"bytes": rows * k + 4 * rows + matrices * (n * k + 4 * n) + 2 * rows * n + extra, "flops": 2 * rows * n * k * matrices}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].double()
    if case["kind"] in ("norm", "quantize"):
        out, total = {}, x
        if state.get("r") is not None:
            total = (x + state["r"].double()).to(state["dtype"]).double()  # the norm is defined on the sum that is stored
            out["total"] = total
        if case["kind"] == "norm":
            product = total * state["w"].double()
            y = product / torch.sqrt(total.square().mean(1, keepdim=True) + EPS)
        else:
            product = y = total
        largest, peak = product.abs().max(1, keepdim=True).values, y.abs().max(1, keepdim=True).values
        scale = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
        q = torch.where(largest > 0, torch.round(product * 127 / largest.clamp_min(1e-300)), torch.zeros_like(product))
        return {**out, "values": q * scale, "scale": scale[:, 0]}
    xs = x * state["xs"].double()[:, None]
    first = torch.matmul(xs, (state["w"].double() * state["ws"].double()[:, None]).T)
    if case["kind"] == "pair":
        second = torch.matmul(xs, (state["u"].double() * state["us"].double()[:, None]).T)
        return first * torch.sigmoid(first) * second
    if state["bias"] is not None:
        first = first + state["bias"].double()
    if case["gelu"]:
        first = first * 0.5 * torch.special.erfc(-first * 0.5**0.5)
    return first if state["addend"] is None else first + state["addend"].double()
