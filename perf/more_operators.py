"""Rotary positions, norms of query and key heads, and paged key/value caches, as measurable cases.

Every case is one call that a serving program makes between a layer's projection of q, k and v and its output projection: the rows' heads are rotated to their positions
(`tp.attention.rotate`), normed on the way where the model has weights for that, handed over to a cache whose positions lie in pages (`tp.paged.append`), and attend to
the positions that are cached (`tp.paged.attend`). Head counts are those of one of two rank shards of this repository's configurations: 16 heads of 128 with as many keys
(d 4096), 64 heads of 64 on 4 keys (d 8192, grouped), and whole models' on one GPU. Sequences differ in length as they do in a serving batch, and their pages lie
scattered over the pool.

kinds:
  rotate   q, k with every pair (a, b) of a head's first `part` elements turned by position * frequency: pairs are neighbours (`interleaved`) or half of `part` apart.
           `norm`: the RMS norm of each head with a weight for queries and one for keys comes first, in the same pass. `factor` scales cos and sin (long contexts)
  append   the same on the new rows of `seqs` sequences, k and v going to their pages. The whole pools are returned
  attend   causal attention of the new rows on their sequence's pages, from a single row (decode) to a whole prompt
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
MOST_PAIRS = 32 * 4096 * 4097 // 2  # (query row, key) pairs of the largest listed case, all query heads together
MOST_POOL = 1 << 28  # elements of a pool of keys or values


def listed():
    return [
        # one user chatting: bound by the call
        {"name": "rotate 1 16+16x128", "kind": "rotate", "rows": 1, "hq": 16, "hkv": 16, "d": 128, "part": 128, "interleaved": False, "norm": False, "factor": 1.0, "far": 4096, "dtype": "bf16"},
        # ragged prompts scored together, neighbours as pairs, half of the head turned
        {"name": "rotate 2103 64+4x64 inter", "kind": "rotate", "rows": 2103, "hq": 64, "hkv": 4, "d": 64, "part": 32, "interleaved": True, "norm": False, "factor": 1.0, "far": 2048, "dtype": "f16"},
        # a serving batch's decode step with normed heads
        {"name": "norm+rotate 40 32+8x128", "kind": "rotate", "rows": 40, "hq": 32, "hkv": 8, "d": 128, "part": 128, "interleaved": False, "norm": True, "factor": 1.0, "far": 32768, "dtype": "f16"},
        # a long document's chunk, frequencies and factor of a context extended to a million positions
        {"name": "norm+rotate 4096 32+32x128", "kind": "rotate", "rows": 4096, "hq": 32, "hkv": 32, "d": 128, "part": 128, "interleaved": False, "norm": True, "factor": 1.2, "far": 1 << 20, "dtype": "bf16"},
        # the decode step of 40 users of the grouped model
        {"name": "append 40x1 64+4x64", "kind": "append", "seqs": 40, "cached": 1000, "new": 1, "ragged": True, "hq": 64, "hkv": 4, "d": 64, "page": 16, "part": 64, "interleaved": False,
         "norm": False, "factor": 1.0, "dtype": "f16"},
        # five prompts that arrive together, packed without padding
        {"name": "append 5 prompts 16+16x128", "kind": "append", "seqs": 5, "cached": 0, "new": 701, "ragged": True, "hq": 16, "hkv": 16, "d": 128, "page": 64, "part": 128, "interleaved": False,
         "norm": True, "factor": 1.0, "dtype": "bf16"},
        # one user chatting on 500 positions: latency
        {"name": "attend 1x1 on 500 16x128", "kind": "attend", "seqs": 1, "cached": 500, "new": 1, "ragged": False, "hq": 16, "hkv": 16, "d": 128, "page": 16, "dtype": "bf16"},
        # 64 users of the grouped model, from a few words to a document
        {"name": "attend 64x1 ragged 64/4x64", "kind": "attend", "seqs": 64, "cached": 8000, "new": 1, "ragged": True, "hq": 64, "hkv": 4, "d": 64, "page": 16, "dtype": "f16"},
        # one question about a long document: few heads, many keys
        {"name": "attend 1x1 on 100k 32/8x128", "kind": "attend", "seqs": 1, "cached": 100000, "new": 1, "ragged": False, "hq": 32, "hkv": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # a step of a server that mixes chunks of prompts with other users' decode steps
        {"name": "attend mixed 24 32/8x128", "kind": "attend", "seqs": 24, "cached": 6000, "new": 512, "ragged": True, "hq": 32, "hkv": 8, "d": 128, "page": 32, "dtype": "bf16"},
        # the last chunk of a long document
        {"name": "attend 500 on 30k 16x128", "kind": "attend", "seqs": 1, "cached": 30000, "new": 500, "ragged": False, "hq": 16, "hkv": 16, "d": 128, "page": 128, "dtype": "f16"},
        # a whole prompt, the largest work here
        {"name": "attend 4096 on 0 32x128", "kind": "attend", "seqs": 1, "cached": 0, "new": 4096, "ragged": False, "hq": 32, "hkv": 32, "d": 128, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "append", "append", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 96, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    hq = hkv * rng.choice([1, 1, 2, 4, 5, 8, 16])
    if kind != "attend":
        shape = {"hq": hq, "hkv": hkv, "d": d, "part": rng.choice([d, d, d // 2, d // 4]), "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.5,
                 "factor": rng.choice([1.0, 1.2]), "dtype": dtype}
    if kind == "rotate":
        rows = _log(rng, 1, max(1, min(8192, 4096 * 64 * 128 // ((hq + hkv) * d))))
        return {"kind": kind, "rows": rows, "far": _log(rng, 512, 1 << 20), **shape}
    page = rng.choice([16, 16, 32, 64, 128, 256])
    seqs = rng.choice([1, 1, _log(rng, 2, 96)])
    decode = rng.random() < 0.5
    ragged = rng.random() < 0.6
    while True:
        cached = _log(rng, 10, 100000) if decode else rng.choice([0, _log(rng, 10, 30000)])
        new = rng.choice([1, 1, 1, 3]) if decode else _log(rng, 2, 4096)
        case = {"kind": kind, "seqs": seqs, "cached": cached, "new": new, "ragged": ragged, "hq": hq, "hkv": hkv, "d": d, "page": page, "dtype": dtype}
        counts, lengths = _lengths(case)
        pairs = hq * seqs * max(counts) * max(lengths)  # what the plain form makes room for
        if pairs <= MOST_PAIRS * 2 and _pool_pages(case) * page * hkv * d <= MOST_POOL and sum(counts) * (hq + 2 * hkv) * d <= 4096 * 96 * 128:
            break
        seqs = max(1, seqs // 2)
    return {**case, **shape} if kind == "append" else case


def _lengths(case):
    """The new rows of each sequence and its positions with them: alike, or spread over the logarithm; of a batch with long chunks every fourth sequence has one and the
    others, in `attend`, a single row."""
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["cached"] + case["new"]] * case["seqs"]
    rng = random.Random("%d %d %d" % (case["seqs"], case["cached"], case["new"]))
    counts, lengths = [], []
    for i in range(case["seqs"]):
        single = case["kind"] == "attend" and i % 4
        counts.append(1 if single else _log(rng, max(1, case["new"] // 8), case["new"]))
        lengths.append((_log(rng, max(1, case["cached"] // 100), case["cached"]) if case["cached"] else 0) + counts[-1])
    return counts, lengths


def _pool_pages(case):
    """The pages of all sequences and as many again of others."""
    return 2 * sum(-(-n // case["page"]) for n in _lengths(case)[1])


# ---- preparation -------------------------------------------------------------------------------------------------------
def _frequencies(part):
    return 10000.0 ** (-torch.arange(0, part, 2, device=DEV, dtype=torch.float32) / part)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]

    def values(*shape, spread=1.0):
        return (torch.randn(*shape, device=DEV, generator=gen) * spread).to(dtype)

    state = {"kind": case["kind"], "dtype": dtype, "d": d}
    if case["kind"] == "rotate":
        rows = case["rows"]
        state["positions"] = torch.randint(0, case["far"], (rows,), device=DEV, generator=gen)
    else:
        counts, lengths = _lengths(case)
        rows, page, pages = sum(counts), case["page"], _pool_pages(case)
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
        for i, n in enumerate(need):
            table[i, :n] = torch.tensor(order[sum(need[:i]):sum(need[:i]) + n], dtype=torch.int32)
        starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32)
        state.update(table=table.to(DEV), lengths=torch.tensor(lengths, dtype=torch.int32).to(DEV), starts=starts.to(DEV), max_new=max(counts), max_length=max(lengths))
        state["packed"] = case["ragged"] and max(counts) > 1  # equal counts need no starts
        state["k_pages"], state["v_pages"] = values(pages, hkv, page, d), values(pages, hkv, page, d)
    if case["kind"] == "attend":
        state["q"] = values(rows, hq, d, spread=2.0)
        return state
    # views of one projection's output, as a fused q/k/v Linear leaves them
    whole = values(rows, (hq + 2 * hkv) * d)
    if rows >= 8:
        whole[rows // 2, :d] = 0  # a head of padding
    state["q"], state["k"], state["v"] = (part.unflatten(1, (-1, d)) for part in whole.split([hq * d, hkv * d, hkv * d], 1))
    state["frequencies"], state["factor"], state["interleaved"] = _frequencies(case["part"]), case["factor"], case["interleaved"]
    state["q_norm"], state["k_norm"] = (((1 + 0.2 * torch.randn(d, device=DEV, generator=gen)).to(dtype)) if case["norm"] else None for _ in "qk")
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def _turned(x, norm, positions, state):
    """The heads of x [rows, heads, d], normed and turned to their rows' positions, in 32 bits (angles in 64)."""
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.float()
    angle = positions.double()[:, None, None] * state["frequencies"].double()
    cos, sin = (torch.cos(angle) * state["factor"]).float(), (torch.sin(angle) * state["factor"]).float()
    half = cos.shape[-1]
    out = x.clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if state["interleaved"] else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out.to(state["dtype"])


def _rows(state):
    """The sequence of each row and its place among the sequence's new rows."""
    row = torch.arange(state["q"].shape[0], device=DEV)
    seq = torch.bucketize(row, state["starts"][1:].long(), right=True)
    return seq, row - state["starts"].long()[seq]


def run(state):
    kind, q = state["kind"], state["q"]
    if own:
        from tensor_parallel_amd import attention, paged

        if kind == "attend":
            return paged.attend(q, state["k_pages"], state["v_pages"], state["table"], state["lengths"], starts=state["starts"] if state["packed"] else None,
                                max_new=state["max_new"], max_length=state["max_length"])
        more = {"inv_freq": state["frequencies"], "scaling": state["factor"], "interleaved": state["interleaved"], "q_norm": state["q_norm"], "k_norm": state["k_norm"], "eps": EPS}
        if kind == "rotate":
            return attention.rotate(q, state["k"], state["positions"], **more)
        q = paged.append(q, state["k"], state["v"], state["k_pages"], state["v_pages"], state["table"], state["lengths"], starts=state["starts"] if state["packed"] else None, **more)
        return q, state["k_pages"], state["v_pages"]
    if kind == "rotate":
        return _turned(q, state["q_norm"], state["positions"], state), _turned(state["k"], state["k_norm"], state["positions"], state)
    seq, place = _rows(state)
    lengths, starts, table = state["lengths"].long(), state["starts"].long(), state["table"].long()
    before = lengths - (starts[1:] - starts[:-1])
    k_pages, v_pages = state["k_pages"], state["v_pages"]
    hkv, page, d = k_pages.shape[1:]
    if kind == "append":
        position = before[seq] + place
        pages, slots = table[seq, position // page], position % page
        k_pages[pages, :, slots] = _turned(state["k"], state["k_norm"], position, state)
        v_pages[pages, :, slots] = state["v"]
        return _turned(q, state["q_norm"], position, state), k_pages, v_pages
    # rows and keys of all sequences, padded to the longest
    seqs, hq = table.shape[0], q.shape[1]
    wide = torch.zeros(seqs, state["max_new"], hq, d, device=DEV)
    wide[seq, place] = q.float() * d**-0.5
    wide = wide.view(seqs, -1, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, d)
    keys = k_pages[table.clamp_min(0)].transpose(1, 2).reshape(seqs, hkv, -1, d)[:, :, :state["max_length"]].float()
    scores = wide @ keys.transpose(2, 3).contiguous()
    del keys
    last = (before[:, None] + torch.arange(state["max_new"], device=DEV)).repeat(1, hq // hkv)[:, None, :, None]
    scores.masked_fill_(torch.arange(scores.shape[3], device=DEV) > last, -math.inf)
    scores -= scores.amax(3, keepdim=True)
    scores.exp_()
    total = scores.sum(3, keepdim=True)
    values = v_pages[table.clamp_min(0)].transpose(1, 2).reshape(seqs, hkv, -1, d)[:, :, :state["max_length"]].float()
    out = (scores @ values) / total
    return out.view(seqs, hq, -1, d).transpose(1, 2)[seq, place].to(state["dtype"])


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rotate":
        return {"bytes": case["rows"] * (4 * (hq + hkv) * d + 8), "flops": 12 * case["rows"] * (hq + hkv) * d}
    counts, lengths = _lengths(case)
    rows, more = sum(counts), 8 * len(counts) + 4 * sum(-(-n // case["page"]) for n in lengths)
    if case["kind"] == "append":
        return {"bytes": rows * 4 * (hq + 2 * hkv) * d + 8 * len(counts), "flops": 12 * rows * (hq + hkv) * d}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
    return {"bytes": 4 * rows * hq * d + 4 * sum(lengths) * hkv * d + more, "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _pairs_turned(x, weight, positions, case):
    """x [rows, heads, d] in 64 bits: pairs of elements as complex numbers, times the unit number of their angle."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    part = case["part"]
    turning, rest = x[..., :part], x[..., part:]
    pairs = turning.unflatten(-1, (-1, 2)) if case["interleaved"] else turning.unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = torch.outer(positions.double(), _frequencies(part).double())
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, case["factor"]), angle)[:, None])
    turned = turned if case["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), rest], -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotate":
        return tuple(_pairs_turned(state[name], state[name + "_norm"], state["positions"], case) for name in "qk")
    counts, lengths = _lengths(case)
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    table = state["table"].cpu().tolist()
    outs, row = [], 0
    pools = None if case["kind"] == "attend" else [state["k_pages"].double(), state["v_pages"].double()]
    for i, (n, length) in enumerate(zip(counts, lengths)):
        rows, pages = slice(row, row + n), torch.tensor(table[i][:-(-length // page)], device=DEV)
        row += n
        if case["kind"] == "append":
            at = torch.arange(length - n, length, device=DEV)
            outs.append(_pairs_turned(state["q"][rows], state["q_norm"], at, case))
            pools[0].index_put_((pages[at // page], torch.arange(hkv, device=DEV)[:, None], at % page),
                                _pairs_turned(state["k"][rows], state["k_norm"], at, case).transpose(0, 1))
            pools[1].index_put_((pages[at // page], torch.arange(hkv, device=DEV)[:, None], at % page), state["v"][rows].double().transpose(0, 1))
            continue
        out = torch.empty(n, hq, d, dtype=torch.float64, device=DEV)
        for head in range(hkv):
            k, v = (pool[pages, head].reshape(-1, d)[:length].double() for pool in (state["k_pages"], state["v_pages"]))
            for g in range(head * hq // hkv, (head + 1) * hq // hkv):
                logits = torch.mm(state["q"][rows, g].double(), k.T) / math.sqrt(d)
                unseen = torch.ones(n, length, dtype=torch.bool, device=DEV).triu(length - n + 1)
                out[:, g] = torch.mm(torch.softmax(logits.masked_fill(unseen, -math.inf), 1), v)
        outs.append(out)
    return torch.cat(outs) if pools is None else (torch.cat(outs), *pools)
