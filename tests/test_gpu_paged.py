"""Rotated and normed heads, paged caches and attention on them (`tp.attention.rotate`, `tp.paged.append`, `tp.paged.attend`) against oracle/paged.py in float64.

Tolerances. u = half a step of the dtype relative to a value (2^-8 in bf16, 2^-11 in fp16), t = 2^-25, half the smallest step of fp16.
  heads    one rounding of the exact result, and fp32 arithmetic in front of it: cos and sin within 2^-23 of their exact values (the angle is reduced in 64 bits), two products and a sum, each off by
           2^-24, and with a norm a factor off by less than 2^-16 (512 additions and the reciprocal root): u |y| + 2^-20 (|a| + |b|) + 2^-15 |y| where there is a norm + t
  attend   probabilities are rounded to the dtype, their sum is not: u sum p |v|. A score is a sum of D products off by D 2^-24 sum |q k| scale at most, twice that (its own
           and those in the denominator) moves p by that factor. The accumulation of n terms in fp32 is off by n 2^-24 of sum p |v|. In fp16 probabilities below 2^-14 of the largest are off by t
           each: n t max |v|. Then one rounding, u |o| + t."""
import ctypes
import math

import pytest
import torch

from oracle import paged as opg
from tensor_parallel_amd import _native, attention, paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16 = torch.bfloat16, torch.float16
T = 2.0**-25


def u(dtype):
    return torch.finfo(dtype).eps / 2


def bits(t):
    return t.detach().cpu().contiguous().view(torch.int16)


def close(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    both = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), both), f"{int((torch.isfinite(got) != both).sum())} values are finite on one side only"
    far = ((got - want).abs() - tol)[both]
    assert far.numel() == 0 or far.max() <= 0, f"off by {far.max():.3g} more than {tol[both][far.argmax()]:.3g}"
    assert torch.equal(got[~both].nan_to_num(7.0, 8.0, 9.0), want[~both].nan_to_num(7.0, 8.0, 9.0))


def close_heads(got, x, norm, want, part, interleaved, scaling, dtype, eps=1e-6):
    y = x.double()
    if norm is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * norm.double()
    size = y.abs()
    half = part // 2
    a, b = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, half), slice(half, part))
    pair = torch.zeros_like(size)
    pair[..., a] = pair[..., b] = (size[..., a] + size[..., b]) * abs(scaling)
    pair[..., part:] = size[..., part:]
    close(got, want, u(dtype) * want.abs() + 2.0**-20 * pair + (2.0**-15 * (want.abs() + pair) if norm is not None else 0.0) + T)


def frequencies(part, base=10000.0):
    return base ** (-torch.arange(0, part, 2, dtype=torch.float32) / max(part, 1))


# ---- heads -------------------------------------------------------------------------------------------------------------
HEADS = [
    # rows, Hq, Hkv, D, part, interleaved, norm
    (1, 16, 16, 128, 128, False, False), (5, 64, 4, 64, 32, True, False), (3, 8, 8, 96, 24, False, False), (33, 4, 2, 256, 64, True, True), (2, 32, 8, 128, 128, False, True),
    (7, 6, 3, 80, 80, False, True), (4, 3, 1, 96, 96, True, True), (2, 5, 5, 6, 4, False, True), (3, 2, 1, 2, 2, True, False), (2, 2, 2, 512, 512, False, True), (2, 1, 1, 512, 6, True, True),
    (300, 71, 1, 64, 64, False, False), (1100, 16, 16, 64, 16, False, True), (2, 4, 4, 64, 0, False, True), (2, 4, 2, 24, 0, False, False),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,Hq,Hkv,D,part,interleaved,norm", HEADS)
def test_rotate(dtype, rows, Hq, Hkv, D, part, interleaved, norm):
    g = torch.Generator().manual_seed(rows + D)
    whole = torch.randn(rows, Hq + 2 * Hkv, D, generator=g).to(dtype)  # one projection's output
    whole[0, 0] = 0
    positions = torch.randint(0, 1 << 20, (rows,), generator=g)
    positions[-1] = (1 << 31) - 5
    positions[0] = 0 if rows > 1 else 77
    weights = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in "qk"]
    inv_freq, scaling = frequencies(part), 1.25
    dev = whole.to(DEV)
    more = {"inv_freq": inv_freq.to(DEV), "positions": positions.to(DEV)} if part else {}
    got = attention.rotate(dev[:, :Hq], dev[:, Hq:Hq + Hkv], **more, scaling=scaling, interleaved=interleaved, q_norm=None if not norm else weights[0].to(DEV),
                           k_norm=None if not norm else weights[1].to(DEV))
    for x, w, y in zip((whole[:, :Hq], whole[:, Hq:Hq + Hkv]), weights, got):
        assert y.dtype == dtype and y.is_contiguous()
        close_heads(y, x, w, opg.heads(x, positions, inv_freq, scaling, interleaved, w), part, interleaved, scaling, dtype)
    if not norm and part == 0:
        assert torch.equal(bits(got[0]), bits(whole[:, :Hq]))


@pytest.mark.parametrize("table_dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("shared", [False, True])
def test_rotate_by_tables(table_dtype, shared):
    """cos and sin as a model's rotary embedding hands them over (here the first half of its columns), one row for all or a row each; heads grouped by their key/value head, rows of two axes."""
    g = torch.Generator().manual_seed(3)
    B, S, Hkv, per, D = 2, 5, 3, 4, 64
    whole = torch.randn(B, S, Hkv, per + 2, D, generator=g).to(BF16)
    angle = torch.rand(1 if shared else B, 1 if shared else S, D // 2, generator=g) * 6
    cos, sin = (torch.cat([t, t], -1).to(table_dtype) for t in (angle.cos(), angle.sin()))
    dev, c, s = whole.to(DEV), cos.to(DEV)[..., :D // 2], sin.to(DEV)[..., :D // 2]
    q, k = attention.rotate(dev[..., :per, :], dev[..., per, :], cos=c, sin=s)
    assert q.shape == (B, S, Hkv * per, D) and k.shape == (B, S, Hkv, D)
    wide = [t[..., :D // 2].expand(B, S, D // 2).reshape(-1, D // 2) for t in (cos, sin)]
    for x, y in ((whole[..., :per, :].reshape(B * S, -1, D), q), (whole[..., per, :].reshape(B * S, -1, D), k)):
        close_heads(y.reshape(B * S, -1, D), x, None, opg.turned(x.double(), *wide, False), D, False, 1.0, BF16)


def test_rotate_off_every_boundary():
    """Heads and weights that begin on odd elements, rows of odd pitch, positions of 32 bits."""
    g = torch.Generator().manual_seed(4)
    flat = torch.randn(3 * 4 * 65 + 1, generator=g).to(F16)
    x = flat[1:].as_strided((3, 4, 64), (4 * 65, 65, 1), 1)
    w = torch.randn(65, generator=g).to(F16)
    positions = torch.tensor([0, 9, 70000], dtype=torch.int32)
    dev, wd = flat.to(DEV), w.to(DEV)[1:]
    xd = dev.as_strided((3, 4, 64), (4 * 65, 65, 1), 1)
    q, k = attention.rotate(xd, xd[:, :2], positions.to(DEV), inv_freq=frequencies(64).to(DEV), q_norm=wd, k_norm=wd)
    want = opg.heads(x, positions, frequencies(64), norm=w[1:])
    close_heads(q, x, w[1:], want, 64, False, 1.0, F16)
    assert torch.equal(k, q[:, :2].contiguous())


def test_frequencies_of_a_long_context():
    """The frequencies and the factor that transformers computes for a context extended by parts, at positions up to its end."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    config = LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=1 << 17,
                         rope_parameters={"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096, "rope_theta": 10000.0})
    inv_freq, factor = ROPE_INIT_FUNCTIONS["yarn"](config, "cpu")
    g = torch.Generator().manual_seed(5)
    x, positions = torch.randn(64, 4, 128, generator=g).to(BF16), torch.randint(0, 1 << 17, (64,), generator=g)
    q, k = attention.rotate(x.to(DEV), x.to(DEV), positions.to(DEV), inv_freq=inv_freq.to(DEV), scaling=factor)
    close_heads(q, x, None, opg.heads(x, positions, inv_freq, factor), 128, False, factor, BF16)
    assert torch.equal(q, k)


def test_no_rows():
    x = torch.zeros(0, 2, 64, dtype=F16, device=DEV)
    q, k = attention.rotate(x, x, torch.zeros(0, dtype=torch.int64, device=DEV), inv_freq=frequencies(64).to(DEV))
    assert q.shape == k.shape == (0, 2, 64)


# ---- a paged batch -----------------------------------------------------------------------------------------------------
class Batch:
    """Sequences with `counts` new rows and `lengths` positions, their pages scattered over a pool whose other positions hold `rest` (NaN: nothing may read them)."""

    def __init__(self, counts, lengths, Hq, Hkv, D, page, dtype, seed, padded=0, behind=0, rest=math.nan, spread=1.0, swapped=False):
        g = torch.Generator().manual_seed(seed)
        self.g, self.counts, self.lengths, self.dtype, self.page = g, counts, lengths, dtype, page
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + 3
        order = torch.randperm(self.pages, generator=g).tolist()
        self.columns = max(need + [1]) + 1
        self.table = [order[sum(need[:b]):sum(need[:b + 1])] + [-1] * (self.columns - n) for b, n in enumerate(need)]
        self.starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
        self.rows = padded * len(counts) if padded else sum(counts) + behind
        self.padded = padded
        self.seqs = opg.rows_of(self.rows, lengths, None if padded else self.starts, counts if padded else None)
        self.k, self.v = (torch.full((self.pages, Hkv, page, D), rest).to(dtype) for _ in "kv")
        for pool, s in ((self.k, spread), (self.v, 1.0)):
            for b, n in enumerate(lengths):
                for j in range(0, n, page):
                    m = min(page, n - j)
                    pool[self.table[b][j // page], :, :m] = (torch.randn(Hkv, m, D, generator=g) * s).to(dtype)
        self.q = torch.randn(self.rows, Hq, D, generator=g).to(dtype)
        self.swapped = swapped  # pools as [pages, positions, heads, D]

    def on(self, device=DEV):
        d = {"k_pages": self.k, "v_pages": self.v}
        d = {n: (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) if self.swapped else t.to(device)) for n, t in d.items()}
        d["table"] = torch.tensor(self.table, dtype=torch.int32).reshape(len(self.counts), self.columns).to(device)
        d["lengths"] = torch.tensor(self.lengths, dtype=torch.int32).to(device)
        name, values = ("counts", self.counts) if self.padded else ("starts", self.starts)
        d[name] = torch.tensor(values, dtype=torch.int32).to(device)
        return d

    def want(self, scale):
        return opg.attend(self.q, self.k, self.v, self.table, self.seqs, scale)

    def tolerance(self, want, weight, scale):
        n, D = max(self.lengths + [1]), self.q.shape[2]
        kmax = torch.nan_to_num(self.k.double(), 0.0, 0.0, 0.0).abs().amax()
        score = D * 2.0**-24 * D * float(self.q.double().abs().amax() * kmax) * abs(scale)
        vmax = float(torch.nan_to_num(self.v.double(), 0.0, 0.0, 0.0).abs().amax())
        return (u(self.dtype) * 1.01 + 2 * score + n * 2.0**-24) * weight + (n * T * vmax if self.dtype == F16 else 0.0) + u(self.dtype) * want.abs() + T


def check_attend(batch, scale=None, **more):
    D = batch.q.shape[2]
    real = D**-0.5 if scale is None else scale
    got = torch.full((batch.rows, *batch.q.shape[1:]), 3.0, dtype=batch.dtype, device=DEV)
    y = paged.attend(batch.q.to(DEV), **batch.on(), scale=scale, out=got, **more)
    assert y is got
    want, weight = batch.want(real)
    mine = torch.zeros(batch.rows, dtype=torch.bool)
    for first, n, _ in batch.seqs:
        mine[first:first + n] = True
    assert (got[~mine.to(DEV)] == 3).all()  # rows of no sequence are left as they were
    close(got[mine.to(DEV)], want[mine], batch.tolerance(want, weight, real)[mine])
    return got


FEW = [
    # counts, lengths, Hq, Hkv, D, page
    ([1], [1], 1, 1, 64, 16), ([1], [500], 16, 16, 128, 16), ([1, 1, 1], [1, 16, 17], 4, 2, 128, 16), ([1] * 5, [63, 64, 65, 128, 1000], 32, 2, 64, 32),
    ([1, 1], [5000, 3], 8, 8, 96, 64), ([1, 1], [700, 2049], 4, 1, 256, 256), ([3, 1, 2], [3, 40, 641], 10, 2, 128, 16), ([4, 4], [4, 90], 4, 1, 64, 128), ([16], [100], 2, 2, 128, 16),
    ([0, 1, 0, 1], [77, 31, 0, 65], 8, 4, 64, 16), ([1], [9000], 16, 1, 64, 16), ([1], [20000], 2, 2, 128, 64), ([2, 3], [1, 0], 4, 2, 96, 16), ([8] * 3, [8, 64, 300], 2, 1, 256, 32),
]
MANY = [
    ([17], [17], 1, 1, 64, 16), ([64], [64], 4, 4, 128, 64), ([300], [300], 2, 1, 128, 16), ([129, 40], [700, 41], 6, 2, 96, 32), ([70], [1070], 8, 2, 256, 64), ([1, 1], [9, 130], 71, 1, 64, 16),
    ([1], [3000], 40, 2, 128, 128), ([257], [257], 1, 1, 64, 256), ([33, 0, 90], [33, 50, 400], 16, 1, 64, 16), ([130], [5130], 4, 4, 128, 16), ([40], [25], 2, 2, 64, 16), ([600], [601], 3, 1, 96, 64),
]
MIXED = [
    ([1, 100, 1, 3, 0, 40], [700, 100, 1, 64, 5, 4040], 8, 2, 128, 16), ([60, 1, 1], [60, 3000, 2], 16, 4, 64, 64), ([9, 1], [200, 33], 4, 2, 256, 32), ([30, 2, 1], [31, 20, 500], 8, 4, 96, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,Hq,Hkv,D,page", FEW + MANY + MIXED)
def test_attend(dtype, counts, lengths, Hq, Hkv, D, page):
    batch = Batch(counts, lengths, Hq, Hkv, D, page, dtype, seed=sum(lengths) + D, behind=2)
    check_attend(batch)                                                                # neither bound known
    check_attend(batch, max_new=max(counts), max_length=max(lengths))


@pytest.mark.parametrize("counts,lengths,Hq,Hkv,D,page", [FEW[3], FEW[6], MANY[3], MIXED[0], MIXED[2]])
def test_attend_on_padded_rows_and_pools_of_another_order(counts, lengths, Hq, Hkv, D, page):
    check_attend(Batch(counts, lengths, Hq, Hkv, D, page, BF16, seed=7, padded=max(counts) + 3, swapped=True))
    check_attend(Batch(counts, lengths, Hq, Hkv, D, page, F16, seed=8, padded=max(counts), spread=3.0), max_new=max(counts))


@pytest.mark.parametrize("seqs,new,Hq,Hkv,D", [(130, 1, 4, 2, 64), (300, 1, 8, 8, 128), (70, 20, 2, 1, 64), (1, 64, 4, 1, 128), (3, 5, 2, 2, 96)])
def test_attend_without_starts(seqs, new, Hq, Hkv, D):
    """All rows new, as many for each sequence; more sequences than a wavefront scans at a time."""
    lengths = [new + (37 * b) % 411 for b in range(seqs)]
    batch = Batch([new] * seqs, lengths, Hq, Hkv, D, 16, BF16, seed=seqs)
    d = batch.on()
    d.pop("starts")
    want, weight = batch.want(D**-0.5)
    got = paged.attend(batch.q.to(DEV).view(seqs, new, Hq, D), **d, max_new=new)
    assert got.shape == (seqs, new, Hq, D)
    close(got.view(-1, Hq, D), want, batch.tolerance(want, weight, D**-0.5))
    d["starts"] = torch.tensor(batch.starts, dtype=torch.int32, device=DEV)
    close(paged.attend(batch.q.to(DEV), **d), want, batch.tolerance(want, weight, D**-0.5))


@pytest.mark.parametrize("counts,lengths", [([1], [300]), ([3], [130]), ([40], [200])])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(counts, lengths, scale):
    check_attend(Batch(counts, lengths, 4, 2, 64, 16, BF16, seed=11), scale=scale)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([1, 4], [70, 133]), ([50, 40], [50, 161])])
def test_values_that_are_not_finite(counts, lengths, D):
    """Infinities and NaN reach the rows that see them, in their columns, and no other; scores that are not finite likewise. (Equal scores: every probability above zero.)"""
    batch = Batch(counts, lengths, 4, 2, D, 16, BF16, seed=12, spread=0.0)
    b, n = 1, lengths[1]
    for back, column, value in ((2, 3, math.inf), (1, 5, -math.inf), (3, 7, math.nan), (0, 11, math.inf), (counts[1] + 1, 13, -math.inf)):
        j = n - 1 - back
        batch.v[batch.table[b][j // 16], :, j % 16, column] = value
    check_attend(batch)
    j = n - 1
    batch.k[batch.table[b][j // 16], :, j % 16, 0] = math.nan  # a key that only the last row sees
    got = paged.attend(batch.q.to(DEV), **batch.on())
    assert got[-1].isnan().all() and not got[:-1, :, 20:].isnan().any()


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([1, 4], [70, 133]), ([50, 40], [50, 161])])
def test_values_that_are_not_finite_in_half_precision(counts, lengths, D):
    batch = Batch(counts, lengths, 4, 2, D, 16, F16, seed=15, spread=0.0)
    b, n = 1, lengths[1]
    for back, column, value in ((2, 3, math.inf), (1, 5, -math.inf), (3, 7, math.nan), (0, 11, math.inf), (2, 11, -math.inf), (counts[1] + 1, 13, -math.inf)):
        j = n - 1 - back
        batch.v[batch.table[b][j // 16], :, j % 16, column] = value
    check_attend(batch)


@pytest.mark.parametrize("max_length", [None, 1, 4040, 1 << 20])
@pytest.mark.parametrize("counts,lengths,Hq,Hkv,D,page", [MIXED[0], MIXED[1], FEW[3], MANY[3],
                                                          ([1] * 70 + [40] + [2] * 20 + [64, 1], [33] * 70 + [3100] + [70] * 20 + [1500, 900], 4, 2, 64, 16)])
def test_bounds_change_nothing_but_the_time(counts, lengths, Hq, Hkv, D, page, max_length):
    """Whatever max_length says (of a captured call, what it said then); max_new as it is."""
    check_attend(Batch(counts, lengths, Hq, Hkv, D, page, BF16, seed=16, behind=2), max_length=max_length, max_new=max(counts))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("counts,lengths,max_length", [([1], [257], 257), ([1, 3, 2, 0], [260, 700, 13, 9], 700), ([4, 2, 1], [4, 2, 600], 700), ([1], [5], 500), ([3, 1], [1, 0], 300)])
def test_short_steps_in_wide_blocks(dtype, D, counts, lengths, max_length):
    """Few items of a few hundred positions: wavefronts without any, and those whose last positions some rows do not see."""
    check_attend(Batch(counts, lengths, 4, 2, D, 16, dtype, seed=17, behind=1), max_length=max_length, max_new=max(counts))
    batch = Batch(counts, lengths, 4, 2, D, 16, dtype, seed=18, spread=0.0)
    b = max(range(len(lengths)), key=lambda i: lengths[i])
    for back, column, value in ((0, 3, math.inf), (1, 5, math.nan), (2, 7, -math.inf)):
        j = lengths[b] - 1 - back
        if j >= 0:
            batch.v[batch.table[b][j // 16], :, j % 16, column] = value
    check_attend(batch, max_length=max_length, max_new=max(counts))


def test_pages_that_the_pool_does_not_have_hold_zeros():
    for counts, lengths in (([1, 2], [100, 90]), ([40, 1], [100, 90])):
        batch = Batch(counts, lengths, 4, 2, 64, 16, F16, seed=13)
        batch.table[0][2], batch.table[1][0], batch.table[1][5] = -1, batch.pages, 1 << 30
        check_attend(batch)


def test_lengths_beyond_the_table_and_rows_beyond_the_batch_stay_in_bounds():
    """Inputs that cannot be checked without reading them back are held to what there is."""
    for counts, lengths in (([1, 2], [100, 90]), ([40, 1], [100, 90])):
        batch = Batch(counts, lengths, 4, 2, 64, 16, F16, seed=14, rest=0.0)
        d = batch.on()
        d["lengths"] = torch.tensor([1 << 30, -5], dtype=torch.int32, device=DEV)
        d["starts"] = torch.tensor([-7, batch.rows + 50, 3], dtype=torch.int32, device=DEV)
        q = batch.q.to(DEV)
        out = paged.attend(q, **d)
        paged.append(q, q[:, :2], q[:, :2], **d)
        torch.cuda.synchronize()
        assert out.shape == q.shape


# ---- append ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,Hq,Hkv,D,page,part,interleaved,norm,padded", [
    ([1], [1], 2, 2, 64, 16, 64, False, False, 0), ([1, 1, 1], [17, 16, 300], 8, 2, 128, 16, 128, False, True, 0), ([5, 0, 33], [5, 9, 70], 4, 4, 96, 32, 24, True, False, 0),
    ([3, 7, 1], [3, 20, 65], 6, 3, 64, 64, 32, False, True, 9), ([2, 2], [1, 40], 4, 1, 256, 128, 0, False, False, 0), ([20], [20], 2, 1, 80, 16, 20, True, True, 0), ([1] * 140, [3] * 140, 2, 1, 64, 16, 64, False, False, 0),
])
def test_append(dtype, counts, lengths, Hq, Hkv, D, page, part, interleaved, norm, padded):
    batch = Batch(counts, lengths, Hq, Hkv, D, page, dtype, seed=D + part, padded=padded, behind=0 if padded else 3, rest=2.0, swapped=padded > 0)
    g = torch.Generator().manual_seed(1)
    whole = torch.randn(batch.rows, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    q, k, v = (t.unflatten(1, (-1, D)) for t in whole.split([Hq * D, Hkv * D, Hkv * D], 1))
    weights = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in "qk"]
    inv_freq = frequencies(part)
    dev, d = whole.to(DEV), batch.on()
    qd, kd, vd = (t.unflatten(1, (-1, D)) for t in dev.split([Hq * D, Hkv * D, Hkv * D], 1))
    got = paged.append(qd, kd, vd, **d, inv_freq=inv_freq.to(DEV) if part else None, interleaved=interleaved, q_norm=None if not norm else weights[0].to(DEV),
                       k_norm=None if not norm else weights[1].to(DEV), scaling=0.9 if part else 1.0)
    kp, vp = d["k_pages"].cpu(), d["v_pages"].cpu()
    want_k, want_v, written = batch.k.clone(), batch.v.clone(), torch.zeros(batch.pages, page, dtype=torch.bool)
    factor = 0.9 if part else 1.0
    for b, (first, n, length) in enumerate(batch.seqs):
        at = torch.arange(length - n, length)
        rows = slice(first, first + n)
        if n == 0:
            continue
        close_heads(got[rows], q[rows], weights[0], opg.heads(q[rows], at, inv_freq, factor, interleaved, weights[0]), part, interleaved, factor, dtype)
        turned = opg.heads(k[rows], at, inv_freq, factor, interleaved, weights[1])
        for i, j in enumerate(at.tolist()):
            if j < 0:
                continue
            p, s = batch.table[b][j // page], j % page
            written[p, s] = True
            close_heads(kp[p, :, s][None], k[first + i][None], weights[1], turned[i][None], part, interleaved, factor, dtype)
            assert torch.equal(bits(vp[p, :, s]), bits(v[first + i]))
    keep = ~written[:, None, :, None].expand_as(kp)
    assert torch.equal(kp[keep], want_k[keep]) and torch.equal(vp[keep], want_v[keep])  # nothing else of the pools


def test_append_at_positions_of_the_callers_and_to_pages_that_are_not_there():
    batch = Batch([2, 3], [18, 40], 2, 2, 64, 16, BF16, seed=2, rest=1.0)
    batch.table[0][1], batch.table[1][2] = -1, batch.pages  # where the new rows of both go
    d = batch.on()
    x = batch.q.to(DEV)
    positions = torch.tensor([5, 1000, 7, 3, 123456])
    got = paged.append(x, x, x, **d, positions=positions.to(DEV), inv_freq=frequencies(64).to(DEV))
    close_heads(got, batch.q, None, opg.heads(batch.q, positions, frequencies(64)), 64, False, 1.0, BF16)
    kp, vp = d["k_pages"].cpu(), d["v_pages"].cpu()
    at = batch.table[0][0], batch.table[1][1]
    assert torch.equal(kp, batch.k) and torch.equal(vp, batch.v), at


def test_positions_behind_four_gigabytes():
    """Offsets into pools pass 32 bits: elements, and bytes of one page's distance."""
    Hkv, page, D = 4, 64, 128
    pages = (5 << 30) // (Hkv * page * D * 2)
    k, v = (torch.zeros(pages, Hkv, page, D, dtype=BF16, device=DEV) for _ in "kv")
    g = torch.Generator().manual_seed(3)
    for counts, lengths, Hq in (([1, 1], [100, 64], 8), ([40, 30], [100, 64], 4)):
        batch = Batch(counts, lengths, Hq, Hkv, D, page, BF16, seed=4)
        where = [pages - 1, pages - 2, pages - 3, 0, 1, pages // 2][:batch.pages] + list(range(3, batch.pages))
        d = batch.on()
        for old, new in enumerate(where[:batch.pages]):
            k[new], v[new] = d["k_pages"][old], d["v_pages"][old]
        table = torch.tensor([[where[p] if p >= 0 else -1 for p in row] for row in batch.table], dtype=torch.int32, device=DEV)
        q = batch.q.to(DEV)
        want, weight = batch.want(D**-0.5)
        close(paged.attend(q, k, v, table, d["lengths"], starts=d["starts"]), want, batch.tolerance(want, weight, D**-0.5))
        new = torch.randn(batch.rows, Hkv, D, generator=g).to(BF16).to(DEV)
        paged.append(q, new, new, k, v, table, d["lengths"], starts=d["starts"])
        for b, (first, n, length) in enumerate(batch.seqs):
            last = table[b, (length - 1) // page].item()
            assert torch.equal(k[last, :, (length - 1) % page], new[first + n - 1]) and torch.equal(v[last, :, (length - 1) % page], new[first + n - 1])


# ---- together, streams and graphs --------------------------------------------------------------------------------------
def test_prompts_then_steps_are_attention_on_contiguous_caches():
    """Prompts in two chunks and single rows behind them, appended and attended to, against the contiguous rotation and attention of the library on each sequence alone."""
    g = torch.Generator().manual_seed(5)
    Hq, Hkv, D, page, lengths = 8, 2, 128, 16, [0, 0, 0]
    chunks = [[40, 7, 100], [33, 1, 5], [1, 1, 1], [1, 0, 1], [1, 1, 1]]
    table = torch.randperm(60, generator=g)[:3 * 12].view(3, 12).to(torch.int32).to(DEV)
    k_pages, v_pages = (torch.full((60, Hkv, page, D), math.nan, dtype=F16, device=DEV) for _ in "kv")
    inv_freq = frequencies(D).to(DEV)
    keys, values = [torch.zeros(1, Hkv, 0, D, dtype=F16, device=DEV) for _ in range(3)], [torch.zeros(1, Hkv, 0, D, dtype=F16, device=DEV) for _ in range(3)]
    for counts in chunks:
        rows = sum(counts)
        whole = torch.randn(rows, Hq + 2 * Hkv, D, generator=g).to(F16).to(DEV)
        q, k, v = whole[:, :Hq], whole[:, Hq:Hq + Hkv], whole[:, Hq + Hkv:]
        lengths = [n + c for n, c in zip(lengths, counts)]
        plan = {"table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV),
                "starts": torch.tensor([sum(counts[:b]) for b in range(4)], dtype=torch.int32, device=DEV)}
        turned = paged.append(q, k, v, k_pages, v_pages, **plan, inv_freq=inv_freq)
        got = paged.attend(turned, k_pages, v_pages, **plan, max_new=max(counts), max_length=max(lengths))
        row = 0
        for b, n in enumerate(counts):
            at = slice(row, row + n)
            row += n
            if n == 0:
                continue
            positions = torch.arange(lengths[b] - n, lengths[b], device=DEV)
            qr, kr = attention.rotate(q[at], k[at], positions, inv_freq=inv_freq)
            assert torch.equal(qr, turned[at])
            keys[b], values[b] = torch.cat([keys[b], kr.transpose(0, 1)[None]], 2), torch.cat([values[b], v[at].transpose(0, 1)[None]], 2)
            want = _native.attention(qr.transpose(0, 1)[None], keys[b], values[b])[0]
            # both sides round probabilities (u of sum p |v|, at most u max |v|) and results
            tol = 4 * u(F16) * float(values[b].abs().max())
            assert (got[at].double() - want.double()).abs().max() <= tol


@pytest.mark.parametrize("counts,lengths,Hq,Hkv", [([1] * 4, [30, 700, 64, 3], 8, 2), ([40, 1, 3, 60], [40, 900, 65, 200], 8, 2)])
def test_a_captured_step_serves_others(counts, lengths, Hq, Hkv):
    """A captured append and attend, replayed with other lengths, tables and values, is each time what the eager calls give, bit for bit."""
    D, page = 64, 16
    batch = Batch(counts, lengths, Hq, Hkv, D, page, BF16, seed=6, rest=0.0)
    d = batch.on()
    # every place of the table has a page of its own, so that no two rows are written to one place whichever way the table is turned
    n = d["table"].numel()
    d["table"] = torch.randperm(n, generator=batch.g).to(torch.int32).view_as(d["table"]).to(DEV)
    d["k_pages"], d["v_pages"] = (torch.randn(n, Hkv, page, D, device=DEV).to(BF16) for _ in "kv")
    q, k = batch.q.to(DEV), torch.randn(batch.rows, Hkv, D, device=DEV).to(BF16)
    inv_freq = frequencies(D).to(DEV)

    def step():
        turned = paged.append(q, k, k, **d, inv_freq=inv_freq)
        return paged.attend(turned, **d, max_new=max(counts))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for turn in range(4):
        with torch.no_grad():
            q.normal_()
            k.normal_()
            d["lengths"].copy_(torch.tensor([max(c, (n * (turn + 2)) // (turn + 3)) for c, n in zip(counts, lengths)], dtype=torch.int32))
            if turn % 2:
                d["table"].copy_(d["table"].flip(1).contiguous())
        kept = {n: d[n].clone() for n in ("k_pages", "v_pages")}
        graph.replay()
        torch.cuda.synchronize()
        first, pools = out.clone(), {n: d[n].clone() for n in kept}
        for n in kept:
            d[n].copy_(kept[n])
        eager = step()
        assert torch.equal(eager, first) and all(torch.equal(pools[n], d[n]) for n in kept)


def test_two_streams_and_graphs_that_run_at_once():
    """Calls on two streams, and replays of two graphs on them, do not share partial results."""
    sides = []
    for seed in range(2):
        batch = Batch([1] * 3, [9000, 300, 5000], 8, 1, 128, 16, BF16, seed=20 + seed)
        d, q = batch.on(), batch.q.to(DEV)
        want, weight = batch.want(128**-0.5)
        sides.append((d, q, want, batch.tolerance(want, weight, 128**-0.5), torch.cuda.Stream(), torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (d, q, _, _, stream, _) in enumerate(sides):
            with torch.cuda.stream(stream):
                outs[i].append(paged.attend(q, **d, max_new=1))
    torch.cuda.synchronize()
    for i, (_, _, want, tol, _, _) in enumerate(sides):
        for out in outs[i]:
            close(out, want, tol)
    held = []
    for d, q, _, _, stream, graph in sides:
        with torch.cuda.graph(graph, stream=stream):
            held.append(paged.attend(q, **d, max_new=1))
    for _ in range(3):
        for (_, _, _, _, stream, graph), out in zip(sides, held):
            out.zero_()
        torch.cuda.synchronize()
        for _, _, _, _, stream, graph in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, want, tol, _, _), out in zip(sides, held):
            close(out, want, tol)


def test_results_do_not_change_from_run_to_run():
    batch = Batch([1, 50, 1, 1], [9000, 4000, 70, 2000], 8, 2, 128, 16, BF16, seed=30)
    d, q = batch.on(), batch.q.to(DEV)
    first = paged.attend(q, **d)
    for _ in range(5):
        assert torch.equal(paged.attend(q, **d), first)


def test_no_backward():
    batch = Batch([1], [20], 2, 2, 64, 16, F16, seed=31)
    d, q = batch.on(), batch.q.to(DEV).requires_grad_()
    for out in (paged.attend(q, **d), paged.append(q, q.detach(), q.detach(), **d), attention.rotate(q, q.detach())[0]):
        with pytest.raises(Exception, match="backward"):
            out.float().sum().backward()


def test_no_backward_to_norms_tables_and_pools():
    """What is learned beside q, k and v gets no gradient in silence either."""
    batch = Batch([1, 2], [20, 9], 2, 2, 64, 16, F16, seed=33)
    d, q = batch.on(), batch.q.to(DEV)
    positions = torch.arange(batch.rows, device=DEV)

    def learned(*shape, dtype=F16):
        return torch.ones(*shape, dtype=dtype, device=DEV, requires_grad=True)

    calls = [lambda: paged.append(q, q, q, **d, q_norm=learned(64)), lambda: paged.append(q, q, q, **d, k_norm=learned(64)), lambda: paged.append(q, q, q, **d, inv_freq=learned(32, dtype=torch.float32)),
             lambda: paged.append(q, q, q, **d, cos=learned(batch.rows, 32), sin=learned(batch.rows, 32)), lambda: paged.attend(q, **{**d, "k_pages": d["k_pages"].clone().requires_grad_()}),
             lambda: paged.attend(q, **{**d, "v_pages": d["v_pages"].clone().requires_grad_()}), lambda: attention.rotate(q, q, positions, inv_freq=learned(32, dtype=torch.float32))[0],
             lambda: attention.rotate(q, q, positions, inv_freq=learned(32, dtype=torch.float32))[1], lambda: attention.rotate(q, q, cos=learned(batch.rows, 32), sin=learned(batch.rows, 32))[1]]
    for call in calls:
        out = call()
        assert out.requires_grad
        with pytest.raises(NotImplementedError, match="backward"):
            out.float().sum().backward()
        with torch.no_grad():
            assert not call().requires_grad


def test_short_of_workspace_is_refused():
    batch = Batch([1], [20000], 2, 2, 64, 16, F16, seed=32)
    d, q = batch.on(), batch.q.to(DEV)
    packed, keep = _native._pages("attend", q, 0, 2, 64, d["k_pages"], d["v_pages"], d["table"], d["lengths"], d["starts"], None)
    need = ctypes.c_uint64()
    assert _native.lib().tpamd_attention_paged_workspace(packed, 1, 2, 2, 64, 1, 20000, ctypes.byref(need)) == 0 and need.value > 0
    out = torch.empty_like(q)
    rc = _native.lib().tpamd_attention_paged(q.data_ptr(), 128, 64, packed, out.data_ptr(), 128, 64, 1, 2, 2, 64, 1, 20000, 0.1, _native.F16, q.data_ptr(), need.value - 1,
                                             _native.current_stream_ptr(DEV))
    assert rc == -1 and b"workspace" in _native.lib().tpamd_last_error()
