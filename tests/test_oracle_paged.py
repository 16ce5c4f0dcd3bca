"""What pins oracle/paged.py: library routines, the contiguous attention oracle, and invariants."""
import math

import pytest
import torch

from oracle import attention as oat
from oracle import paged as opg


def test_half_layout_is_transformers_rotation():
    from transformers.models.llama.modeling_llama import apply_rotary_pos_emb

    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 3, 16, generator=g, dtype=torch.float64)
    positions, inv_freq = torch.randint(0, 10000, (7,), generator=g), 10000.0 ** (-torch.arange(0, 16, 2).double() / 16)
    angle = torch.outer(positions.double(), inv_freq)
    cos, sin = torch.cat([angle, angle], -1).cos()[None], torch.cat([angle, angle], -1).sin()[None]
    want, _ = apply_rotary_pos_emb(x.transpose(0, 1)[None], x.transpose(0, 1)[None], cos, sin)
    assert torch.allclose(opg.heads(x, positions, inv_freq), want[0].transpose(0, 1), rtol=0, atol=1e-12)


def test_neighbours_are_complex_numbers_and_the_rest_stays():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 2, 24, generator=g, dtype=torch.float64)
    positions, inv_freq = torch.arange(5) * 1000003, torch.rand(4, generator=g, dtype=torch.float64)
    got = opg.heads(x, positions, inv_freq, scaling=1.5, interleaved=True)
    angle = torch.outer(positions.double(), inv_freq)
    want = torch.view_as_real(torch.view_as_complex(x[..., :8].unflatten(-1, (4, 2)).contiguous()) * torch.polar(torch.full_like(angle, 1.5), angle)[:, None]).flatten(-2)
    assert torch.allclose(got[..., :8], want, rtol=0, atol=1e-12) and torch.equal(got[..., 8:], x[..., 8:])


def test_norm_and_what_a_rotation_keeps():
    x, w = torch.randn(3, 2, 16, dtype=torch.float64), torch.ones(16)
    got = opg.heads(x, torch.arange(3), torch.rand(8), norm=w, eps=0.0)
    assert torch.allclose(got.square().mean(-1), torch.ones(3, 2, dtype=torch.float64))
    assert torch.equal(opg.heads(x, torch.zeros(3), torch.rand(8)), x)


@pytest.mark.parametrize("page", [16, 64])
def test_attend_on_pages_is_the_contiguous_attention(page):
    g = torch.Generator().manual_seed(2)
    B, Hq, Hkv, D, n, length = 2, 4, 2, 8, 3, 37
    q, k, v = (torch.randn(B, h, s, D, generator=g) for h, s in ((Hq, n), (Hkv, length), (Hkv, length)))
    want = oat.attention_f64(q.numpy(), k.numpy(), v.numpy(), 0.3, True)  # [B, n, Hq, D]
    per = -(-length // page)
    order = torch.randperm(B * per + 1, generator=g)[:B * per].view(B, per).tolist()
    pools = []
    for t in (k, v):
        pool = torch.full((B * per + 1, Hkv, page, D), math.nan)
        for b in range(B):
            for j in range(length):
                pool[order[b][j // page], :, j % page] = t[b, :, j]
        pools.append(pool)
    rows = q.permute(0, 2, 1, 3).reshape(B * n, Hq, D)
    got, _ = opg.attend(rows, *pools, order, opg.rows_of(B * n, [length] * B), 0.3)
    assert torch.allclose(got, torch.as_tensor(want).reshape(B * n, Hq, D).double(), rtol=0, atol=1e-12)


def test_rows_that_see_nothing_and_rows_of_no_sequence():
    pool = torch.randn(1, 1, 16, 4)
    out, _ = opg.attend(torch.randn(5, 1, 4), pool, pool, [[0]], [(1, 3, 2)], 1.0)
    assert out[1].abs().sum() == 0 and torch.allclose(out[2], pool[0, :, 0].double()) and out[0].isnan().all() and out[4].isnan().all()
