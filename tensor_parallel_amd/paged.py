"""Key/value caches whose positions lie in pages, for batches of sequences that differ in length.

The reference leaves caches to the wrapped model and only routes them between ranks (src/tensor_parallel/aux_actions.py:7-15, src/tensor_parallel/slicing_configs.py:440,446). A
server's sequences come and go and differ in length, so here a rank's keys and values of a layer may lie in a pool of pages, k_pages and v_pages [pages, Hkv, page, D] (any strides, D
contiguous; `page` positions, a power of two from 16 on), and position j of sequence b in slot j % page of page table[b, j // page]. `lengths` count a sequence's positions with the
new rows of the call, which are its last ones. The new rows of all sequences follow one another on the rows' axis:

  starts                the rows of sequence b are starts[b] ... starts[b + 1] - 1 (packed; rows behind starts[-1] are left alone)
  counts                each sequence has as many rows as any other, the first counts[b] of which are new (padded on the right)
  neither               all of them are new

table, lengths, starts and counts are int32 tensors on the device. The kernels read them when they run, so a call that was captured into a HIP graph serves every step; nothing is read
back. A page outside of the pool (-1, say) holds zeros and takes nothing.

  append(...)   rotates q and k (and norms their heads before, where weights are given) and writes k and v to their pages; returns q          tpamd_append_paged
  attend(...)   softmax(scale q k^T) v of the new rows, each on the positions up to its own                                                  tpamd_attention_paged

Two calls that write to the same pages, or one that reads what another writes, are the caller's to order, as for any two kernels (calls on one stream are). Inference only: a backward
pass through either raises.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .shard_modules import _guard


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
           starts: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
           cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, scaling: float = 1.0, interleaved: bool = False, q_norm: Optional[torch.Tensor] = None,
           k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """The new rows q [..., Hq, D] (or [..., Hkv, Hq / Hkv, D]), k and v [..., Hkv, D], views of projection outputs: k and v go to their positions' pages, k and q rotated as
    `attention.rotate` does (frequencies or tables; neither: as they are). A row is rotated to its place in its sequence, or to `positions` [...]. Returns q as [..., Hq, D]; rows of no
    sequence are left as the memory was."""
    return _guard(_native.append_paged(q, k, v, k_pages, v_pages, table, lengths, starts, counts, positions, inv_freq, cos, sin, scaling, interleaved, q_norm, k_norm, eps), q, k, v)


def attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, starts: Optional[torch.Tensor] = None,
           counts: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_new: Optional[int] = None, max_length: Optional[int] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new rows q [..., Hq, D] on their sequences' pages (which hold the new rows' keys and values already): [..., Hq, D], `out` if it is given. Hq a multiple of
    Hkv, D 64, 96, 128 or 256; scale D ** -0.5 by default. Rows of no sequence are left as the memory was, a row in front of position 0 (more new rows than positions) is zeros.

    max_new: no sequence has more new rows (rows of one that does may be left out); tell it where it is known, a step of single rows is then one or two launches. max_length: no sequence
    has more positions; only the time depends on it. Both have to hold for every replay where the call is captured."""
    return _guard(_native.attention_paged(q, k_pages, v_pages, table, lengths, starts, counts, scale, max_new, max_length, out), q)
