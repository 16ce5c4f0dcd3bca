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

  PagedCache    pools, page table and lengths of a wrapped model's layers: handed to a model as `past_key_values` once `attention.fuse_rotary_` has given its attention modules their
                fused forward, on one rank or on several

Two calls that write to the same pages, or one that reads what another writes, are the caller's to order, as for any two kernels (calls on one stream are). Inference only: a backward
pass through either raises.
"""
from __future__ import annotations

import copy
import operator
import threading
from typing import Dict, List, Optional, Sequence, Set, Tuple

import torch

from . import _native, kv_cache
from .shard_modules import _guard


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
           starts: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
           cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, scaling: float = 1.0, interleaved: bool = False, q_norm: Optional[torch.Tensor] = None,
           k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """The new rows q [..., Hq, D] (or [..., Hkv, Hq / Hkv, D]), k and v [..., Hkv, D], views of projection outputs: k and v go to their positions' pages, k and q rotated as
    `attention.rotate` does (frequencies or tables; neither: as they are). By frequencies a row is rotated to its place in its sequence, or to
    `positions` [...]; tables have its position in them, and positions beside them are refused. Returns q as [..., Hq, D]; rows of no
    sequence are left as the memory was."""
    return _guard(_native.append_paged(q, k, v, k_pages, v_pages, table, lengths, starts, counts, positions, inv_freq, cos, sin, scaling, interleaved, q_norm, k_norm, eps), q, k, v,
                  q_norm, k_norm, inv_freq, cos, sin)


def attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, starts: Optional[torch.Tensor] = None,
           counts: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_new: Optional[int] = None, max_length: Optional[int] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new rows q [..., Hq, D] on their sequences' pages (which hold the new rows' keys and values already): [..., Hq, D], `out` if it is given (which overlaps no
    operand). Hq a multiple of Hkv, D 64, 96, 128 or 256, rows of q and of the pools on 16-byte boundaries (others are refused); scale D ** -0.5 by default. Rows of no
    sequence are left as the memory was, a row in front of position 0 (more new rows than positions) is zeros, one whose scores all are -inf is NaN. What stands at positions that a row does not see does
    not reach it; an infinite value that it sees gives it that infinity, or NaN where its probability is too small for the dtype. Probabilities are rounded to the dtype in front of the product with v,
    sums are in 32 bits.

    max_new: no sequence has more new rows (rows of one that does may be left out); tell it where it is known, a step of single rows is then one or two launches. max_length: no sequence
    has more positions; only the time depends on it. Both have to hold for every replay where the call is captured."""
    return _guard(_native.attention_paged(q, k_pages, v_pages, table, lengths, starts, counts, scale, max_new, max_length, out), q, k_pages, v_pages)


def _capturing(t: torch.Tensor) -> bool:
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class _Book:
    """What the caches of all ranks and layers have in common: which pages each sequence has, how many positions, and the rows of the step that is on its way."""

    def __init__(self, sequences: int, pages: int, page: int, columns: int):
        self.sequences, self.pages, self.page, self.columns = sequences, pages, page, columns
        self.states: Dict[torch.device, torch.Tensor] = {}
        self.uploaded: Dict[torch.device, int] = {}  # the version of it that is there
        self.lock = threading.Lock()  # ranks on different devices are threads
        self.captured: Set[int] = set()  # rows (of each sequence) of the forwards that were captured
        self.number = self.version = 0  # of the step and of what devices are told, never given twice
        self.reset()

    def reset(self) -> None:
        self.free: List[int] = list(range(self.pages - 1, -1, -1))
        self.tables: List[List[int]] = [[] for _ in range(self.sequences)]
        self.before = [0] * self.sequences  # positions without the step's rows
        self.end()

    def end(self) -> None:
        """No step is on its way: the next forward, of whichever rank, begins another, and replays have no new rows."""
        self.counts = [0] * self.sequences  # the step's rows
        self.taken, self.hold, self.over = True, False, True  # whether a forward has begun the step; whether further forwards are the same step; whether it has ended for all
        self.rows: Optional[int] = None  # of a held step's forwards, where the caller has said it
        self.version += 1

    def __deepcopy__(self, memo) -> "_Book":
        with self.lock:
            other = _Book(self.sequences, self.pages, self.page, self.columns)
            for name, value in self.__dict__.items():
                if name not in ("states", "uploaded", "lock", "captured"):  # (what a device was told is told anew, and what was captured reads the original's)
                    setattr(other, name, copy.deepcopy(value, memo))
        return other

    def after(self) -> List[int]:
        return [n + c for n, c in zip(self.before, self.counts)]

    def begin(self, counts: Sequence[int], hold: bool, rows: Optional[int] = None) -> None:
        counts = [int(c) for c in counts]
        if len(counts) != self.sequences or min(counts, default=0) < 0:
            raise ValueError(f"PagedCache: {self.sequences} counts of new rows, none below 0, are needed, got {counts}")
        if rows is not None and (not hold or rows < 1):
            raise ValueError(f"PagedCache: rows says how many rows of each sequence the forwards of a held step have, got {rows}{'' if hold else ' for a step that is not held'}")
        most = rows if rows is not None else min(self.captured) if hold and self.captured else None
        if most is not None and max(counts) > most:
            raise ValueError(f"PagedCache: {counts} new rows for a forward of {most} rows a sequence" + ("" if rows is not None else ", as was captured; rows= says which one will be replayed"))
        before = self.after() if self.taken else self.before
        need = [-(-(n + c) // self.page) - len(t) for n, c, t in zip(before, counts, self.tables)]
        if max((len(t) + max(n, 0) for n, t in zip(need, self.tables)), default=0) > self.columns:
            raise RuntimeError(f"PagedCache: a sequence of {max(n + c for n, c in zip(before, counts))} positions needs more than {self.columns} pages of {self.page}")
        if sum(max(n, 0) for n in need) > len(self.free):
            raise RuntimeError(f"PagedCache: {sum(max(n, 0) for n in need)} more pages of {self.page} positions are needed, {len(self.free)} of {self.pages} are free")
        for table, n in zip(self.tables, need):
            table.extend(self.free.pop() for _ in range(n))
        self.before, self.counts, self.rows = before, counts, rows
        self.number, self.version = self.number + 1, self.version + 1
        self.taken, self.hold, self.over = hold, hold, False  # (replays of a captured forward do not come by here)

    def release(self, sequence: int) -> None:
        sequence = operator.index(sequence)
        if not 0 <= sequence < self.sequences:
            raise IndexError(f"PagedCache: there is no sequence {sequence} among {self.sequences}")
        if not self.taken:
            raise RuntimeError("PagedCache: a step was prepared that no forward has made yet")
        self.before = self.after()
        self.end()
        self.free.extend(reversed(self.tables[sequence]))
        self.tables[sequence], self.before[sequence] = [], 0

    def on(self, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """table, lengths and counts of the step on the device: always the same memory, which a captured forward reads."""
        n = self.sequences
        state = self.states.get(device)
        if state is None:
            with torch.inference_mode(False):  # (written outside of that mode too)
                state = self.states[device] = torch.zeros(n * (self.columns + 2), dtype=torch.int32, device=device)
        if self.uploaded.get(device) != self.version:
            rows = torch.full((n, self.columns), -1, dtype=torch.int32)
            for row, table in zip(rows, self.tables):
                row[:len(table)] = torch.tensor(table, dtype=torch.int32)
            state.copy_(torch.cat([rows.flatten(), torch.tensor(self.after() + self.counts, dtype=torch.int32)]))
            self.uploaded[device] = self.version
        return state[:n * self.columns].view(n, self.columns), state[n * self.columns:n * (self.columns + 1)], state[n * (self.columns + 1):]

    def tell(self) -> None:
        """Brings the devices' state up to date, where captured forwards look for it."""
        for device in self.states:
            self.on(device)

    def tell_captured(self) -> None:
        if self.captured:  # (eager forwards ask by themselves)
            self.tell()


class PagedCache:
    """A key/value cache in pages for `sequences` sequences, which differ in length and come and go, as `past_key_values` of a model whose attention modules have the fused forward
    (`attention.fuse_rotary_`; others raise). Each layer of each rank gets a pool of `pages` pages with `page` positions when it is first used; all of them share one page table, which has
    room for `most_pages` pages of a sequence (`pages` by default).

        cache = tp.paged.PagedCache(sequences=3, pages=512)
        positions = cache.prepare([40, 7, 100])                           # rows of each sequence in the next forward
        model(input_ids=padded, position_ids=positions, past_key_values=cache, use_cache=True)      # [3, 100], rows padded on the right; what stands behind a sequence's rows means nothing
        positions = cache.prepare([1, 1, 1])
        logits = model(input_ids=tokens, position_ids=positions, past_key_values=cache, use_cache=True).logits
        cache.release(1)                                                  # sequence 1 has ended: its pages are free, row 1 may begin another

    A forward that nothing was prepared for has all of its rows new, in every sequence. Positions are the model's business: it counts from the longest sequence where it is given none, so
    sequences of different lengths need `position_ids` (a forward without them is refused). Masks of padding are refused too (rows are padded on the right, and counted) where an attention module can
    tell them: with `fuse_rotary_(model, assume_no_padding=True)`, which Falcon always needs, any mask is the causal one by the caller's word, and is ignored. Rotations are by the model's own tables of
    cos and sin, in the model's dtype.

    `prepare(counts, hold=True)`: all forwards up to the next `prepare` are the same step, which counts as made. A forward captured under it (`tp.graphs.capture`, with
    `fuse_rotary_(model, assume_no_padding=True)`: transformers makes a mask, the causal one, where a forward is captured) reads table and lengths when it is replayed:

        positions = cache.prepare([1] * 3, hold=True).to(device)
        step = tp.graphs.capture(model, input_ids=tokens, position_ids=positions, past_key_values=cache, use_cache=True)
        positions = cache.prepare([1] * 3, hold=True).to(device)          # every further token, the first of them with the step's own
        logits = step(input_ids=tokens, position_ids=positions, past_key_values=cache, use_cache=True).logits

    A capture needs a step that is held, and a row of position_ids for each sequence; any other is refused. `prepare`, and `release`, `reset` and `abandon` where a forward was captured, write the state
    that captured forwards read on the current streams of their devices: replays on other streams are the caller's to order.

    `copy.deepcopy(cache)` is a cache of its own, with the same sequences in pages of its own; a shallow copy is refused.

    A forward that failed has to be taken back with `abandon()` before it is made again.

    One caller at a time (the ranks of its forward may be threads); beam search (which would have sequences share pages) is not supported."""

    is_compileable = False

    def __init__(self, sequences: int, pages: int, page: int = 64, most_pages: Optional[int] = None):
        if sequences < 1 or pages < 1 or page < 16 or page & (page - 1) or (most_pages is not None and most_pages < 1):
            raise ValueError(f"PagedCache: at least one sequence and one page are needed, and a power of two from 16 on of positions in it, got {sequences}, {pages}, {page}, {most_pages}")
        self._book = _Book(sequences, pages, page, pages if most_pages is None else most_pages)
        self._own()

    def _own(self) -> None:
        self._pools: dict = {}          # layer -> (keys, values)
        self._number, self._seen = -1, set()  # the step that this rank's forward is in, and its layers that have been there

    def rank_sibling(self) -> "PagedCache":
        """Another rank's cache: pools of its own, the same sequences (kv_cache.rank_caches)."""
        return self._with(self._book)

    def _with(self, book: _Book) -> "PagedCache":
        other = type(self).__new__(type(self))
        other._book = book
        other._own()
        return other

    def __deepcopy__(self, memo) -> "PagedCache":
        """A cache of its own that holds the same sequences (a prefix to go on from in two ways, say): its pages and those of its ranks are copied, the two know nothing of each other."""
        book = copy.deepcopy(self._book, memo)
        others = []
        for one in [self] + self.__dict__.get("_tp_rank_siblings", []):
            other = memo[id(one)] = self._with(book)
            with torch.inference_mode(False):
                other._pools = {layer: tuple(pool.clone() for pool in pools) for layer, pools in one._pools.items()}
            other._number, other._seen = one._number, set(one._seen)
            others.append(other)
        if "_tp_rank_siblings" in self.__dict__:
            kv_cache.link(others[0], others[1:])
        return others[0]

    def __copy__(self):
        raise NotImplementedError("PagedCache: a copy that shares its pages would write to them too; copy.deepcopy copies them")

    def prepare(self, counts: Sequence[int], hold: bool = False, rows: Optional[int] = None) -> torch.Tensor:
        """The next forward has counts[b] new rows of sequence b (of as many rows as the largest count has, padded on the right). Takes their pages, or raises with nothing changed. Returns the
        rows' positions [sequences, largest count] on the host: `position_ids`, once they are on the model's device.

        rows: how many rows of each sequence the forwards of a held step have (and the positions returned). A replay cannot have more rows than it was captured with, so larger counts raise; with
        captured forwards of several widths those larger than the narrowest one's have to be told which one is meant."""
        book = self._book
        book.begin(counts, hold, rows)
        book.tell()
        return torch.tensor(book.before)[:, None] + torch.arange(max(book.counts) if rows is None else rows)

    @property
    def sequences(self) -> int:
        return self._book.sequences

    @property
    def held(self) -> bool:
        """Whether all forwards up to the next `prepare` are the same step."""
        return self._book.hold

    def release(self, sequence: int) -> None:
        """Sequence `sequence` has ended: its pages are free and its length is 0. A step that was held has ended too: a replay before the next `prepare` has no new rows."""
        self._book.release(sequence)
        self._book.tell_captured()

    def lengths(self) -> List[int]:
        """The positions of each sequence, those of a step that a forward has begun among them."""
        return self._book.after() if self._book.taken else list(self._book.before)

    def abandon(self) -> None:
        """The last step is taken back, prepared, held or begun as it is: a forward that failed on its way (behind its first attention module the step counts as made) is made again after this, as if
        it had not been begun. Sequences keep the pages that were taken for it."""
        self._book.end()
        self._book.tell_captured()

    def reset(self) -> None:
        """All sequences have ended, and a step that was held. The pools stay."""
        self._book.reset()
        self._book.tell_captured()

    # ---- what transformers asks of a cache
    def get_seq_length(self, layer_idx: int = 0) -> int:
        """The longest sequence's positions, as this rank's forward sees them: with a step's rows from its first attention module on, but for a step that is held: its next forward is the same one."""
        book = self._book
        return max(book.after() if book.taken and not book.hold and self._number == book.number else book.before)

    def get_max_length(self, layer_idx: int = 0) -> int:
        return self._book.columns * self._book.page

    get_max_cache_shape = get_max_length

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> Tuple[int, int]:
        return query_length, 0  # of the forward's own rows: the plain causal mask, which is not made; what a row sees is the kernels' business

    def get_query_offset(self, layer_idx: int = 0) -> int:
        return 0

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        raise NotImplementedError("PagedCache: this attention module works on keys and values that lie one after another; tp.attention.fuse_rotary_(model) gives those of the Llama pattern and "
                                  "rotary Falcon a forward that works on pages")

    def reorder_cache(self, beam_idx):
        raise NotImplementedError("PagedCache: sequences do not share pages, so there is no beam search on it")

    # ---- the fused attention modules' side
    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layer_idx: int, scale: Optional[float] = None) -> torch.Tensor:
        """One attention module's share of a forward: q [B, S, Hq, D] (or grouped by key/value head), k, v [B, S, Hkv, D], the rotary embedding's tables cos, sin [B or 1, S, part]; [B, S, Hq, D]."""
        with self._book.lock:
            plan, whole, longest = self._step_of(k, cos, layer_idx)
        pools = self._pools[layer_idx]
        half = cos.shape[-1] // 2  # (transformers' tables have each pair's value twice)
        q = append(q, k, v, *pools, **plan, cos=cos[..., :half], sin=sin[..., :half])
        return attend(q, *pools, **plan, scale=scale, max_new=k.shape[1], max_length=longest, out=None if whole else torch.zeros_like(q))

    def _step_of(self, k: torch.Tensor, cos: torch.Tensor, layer_idx: int) -> Tuple[dict, bool, Optional[int]]:
        """Begins the step where this module is the first to come by. Where its rows are, whether all of them are new, and the longest sequence's positions (None: replays differ)."""
        book = self._book
        B, S, Hkv, D = k.shape
        if B != book.sequences:
            raise ValueError(f"PagedCache: {B} sequences in a forward on a cache for {book.sequences}")
        if not book.hold and _capturing(k):
            raise RuntimeError("PagedCache: a forward is captured under a step that is held (prepare(counts, hold=True))")
        first = book.over or self._number != book.number or (layer_idx in self._seen and not book.hold)  # this rank's first module in a forward
        begins = book.over or (first and book.number == self._number)  # a step that nothing was prepared for
        if begins and not book.taken:
            raise RuntimeError("PagedCache: a rank is a forward ahead of the others")
        counts, before = ([S] * B, book.after()) if begins else (book.counts, book.before)
        if max(counts) > S or (max(counts) < S and not book.hold):
            raise ValueError(f"PagedCache: {counts} new rows were prepared, the forward has {S}")
        if book.hold and book.rows not in (None, S):
            raise ValueError(f"PagedCache: forwards of {book.rows} rows a sequence were prepared, this one has {S}")
        if B > 1 and cos.shape[0] == 1 and (min(before) != max(before) or _capturing(k)):  # (of a captured forward they may differ in any replay)
            raise ValueError(f"PagedCache: sequences of {before} positions in one forward need position_ids of their own")
        if begins:
            book.begin(counts, False)
        if first:
            book.taken, self._number, self._seen = True, book.number, set()
        self._seen.add(layer_idx)
        if book.hold and _capturing(k):
            book.captured.add(S)
        lengths = book.after()
        if layer_idx not in self._pools:
            with torch.inference_mode(False):
                self._pools[layer_idx] = tuple(torch.zeros((book.pages, Hkv, book.page, D), dtype=k.dtype, device=k.device) for _ in "kv")
        table, lengths_there, counts_there = book.on(k.device)
        whole = min(counts) == S and not book.hold
        return {"table": table, "lengths": lengths_there, "counts": None if whole else counts_there}, whole, None if book.hold else max(lengths)
