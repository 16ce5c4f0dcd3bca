"""What a `tp.paged.PagedCache` does between steps: copies, steps that are held, taken back or ended, and ranks. Nothing is computed, so no GPU is needed."""
import copy

import pytest
import torch

from tensor_parallel_amd import graphs, kv_cache, paged


@pytest.fixture
def written(monkeypatch):
    """attend and append without kernels: the new rows of each sequence are written to its pages, as the kernels do."""
    def append(q, k, v, k_pages, v_pages, table, lengths, counts=None, **kwargs):
        page = k_pages.shape[2]
        for b in range(k.shape[0]):
            n = k.shape[1] if counts is None else min(int(counts[b]), k.shape[1])
            for i in range(n):
                at = int(lengths[b]) - n + i
                k_pages[int(table[b, at // page]), :, at % page], v_pages[int(table[b, at // page]), :, at % page] = k[b, i], v[b, i]
        return q

    monkeypatch.setattr(paged, "append", append)
    monkeypatch.setattr(paged, "attend", lambda q, *args, **kwargs: q)


def forward(cache, rows, layers=2, value=1.0):
    """The attention modules' share of a rank's forward."""
    B = cache._book.sequences
    for layer in range(layers):
        q, kv, table = torch.zeros(B, rows, 2, 64), torch.full((B, rows, 1, 64), value), torch.zeros(B, rows, 64)
        cache.attend(q, kv, kv, table, table, layer)


def keys(cache, layer=0):
    """The keys of each sequence, by the page table, one value a position."""
    book = cache._book
    pool = cache._pools[layer][0]
    return [[float(pool[book.tables[b][j // book.page], 0, j % book.page, 0]) for j in range(n)] for b, n in enumerate(cache.lengths())]


# ---- copies ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ranks", [1, 2])
def test_a_copy_of_a_filled_cache_is_a_cache_of_its_own(written, ranks):
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    of_ranks = kv_cache.rank_caches(cache, ranks)
    for rank in of_ranks:
        forward(rank, 20, value=3.0)
    other = copy.deepcopy(cache)
    of_others = kv_cache.rank_caches(other, ranks)
    assert other.lengths() == [20] and [keys(c) for c in of_others] == [[[3.0] * 20]] * ranks
    for rank in of_others:
        forward(rank, 1, value=5.0)  # (a step that nothing was prepared for)
    assert cache.lengths() == [20] and other.lengths() == [21]
    cache.prepare([2])
    for rank in of_ranks:
        forward(rank, 2, value=7.0)
    assert [keys(c) for c in of_ranks] == [[[3.0] * 20 + [7.0] * 2]] * ranks
    assert [keys(c) for c in of_others] == [[[3.0] * 20 + [5.0]]] * ranks
    other.reset()
    assert other.lengths() == [0] == of_others[-1].lengths() and cache.lengths() == [22] == of_ranks[-1].lengths()
    cache.reset()
    assert cache.lengths() == [0]


def test_a_copy_has_the_step_that_was_prepared(written):
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    cache.prepare([3, 1])
    other = copy.deepcopy(cache)
    forward(other, 3)
    assert other.lengths() == [3, 1] and cache.lengths() == [0, 0]
    forward(cache, 3)
    assert cache.lengths() == [3, 1]


def test_a_shallow_copy_is_refused():
    with pytest.raises(NotImplementedError, match="deepcopy"):
        copy.copy(paged.PagedCache(1, 1))


# ---- steps that are held -----------------------------------------------------------------------------------------------
def test_forwards_of_a_held_step_begin_at_the_same_position(written):
    """A model that is given no positions counts from this."""
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    forward(cache, 5)
    assert cache.get_seq_length() == 5
    for before in (5, 6):
        cache.prepare([1], hold=True)
        for _ in range(3):
            assert cache.get_seq_length() == before
            forward(cache, 1)
        assert cache.get_seq_length() == before and cache.lengths() == [before + 1]
    cache.prepare([1])
    assert cache.get_seq_length() == 7
    forward(cache, 1)
    assert cache.get_seq_length() == 8


def captured(monkeypatch, cache, width, **how):
    """A held forward while a stream is captured, and the replay of it: what the kernels read."""
    cache.prepare([1] * cache._book.sequences, hold=True, **how)
    with monkeypatch.context() as m:
        m.setattr(paged, "_capturing", lambda t: True)
        forward(cache, width)


def test_a_step_of_more_rows_than_were_captured_is_refused(written, monkeypatch):
    """A replay has the rows it was captured with: counted beyond them, positions would be attended to that nothing was written to."""
    cache = paged.PagedCache(sequences=2, pages=16, page=16)
    forward(cache, 5)
    cache.prepare([3, 1], hold=True)  # (nothing is captured yet: a forward says by itself that it has fewer)
    with pytest.raises(ValueError, match="prepared"):
        forward(cache, 1)
    captured(monkeypatch, cache, 1)
    lengths = cache.lengths()
    state = [t.clone() for t in cache._book.on(torch.device("cpu"))]
    for how in ({}, {"rows": 2}):
        with pytest.raises(ValueError, match="rows"):
            cache.prepare([3, 1], hold=True, **how)
        assert cache.lengths() == lengths and all(torch.equal(a, b) for a, b in zip(state, cache._book.on(torch.device("cpu"))))
    cache.prepare([3, 1])  # forwards that are not held are not captured ones
    forward(cache, 3)
    cache.reset()
    with pytest.raises(ValueError, match="rows"):
        cache.prepare([2, 1], hold=True)


def test_captured_forwards_of_several_widths(written, monkeypatch):
    cache = paged.PagedCache(sequences=1, pages=16, page=16)
    captured(monkeypatch, cache, 4, rows=4)
    cache.prepare([3], hold=True)
    captured(monkeypatch, cache, 1)
    with pytest.raises(ValueError, match="rows"):
        cache.prepare([3], hold=True)  # which of the two will be replayed is not known
    assert cache.prepare([3], hold=True, rows=4).shape == (1, 4)
    with pytest.raises(ValueError, match="4"):
        forward(cache, 3)
    forward(cache, 4)
    with pytest.raises(ValueError):
        cache.prepare([1], rows=4)  # of steps that are held
    other = copy.deepcopy(cache)
    other.prepare([9], hold=True)  # what was captured works on the original


class Model(torch.nn.Module):
    """Takes positions as a transformers model does, by name or in their place."""

    def __init__(self):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.zeros(1))

    def forward(self, input_ids, attention_mask=None, position_ids=None, past_key_values=None, **kwargs):
        raise AssertionError("the capture was not refused")


class OwnPositions(Model):
    def forward(self, input_ids, past_key_values=None):
        raise AssertionError("the capture was not refused")


def test_a_capture_without_positions_is_refused():
    """Positions that the model counts on the host would be the captured step's in every replay."""
    ids = torch.zeros(2, 1, dtype=torch.int64)
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    positions = cache.prepare([1, 1], hold=True)
    nested = torch.nn.Module()
    nested.module_shards = [Model()]
    outer = torch.nn.Module()
    outer.wrapped_model = nested
    for model in (Model(), nested, outer):
        with pytest.raises(ValueError, match="position_ids"):
            graphs.capture(model, input_ids=ids, past_key_values=cache)
    # (these get as far as the devices, of which there are none here)
    for call in (lambda: graphs.capture(Model(), input_ids=ids, position_ids=positions, past_key_values=cache), lambda: graphs.capture(Model(), ids, None, positions, past_key_values=cache),
                 lambda: graphs.capture(OwnPositions(), ids, past_key_values=cache)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_a_capture_of_a_step_that_is_not_held_is_refused(written, monkeypatch):
    """Each of a capture's own forwards would be counted as a step, and no replay."""
    ids = torch.zeros(2, 1, dtype=torch.int64)
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    forward(cache, 3)
    for prepared in (False, True):
        positions = cache.prepare([1, 1]) if prepared else torch.tensor([[3], [3]])
        with pytest.raises(ValueError, match="hold"):
            graphs.capture(Model(), input_ids=ids, position_ids=positions, past_key_values=cache)
        assert cache.lengths() == [3, 3]
        with monkeypatch.context() as m:  # by torch's own means
            m.setattr(paged, "_capturing", lambda t: True)
            with pytest.raises(RuntimeError, match="hold"):
                forward(cache, 1)
        assert cache.lengths() == [3, 3]


def test_a_capture_with_one_row_of_positions_for_several_sequences_is_refused(written, monkeypatch):
    """They may be as long as one another now; replays would turn them alike when they no longer are."""
    ids = torch.zeros(2, 1, dtype=torch.int64)
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    cache.prepare([1, 1], hold=True)
    with pytest.raises(ValueError, match="each"):
        graphs.capture(Model(), input_ids=ids, position_ids=torch.zeros(1, 1, dtype=torch.int64), past_key_values=cache)
    q, kv = torch.zeros(2, 1, 2, 64), torch.zeros(2, 1, 1, 64)
    tables = {rows: torch.zeros(rows, 1, 64) for rows in (1, 2)}
    cache.attend(q, kv, kv, tables[1], tables[1], 0)  # (an eager forward is told when they no longer fit)
    monkeypatch.setattr(paged, "_capturing", lambda t: True)
    with pytest.raises(ValueError, match="of their own"):
        cache.attend(q, kv, kv, tables[1], tables[1], 0)
    cache.attend(q, kv, kv, tables[2], tables[2], 0)


# ---- sequences that end ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sequence", [-1, 2, 1.0, None])
def test_a_sequence_that_there_is_not_is_not_released(written, sequence):
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    forward(cache, 20)
    with pytest.raises((IndexError, TypeError)):
        cache.release(sequence)
    assert cache.lengths() == [20, 20] and len(cache._book.free) == 4
    cache.release(1)
    assert cache.lengths() == [20, 0]


@pytest.mark.parametrize("end", ["release", "reset"])
def test_replays_after_a_sequence_has_ended_write_nothing_to_its_pages(written, monkeypatch, end):
    """What a captured forward reads is told that there are no new rows, and that the pages are another's, before the next step is prepared."""
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    forward(cache, 20)
    captured(monkeypatch, cache, 1)
    table, lengths, counts = (t for t in cache._book.on(torch.device("cpu")))  # what the captured forward reads
    assert lengths.tolist() == [21, 21] and counts.tolist() == [1, 1]
    cache.release(0) if end == "release" else cache.reset()
    assert counts.tolist() == [0, 0] and lengths.tolist() == ([0, 21] if end == "release" else [0, 0])
    assert (table[0] == -1).all() and (end == "release" or (table == -1).all())
    if end == "release":
        assert table[1, :2].tolist() == pages_of(cache)[1]
    # the held step has ended with it: an eager forward that nothing was prepared for is a step of its own
    before = cache.lengths()
    forward(cache, 2)
    assert cache.lengths() == [n + 2 for n in before] and counts.tolist() == [2, 2]
    assert not cache.held


def pages_of(cache):
    return cache._book.tables


# ---- modes of torch ----------------------------------------------------------------------------------------------------
def test_forwards_in_inference_mode_and_steps_outside_of_it(written):
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    with torch.inference_mode():
        forward(cache, 5)
    cache.prepare([2])
    forward(cache, 2)
    with torch.inference_mode():
        cache.prepare([1])
        forward(cache, 1)
        other = copy.deepcopy(cache)
    other.prepare([1])
    forward(other, 1)
    cache.release(0)
    assert other.lengths() == [9] and cache.lengths() == [0]


# ---- forwards that fail ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("prepared", [False, True])
@pytest.mark.parametrize("came_by", [(1, 0), (2, 0), (2, 1), (0, 1)])
def test_a_step_that_failed_is_taken_back_and_made_again(written, prepared, came_by):
    """Some modules of some ranks have come by when a forward fails; made again, whichever rank is first, it counts once and fills every layer."""
    cache = paged.PagedCache(sequences=2, pages=12, page=16)
    ranks = kv_cache.rank_caches(cache, 2)
    for rank in ranks:
        forward(rank, 15, value=1.0)
    if prepared:
        cache.prepare([3, 2])
    for rank, layers in zip(ranks, came_by):
        forward(rank, 3, layers=layers, value=9.0)
    cache.abandon()
    assert cache.lengths() == [15, 15] and [r.get_seq_length() for r in ranks] == [15, 15]
    if prepared:
        assert cache.prepare([3, 2])[:, 0].tolist() == [15, 15]
    for rank in ranks[::-1]:
        forward(rank, 3, value=2.0)
    assert cache.lengths() == [18, 17 if prepared else 18]
    for rank in ranks:
        for layer in (0, 1):
            assert [k[15:] for k in keys(rank, layer)] == [[2.0] * (n - 15) for n in cache.lengths()]
    used = [p for t in pages_of(cache) for p in t]
    assert len(set(used)) == len(used) == 12 - len(cache._book.free)


def test_a_prepared_and_a_held_step_are_taken_back(written, monkeypatch):
    cache = paged.PagedCache(sequences=1, pages=4, page=16)
    cache.abandon()  # there is nothing to take back
    cache.prepare([40])
    cache.abandon()
    cache.release(0)  # (a step that no forward has made would be in its way)
    forward(cache, 5)
    captured(monkeypatch, cache, 1)
    _, lengths, counts = cache._book.on(torch.device("cpu"))
    cache.prepare([1], hold=True)
    assert lengths.tolist() == [7]
    cache.abandon()
    assert cache.lengths() == [6] == lengths.tolist() and counts.tolist() == [0] and not cache.held
    assert cache.prepare([1], hold=True).tolist() == [[6]] and lengths.tolist() == [7] and counts.tolist() == [1]


def test_nothing_is_uploaded_at_the_end_of_a_sequence_where_nothing_was_captured(written, monkeypatch):
    """A server's sequences end many at a time, and its next step brings the state up to date anyway."""
    cache = paged.PagedCache(sequences=2, pages=8, page=16)
    forward(cache, 5)
    uploads = []
    on = paged._Book.on
    monkeypatch.setattr(paged._Book, "on", lambda book, device: uploads.append(device) or on(book, device))
    cache.release(0)
    cache.release(1)
    cache.abandon()
    cache.reset()
    assert not uploads
    forward(cache, 5, layers=1)
    assert len(uploads) == 1 and on(cache._book, torch.device("cpu"))[1].tolist() == [5, 5]
