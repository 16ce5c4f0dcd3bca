"""The bookkeeping of `tp.paged.PagedCache`: pages, lengths, steps and ranks. Nothing is computed, so no GPU is needed."""
import copy
import threading
import time

import pytest
import torch

from tensor_parallel_amd import kv_cache, paged


def pages_of(cache):
    return cache._book.tables


def step(cache, layers=(0,)):
    """What a forward does to the bookkeeping: the first attention module takes the step."""
    cache._book.taken, cache._number = True, cache._book.number


def test_pages_are_taken_as_sequences_grow_and_given_back():
    cache = paged.PagedCache(sequences=3, pages=10, page=16)
    positions = cache.prepare([40, 0, 16])
    assert positions.shape == (3, 40) and positions[0].tolist() == list(range(40))
    assert [len(t) for t in pages_of(cache)] == [3, 0, 1] and cache.lengths() == [0, 0, 0] and cache.get_seq_length() == 0
    step(cache)
    assert cache.lengths() == [40, 0, 16] and cache.get_seq_length() == 40
    assert cache.prepare([1, 5, 1])[:, 0].tolist() == [40, 0, 16]
    assert [len(t) for t in pages_of(cache)] == [3, 1, 2]
    step(cache)
    used = [p for t in pages_of(cache) for p in t]
    assert len(set(used)) == len(used) == 6
    cache.release(0)
    assert cache.lengths() == [0, 5, 17] and len(cache._book.free) == 7
    cache.prepare([96, 1, 1])
    assert len(pages_of(cache)[0]) == 6
    cache.reset()
    assert cache.lengths() == [0, 0, 0] and len(cache._book.free) == 10


def test_a_step_that_does_not_fit_changes_nothing():
    cache = paged.PagedCache(sequences=2, pages=4, page=16, most_pages=3)
    cache.prepare([30, 16])
    step(cache)
    before = copy.deepcopy(pages_of(cache))
    for counts in ([3, 1, 1], [-1, 2], [20, 17], [40, 1]):
        with pytest.raises((RuntimeError, ValueError)):
            cache.prepare(counts)
        assert pages_of(cache) == before and cache.lengths() == [30, 16] and len(cache._book.free) == 1


def test_a_step_is_prepared_anew_until_a_forward_takes_it():
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    cache.prepare([100])
    cache.prepare([5])
    assert cache.lengths() == [0]
    with pytest.raises(RuntimeError):
        cache.release(0)
    step(cache)
    assert cache.lengths() == [5]


def test_a_held_step_counts_as_made():
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    for n in (1, 2, 3):
        assert cache.prepare([1], hold=True).tolist() == [[n - 1]] and cache.lengths() == [n]
    cache.release(0)
    assert cache.lengths() == [0]


def test_state_on_the_device_keeps_its_memory():
    cache = paged.PagedCache(sequences=2, pages=8, page=16, most_pages=3)
    cache.prepare([17, 3])
    table, lengths, counts = cache._book.on(torch.device("cpu"))
    assert table.shape == (2, 3) and table[0, :2].tolist() == pages_of(cache)[0] and table[0, 2] == -1 and lengths.tolist() == [17, 3] and counts.tolist() == [17, 3]
    step(cache)
    cache.prepare([1, 0])
    again = cache._book.on(torch.device("cpu"))
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip((table, lengths, counts), again)) and lengths.tolist() == [18, 3] and counts.tolist() == [1, 0]


def test_ranks_share_pages_and_lengths():
    cache = paged.PagedCache(sequences=1, pages=8)
    assert kv_cache.is_kv_cache(cache)
    cache.prepare([70])
    first, second = kv_cache.rank_caches(cache, 2)
    assert first is cache and second._book is cache._book and second._pools is not cache._pools
    step(first)
    assert first.get_seq_length() == 70 and second.get_seq_length() == 0  # its forward has not come to the step yet
    step(second)
    assert second.get_seq_length() == 70
    cache.reset()
    assert second.lengths() == [0]


@pytest.mark.parametrize("args", [(0, 1), (1, 0), (1, 1, 8), (1, 1, 48), (1, 1, 16, 0)])
def test_sizes_that_are_refused(args):
    with pytest.raises(ValueError):
        paged.PagedCache(*args)


def test_modules_of_other_kinds_are_refused():
    cache = paged.PagedCache(1, 1)
    with pytest.raises(NotImplementedError, match="fuse_rotary_"):
        cache.update(None, None, 0)
    with pytest.raises(NotImplementedError, match="beam"):
        cache.reorder_cache(None)


def forward(cache, rows, layers=2):
    """The attention modules' share of a rank's forward, without the kernels."""
    for layer in range(layers):
        q, kv, table = torch.zeros(1, rows, 2, 64), torch.zeros(1, rows, 1, 64), torch.zeros(1, rows, 64)
        cache.attend(q, kv, kv, table, table, layer)


@pytest.fixture
def no_kernels(monkeypatch):
    monkeypatch.setattr(paged, "append", lambda q, *args, **kwargs: q)
    monkeypatch.setattr(paged, "attend", lambda q, *args, **kwargs: q)


@pytest.mark.parametrize("prepared", [False, True])
def test_ranks_that_are_threads_begin_a_step_once(no_kernels, monkeypatch, prepared):
    after = paged._Book.after

    def slowly(book):
        counts = after(book)
        time.sleep(0.02)  # the other rank comes by between reading the book and writing it
        return counts

    monkeypatch.setattr(paged._Book, "after", slowly)
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    ranks = kv_cache.rank_caches(cache, 3)
    failed = []

    def run(rank, barrier):
        try:
            barrier.wait(10)
            forward(rank, 5)
        except BaseException as e:
            failed.append(e)

    for n in (1, 2):
        if prepared:
            cache.prepare([5])
        barrier = threading.Barrier(len(ranks))
        threads = [threading.Thread(target=run, args=(r, barrier)) for r in ranks]
        [t.start() for t in threads]
        [t.join(30) for t in threads]
        assert not failed and cache.lengths() == [5 * n]


def test_a_cache_that_was_reset_begins_a_step_once(no_kernels):
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    ranks = kv_cache.rank_caches(cache, 2)
    for _ in range(3):
        for n in (1, 2):
            [forward(r, 5) for r in ranks]
            assert cache.lengths() == [5 * n]
        cache.reset()
        assert cache.lengths() == [0] and [r.get_seq_length() for r in ranks] == [0, 0]


def test_devices_have_state_of_their_own():
    cache = paged.PagedCache(sequences=1, pages=8, page=16)
    cache.prepare([3])
    devices = torch.device("cpu"), torch.device("meta")
    first = [cache._book.on(d) for d in devices]
    step(cache)
    cache.prepare([1])  # (both are brought up to date: captured forwards on either read them)
    assert first[0][1].tolist() == [4]
    for device, state in zip(devices, first):
        assert all(a is b or (a.device == device and a.untyped_storage()._cdata == b.untyped_storage()._cdata) for a, b in zip(cache._book.on(device), state))
