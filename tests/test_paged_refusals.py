"""What the calls on heads and paged caches refuse, through the Python layer and at the C entry points: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

from tensor_parallel_amd import _native, attention, paged

INVALID, UNSUPPORTED = -1, -2
F16, BF16, I32 = torch.float16, torch.bfloat16, torch.int32


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def test_host_tensors():
    x, pool, table, lengths = z(2, 2, 64), z(3, 2, 16, 64), z(2, 2, dtype=I32), z(2, dtype=I32)
    for call in (lambda: attention.rotate(x, x), lambda: paged.append(x, x, x, pool, pool, table, lengths), lambda: paged.attend(x, pool, pool, table, lengths)):
        with pytest.raises(_native.NativeLibraryError):
            call()


@pytest.fixture
def checks(monkeypatch):
    """The checks of arguments on host tensors; a call that got past them would fail at the library."""
    monkeypatch.setattr(_native, "require_device", lambda *_: None)
    monkeypatch.setattr(_native, "lib", lambda: pytest.fail("the call was not refused"))


def rotate(q=z(2, 4, 64), k=z(2, 2, 64), positions=torch.zeros(2, dtype=torch.int64), inv_freq=torch.zeros(32), **more):
    return attention.rotate(q, k, positions, inv_freq=inv_freq, **more)


def append(q=z(2, 4, 64), k=z(2, 2, 64), v=z(2, 2, 64), k_pages=z(3, 2, 16, 64), v_pages=z(3, 2, 16, 64), table=z(2, 2, dtype=I32), lengths=z(2, dtype=I32), **more):
    return paged.append(q, k, v, k_pages, v_pages, table, lengths, **more)


def attend(q=z(2, 4, 64), k_pages=z(3, 2, 16, 64), v_pages=z(3, 2, 16, 64), table=z(2, 2, dtype=I32), lengths=z(2, dtype=I32), **more):
    return paged.attend(q, k_pages, v_pages, table, lengths, **more)


@pytest.mark.parametrize("call,error", [
    (lambda: rotate(q=z(2, 4, 64, dtype=torch.float32), k=z(2, 2, 64, dtype=torch.float32)), TypeError),
    (lambda: rotate(k=z(2, 2, 64, dtype=BF16)), TypeError),
    (lambda: rotate(k=z(3, 2, 64)), ValueError),
    (lambda: rotate(k=z(2, 2, 32)), ValueError),
    (lambda: rotate(q=z(2, 4, 3, 64)), ValueError),  # groups of another number of key/value heads
    (lambda: rotate(q=z(64), k=z(64)), ValueError),
    (lambda: rotate(positions=None), ValueError),
    (lambda: rotate(positions=torch.zeros(3, dtype=torch.int64)), ValueError),
    (lambda: rotate(positions=torch.zeros(2)), ValueError),
    (lambda: rotate(inv_freq=torch.zeros(2, 32)), ValueError),
    (lambda: rotate(cos=torch.zeros(2, 32)), ValueError),
    (lambda: rotate(inv_freq=None, cos=torch.zeros(2, 32)), ValueError),
    (lambda: rotate(inv_freq=None, cos=torch.zeros(2, 32), sin=torch.zeros(2, 31)), ValueError),
    (lambda: rotate(inv_freq=None, cos=torch.zeros(2, 32, dtype=torch.float64), sin=torch.zeros(2, 32, dtype=torch.float64)), TypeError),
    (lambda: rotate(q_norm=z(63)), ValueError),
    (lambda: rotate(k_norm=torch.zeros(64)), ValueError),
    (lambda: rotate(q=z(2, 64, 4).transpose(1, 2)), ValueError),
    (lambda: append(v=z(2, 1, 64)), ValueError),
    (lambda: append(v=z(2, 2, 64, dtype=BF16)), TypeError),
    (lambda: append(k_pages=z(3, 1, 16, 64)), ValueError),
    (lambda: append(v_pages=z(3, 2, 32, 64)), ValueError),
    (lambda: append(k_pages=z(3, 2, 16, 64, dtype=BF16)), TypeError),
    (lambda: append(k_pages=z(3, 2, 64, 16).transpose(2, 3)), ValueError),
    (lambda: append(table=z(2, 2, dtype=torch.int64)), TypeError),
    (lambda: append(lengths=z(2, dtype=torch.int64)), TypeError),
    (lambda: append(lengths=z(3, dtype=I32)), ValueError),
    (lambda: append(starts=z(2, dtype=I32)), ValueError),
    (lambda: append(counts=z(3, dtype=I32)), ValueError),
    (lambda: append(starts=z(3, dtype=torch.int64)), TypeError),
    (lambda: attend(q=z(2, 4, 64, dtype=torch.float32)), TypeError),
    (lambda: attend(q=z(64)), ValueError),
    (lambda: attend(q=z(2, 4, 128)), ValueError),
    (lambda: attend(k_pages=z(3, 2, 16)), ValueError),
    (lambda: attend(v_pages=z(3, 2, 16, 64, dtype=BF16)), TypeError),
    (lambda: attend(table=z(2, dtype=I32)), ValueError),
    (lambda: attend(out=z(2, 4, 32)), ValueError),
    (lambda: attend(out=z(2, 4, 64, dtype=BF16)), ValueError),
])
def test_refused_by_the_python_layer(checks, monkeypatch, call, error):
    with pytest.raises(error):
        call()


# ---- the C entry points ------------------------------------------------------------------------------------------------
KEEP = (ctypes.c_char * 4096)()
AT = (ctypes.addressof(KEEP) + 255) // 256 * 256
HEADS = dict(q=AT, k=AT, v=AT, q_row=256, q_group=128, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, q_norm=0, k_norm=0, eps=1e-6, scaling=1.0, inv_freq=AT, cos=0, sin=0, table_row=0,
             table_dtype=0, interleaved=0, part=64, positions=AT, q_out=AT, k_out=AT, qo_row=256, qo_head=64, ko_row=128, ko_head=64)
PAGES = dict(k=AT, v=AT, pages=3, page=16, k_page=2048, k_head=1024, k_pos=64, v_page=2048, v_head=1024, v_pos=64, table=AT, table_row=2, columns=2, lengths=AT, starts=AT, counts=0, seqs=2)


def packed(form, base, **changes):
    return form.pack(*{**base, **changes}.values())


def refused(rc, status, word):
    assert rc == status
    assert word in _native.lib().tpamd_last_error().decode()


needs_library = pytest.mark.skipif(not _native.available(), reason="the library is not built")


@needs_library
@pytest.mark.parametrize("heads,sizes,dtype,word", [
    ({}, (2, 4, 2, 64), 2, "dtype"), ({}, (-1, 4, 2, 64), 1, "dimension"), ({}, (1 << 24, 4, 2, 64), 1, "dimension"), ({}, (2, 4, 3, 64), 1, "multiple"), ({}, (2, 4, 2, 63), 1, "even"),
    ({}, (2, 4, 2, 514), 1, "even"), ({"part": 66}, (2, 4, 2, 64), 1, "pairs"), ({"part": 3}, (2, 4, 2, 64), 1, "pairs"), ({"inv_freq": 0}, (2, 4, 2, 64), 1, "tables"),
    ({"cos": AT, "sin": AT}, (2, 4, 2, 64), 1, "tables"), ({"positions": 0}, (2, 4, 2, 64), 1, "positions"), ({"k_out": 0}, (2, 4, 2, 64), 1, "null"), ({"q": 0}, (2, 4, 2, 64), 1, "null"),
    ({"inv_freq": 0, "cos": AT, "sin": AT, "table_dtype": 9}, (2, 4, 2, 64), 1, "unknown"),
])
def test_rotate_heads_refuses(heads, sizes, dtype, word):
    refused(_native.lib().tpamd_rotate_heads(packed(_native._HEADS, HEADS, **heads), *sizes, dtype, 0), INVALID, word)


PAGE_FAULTS = [
    ({"page": 8}, "power of two"), ({"page": 48}, "power of two"), ({"columns": 1 << 27}, "too many"), ({"counts": AT}, "not both"), ({"starts": 0, "seqs": 3}, "same number"),
    ({"lengths": 0}, "null"), ({"table": 0}, "null"), ({"k": 0}, "null"), ({"k_pos": -64}, "stride"), ({"seqs": -1}, "dimension"), ({"pages": 1 << 31}, "dimension"),
]


@needs_library
@pytest.mark.parametrize("pages,word", PAGE_FAULTS)
def test_append_paged_refuses(pages, word):
    refused(_native.lib().tpamd_append_paged(packed(_native._HEADS, HEADS), packed(_native._PAGES, PAGES, **pages), 2, 4, 2, 64, 1, 0), INVALID, word)


def attend_c(pages={}, rows=2, Hq=4, Hkv=2, D=64, dtype=1, q=AT, out=AT, q_row=256, max_new=2, max_length=32, work=0, work_bytes=0):
    return _native.lib().tpamd_attention_paged(q, q_row, 64, packed(_native._PAGES, PAGES, **pages), out, 256, 64, rows, Hq, Hkv, D, max_new, max_length, 0.125, dtype, work, work_bytes, 0)


@needs_library
@pytest.mark.parametrize("pages,word", PAGE_FAULTS)
def test_attention_paged_refuses_pages(pages, word):
    refused(attend_c(pages), INVALID, word)
    need = ctypes.c_uint64()
    refused(_native.lib().tpamd_attention_paged_workspace(packed(_native._PAGES, PAGES, **pages), 2, 4, 2, 64, 2, 32, ctypes.byref(need)), INVALID, word)


@needs_library
@pytest.mark.parametrize("more,status,word", [
    ({"dtype": 2}, INVALID, "dtype"), ({"D": 80}, UNSUPPORTED, "head_dim"), ({"Hq": 5}, INVALID, "multiple"), ({"rows": -1}, INVALID, "dimension"), ({"q": 0}, INVALID, "null"),
    ({"max_new": -1}, INVALID, "argument"), ({"q": AT + 8}, UNSUPPORTED, "boundaries"), ({"out": AT + 4}, UNSUPPORTED, "boundaries"), ({"q_row": 260}, UNSUPPORTED, "boundaries"),
    ({"pages": {"k_pos": 68}}, UNSUPPORTED, "boundaries"), ({"pages": {"v_pos": 1 << 26}}, UNSUPPORTED, "boundaries"), ({"rows": 1 << 20, "Hq": 1 << 12, "Hkv": 1 << 12}, INVALID, "too many"),
])
def test_attention_paged_refuses(more, status, word):
    refused(attend_c(**more), status, word)


@needs_library
def test_nothing_to_do_needs_no_pointers():
    nothing = dict(q=0, k=0, v=0, inv_freq=0, positions=0, q_out=0, k_out=0)
    none = packed(_native._PAGES, PAGES, k=0, v=0, pages=0, table=0, columns=0, lengths=0, starts=0, seqs=0)
    lib = _native.lib()
    assert lib.tpamd_rotate_heads(packed(_native._HEADS, HEADS, **nothing), 0, 4, 2, 64, 1, 0) == 0
    assert lib.tpamd_append_paged(packed(_native._HEADS, HEADS, **nothing), none, 0, 4, 2, 64, 1, 0) == 0
    assert lib.tpamd_attention_paged(0, 0, 0, none, 0, 0, 0, 0, 4, 2, 64, 0, 0, 0.1, 1, 0, 0, 0) == 0
