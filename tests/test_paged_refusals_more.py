"""Further calls on heads and paged caches that are refused: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

from tensor_parallel_amd import _native, attention, paged
from test_paged_refusals import AT, HEADS, INVALID, PAGES, append, attend_c, checks, needs_library, packed, refused, rotate, z  # noqa: F401 (checks is a fixture)


def test_positions_beside_tables(checks):
    """Tables have a row for each of the call's rows: positions would be ignored."""
    tables = {"inv_freq": None, "cos": torch.zeros(2, 32), "sin": torch.zeros(2, 32)}
    with pytest.raises(ValueError, match="positions"):
        rotate(**tables)
    with pytest.raises(ValueError, match="positions"):
        append(**tables, positions=torch.zeros(2, dtype=torch.int64))


@needs_library
def test_positions_beside_tables_at_the_entry_points():
    heads = packed(_native._HEADS, HEADS, inv_freq=0, cos=AT, sin=AT)
    refused(_native.lib().tpamd_rotate_heads(heads, 2, 4, 2, 64, 1, 0), INVALID, "positions")
    refused(_native.lib().tpamd_append_paged(heads, packed(_native._PAGES, PAGES), 2, 4, 2, 64, 1, 0), INVALID, "positions")


def test_a_module_that_is_not_causal():
    """Attention on pages is causal."""
    module = torch.nn.Module()
    module.training, module.head_dim, module.is_causal = False, 64, False
    tables = torch.zeros(1, 2, 64), torch.zeros(1, 2, 64)
    with pytest.raises(NotImplementedError, match="causal"):
        attention._fused_rotary_forward(module, z(1, 2, 128), position_embeddings=tables, past_key_values=paged.PagedCache(1, 1))
    falcon = torch.nn.Module()
    falcon.training, falcon.head_dim, falcon.is_causal, falcon.new_decoder_architecture = False, 64, False, True
    with pytest.raises(NotImplementedError, match="causal"):
        attention._fused_falcon_forward(falcon, z(1, 2, 128), position_embeddings=tables, layer_past=paged.PagedCache(1, 1))


@needs_library
@pytest.mark.parametrize("page,columns", [(16, (1 << 27) - 1), (64, (1 << 25) - 1), (16, (1 << 27) - (1 << 12) + 1), (1 << 15, (1 << 16) - 1)])
def test_sequences_whose_end_is_counted_past_31_bits(page, columns):
    """Positions are counted in 32 bits, and up to 2^16 further ones behind the last: whole tiles, ranges of whole tiles, and the pages of the next 64 tiles."""
    at, room = {"page": page, "columns": columns}, page * columns
    assert (1 << 31) - (1 << 16) < room < 1 << 31
    pages = packed(_native._PAGES, PAGES, **at)
    refused(attend_c(at, max_length=room), INVALID, "too many")
    refused(_native.lib().tpamd_append_paged(packed(_native._HEADS, HEADS), pages, 2, 4, 2, 64, 1, 0), INVALID, "too many")
    refused(attend_c({"page": 16, "columns": 1 << 60}), INVALID, "too many")  # (2^64)
    need = ctypes.c_uint64()
    refused(_native.lib().tpamd_attention_paged_workspace(pages, 2, 4, 2, 64, 2, room, ctypes.byref(need)), INVALID, "too many")
    # the longest that are taken (without a GPU the call ends where it asks for one)
    fits = packed(_native._PAGES, PAGES, page=16, columns=(1 << 27) - (1 << 12))
    assert _native.lib().tpamd_attention_paged_workspace(fits, 2, 4, 2, 64, 2, room, ctypes.byref(need)) != INVALID
