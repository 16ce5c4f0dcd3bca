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
