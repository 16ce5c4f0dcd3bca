"""Ranges of K of products of 8-bit rows and the scratch memory that their partial sums lie in."""
import pytest
import torch

from tensor_parallel_amd import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("M,N,K,ranges,split", [(300, 512, 8192, 4, True), (1024, 2048, 8192, 64, True), (8200, 2048, 1024, 2, False)])
def test_a_stream_s_buffer_has_one_size(tune, M, N, K, ranges, split):
    """TPAMD_A8_SPLITS is held to it: as many ranges as it has room for, none where a single one's partial tiles have not, whether the stream has its buffer already or gets it in this call."""
    g = torch.Generator(device=DEV).manual_seed(0)
    q, w = (torch.randint(-127, 128, (n, K), dtype=torch.int8, device=DEV, generator=g) for n in (M, N))
    qs, ws = torch.rand(M, device=DEV, generator=g) / 4096, torch.rand(N, device=DEV, generator=g)
    tune("TPAMD_A8_TILE", 64128)
    tune("TPAMD_A8_SPLITS", 1)
    want = _native.linear_a8(q, qs, w, ws)
    tune("TPAMD_A8_SPLITS", ranges)
    torch.cuda.synchronize()
    reserve = torch.cuda.get_device_properties(DEV).multi_processor_count * 4 * 128 * 128 * 4 + (4 << 20)
    stream = torch.cuda.Stream(DEV)
    _native.release_scratch(DEV, stream.cuda_stream)  # (torch hands a small number of streams out in turn)
    try:
        with torch.cuda.stream(stream):
            got = [_native.linear_a8(q, qs, w, ws) for _ in range(2)]
        stream.synchronize()
        assert _native.scratch_of_stream(DEV, stream.cuda_stream)[1] == (reserve if split else 0)
        assert all(torch.equal(t, want) for t in got)
    finally:
        _native.release_scratch(DEV, stream.cuda_stream)
