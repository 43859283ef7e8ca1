"""The cut time axis of the gated recurrence where a chunk holds several tiles: ragged ends inside a chunk that is not the
last, both directions, with and without wide lanes."""
import pytest
import torch

from test_gpu_recurrence import TYPES, _check_backward, _check_scan, _gpu, _inputs

pytestmark = pytest.mark.gpu

T = 1200
LARGEST_TILE = 256
ENDS = [T, 560, 180]   # an odd number of tiles of 64, 128 or 256 rows lies behind each end in its chunk


def _chunks(B, D, dtype, backward):
    """Chunks of a call: its workspace is a pair of fp32 numbers for every request, chunk and channel."""
    from tts_amd import _lib
    from tts_amd._seq import DTYPES
    return _lib.load().ttsx_gated_scan_workspace(B, T, D, DTYPES[dtype], backward) // (8 * B * D)


def _case(dtype, wide):
    D = 4091 if not wide else 2560 if dtype == torch.float32 else 5120
    for backward in (0, 1):
        chunks = _chunks(3, D, dtype, backward)
        assert chunks > 1 and T / chunks > (LARGEST_TILE if wide else 64)
    x, g, h0, _ = _inputs(3, T, D, dtype, 17)
    return x, g, h0, torch.tensor(ENDS, dtype=torch.int32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
@pytest.mark.parametrize("reverse", [False, True])
def test_chunks_of_several_tiles(dtype, wide, reverse):
    x, g, h0, lengths = _case(dtype, wide)
    _check_scan(x, g, h0, lengths, reverse, dtype)
    _check_backward(x, g, h0, lengths, reverse, dtype, 18)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_chunks_of_several_tiles_repeat_themselves(dtype):
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    x, g, h0, lengths = _case(dtype, True)
    gx, gg, gh, gl = _gpu(x), _gpu(g), h0.cuda(), lengths.cuda()
    dh = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()

    def work():
        h, last, states = gated_scan(gx, gg, h0=gh, lengths=gl, save_states=True)
        return [h, last, states, *gated_scan_backward(dh, gx, gg, states, lengths=gl)]
    first = work()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, work()))
    for b, n in enumerate(ENDS):
        for t in (first[0], first[3], first[4]):
            assert not t[b, n:].any()
