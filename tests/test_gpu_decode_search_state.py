"""What the decoder's searches leave behind: outputs of a refused call (include/hako_decode.h)."""
import numpy as np
import pytest

from hako_amd.decoder import Decoder
from hako_amd.gpu import KV_Q8
from test_gpu_decode_batched import TINY
from test_gpu_decode_search import model   # noqa: F401

pytestmark = pytest.mark.gpu


def test_refused_beams_leave_the_outputs(gpu, model):   # noqa: F811
    """Also where a later request is the one that is refused."""
    dec = Decoder(gpu, model(TINY, 3), 4, 64, KV_Q8)
    out, score = np.full((4, 8), 7, np.int32), np.full(4, 7.0, np.float32)

    def beam(tokens, n):
        t = np.array(tokens, np.int32)
        return gpu.lib.hako_gpu_decoder_beam(dec.d, 2, t.ctypes.data, n, -1, out.ctypes.data, score.ctypes.data)

    try:
        dec.set_pos([5, 5, 60, 60])
        assert beam([1, 2], 8) == -1                      # no room in the second request
        dec.set_pos([5, 5, 9, 9])
        assert beam([1, TINY.vocab], 8) == -1
        dec.share_prefix(0, 5)
        dec.set_pos([5, 5, 4, 4])
        assert beam([1, 2], 8) == -1                      # ... inside the prefix
        assert (out == 7).all() and (score == 7.0).all()
        dec.set_pos([5, 5, 9, 9])
        assert beam([1, 2], 8) == 0
        assert (out != 7).any() and (score < 0).all()
    finally:
        dec.close()
