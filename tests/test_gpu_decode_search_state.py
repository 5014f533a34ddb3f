"""What the decoder's searches leave behind: outputs of a refused call, captured steps across windows, ends and sizes of
beams, prompts of many tokens under a window (include/hako_decode.h)."""
import numpy as np
import pytest

from hako_amd.decoder import Decoder
from hako_amd.gpu import KV_F16, KV_Q8
from test_gpu_beam import choose
from test_gpu_decode_batched import KQM, SMALL_128, TINY
from test_gpu_decode_kv import rows_of
from test_gpu_decode_search import model   # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = [KV_Q8, KV_F16]


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


def hide(gpu, dec, n_layers, a, b):
    """Positions [a, b) of every sequence become NaN: a head that sees one, at whatever weight, answers NaN, which the
    matmuls' 8-bit activations take for 0."""
    for l in range(n_layers):
        kv = dec.cache(l)
        shape = (kv.n_slots, kv.n_kv_heads, kv.max_seq)
        scale = gpu.download(kv.v_scale, np.float32, shape)
        scale[:, :, a:b] = np.nan
        gpu.h2d(kv.v_scale, scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cfg,before,n,window,sinks", [(TINY, 60, 40, 30, 3), (SMALL_128, 100, 64, 20, 0), (SMALL_128, 80, 560, 70, 2),
                                                       (KQM, 90, 17, 50, 5), (KQM, 90, 3, 1, 0)])
def test_prompt_of_many_tokens_under_a_window(gpu, model, kind, cfg, before, n, window, sinks):   # noqa: F811
    """Its logits and rows do not move by a bit with what lies between the sinks and its first token's window; without the
    window they would."""
    path = model(cfg, 23)
    prompt = np.random.default_rng(n).integers(0, cfg.vocab, before + n)
    dec = Decoder(gpu, path, 2, 700, kind)

    def passes():
        dec.set_pos(before)
        _, lg = dec.prefill(prompt[before:], 1, logits=True)
        return lg, [rows_of(gpu, dec, dec.cache(l), 1, before + n) for l in range(cfg.n_layers)]

    try:
        dec.prefill(prompt[:before], 1)
        dec.window(window, sinks)
        lg, rows = passes()
        assert np.isfinite(lg).all()
        hide(gpu, dec, cfg.n_layers, sinks, before - window + 1)
        hidden, left = passes()
        np.testing.assert_array_equal(hidden, lg)
        for a, b in zip(left, rows):
            for x, y in zip(a, b):
                np.testing.assert_array_equal(x[before:], y[before:])
        dec.window(window + 1, sinks)
        assert not np.array_equal(passes()[1][1][0][before], rows[1][0][before])   # the first token sees one position more
        dec.window(0)
        assert not np.array_equal(passes()[0], lg)
    finally:
        dec.close()


def chosen(gpu, dec, n_layers, K, first, n, eos, at):
    """A beam search of one request of the decoder's sequences by its own steps, with the choice in float64."""
    S, bufs = dec.n_seq, [gpu.alloc(4 * dec.n_seq) for _ in range(3)]
    kv = gpu.kv_layers([dec.cache(l) for l in range(n_layers)])

    def reorder(parent, since, length):
        for b, v in zip(bufs, (parent, [since], [length])):
            gpu.h2d(b, np.ascontiguousarray(v, dtype=np.int32))
        gpu.kv_reorder(kv, None, bufs[0], 1, K, bufs[1], bufs[2])

    reorder(np.zeros(S), 0, at)
    dec.set_pos(at)
    tok, texts = np.full(S, first, np.int32), [[] for _ in range(S)]
    score, done = np.array([0] + [-np.inf] * (K - 1), np.float32), np.zeros(S, int)
    for i in range(n):
        picks = choose(dec.step(tok, logits=True)[1], score, done, eos, K, K, True)
        reorder([p for p, *_ in picks], at, at + i + 1)
        texts = [texts[p] + [t] for p, t, _, _ in picks]
        tok, score, done = (np.array([c[j] for c in picks], x) for j, x in ((1, np.int32), (2, np.float32), (3, int)))
    for b in bufs:
        b.free()
    return np.array(texts), score


@pytest.mark.parametrize("kind", KINDS)
def test_beams_of_one_decoder(gpu, model, kind):   # noqa: F811
    """Windows that come and go between searches, other ends, other numbers of beams: each the search of a decoder of its
    own, and of steps with a choice in float64. What lies outside the window is NaN: without it the beams are others."""
    cfg, S, at, n, window, sinks = SMALL_128, 4, 90, 10, 20, 2
    path = model(cfg, 12)
    prompt = np.random.default_rng(6).integers(0, cfg.vocab, at)

    def fresh():
        dec = Decoder(gpu, path, S, 128, kind)
        for s in range(S):
            dec.prefill(prompt, s)
        hide(gpu, dec, cfg.n_layers, sinks, at - window + 1)
        return dec

    dec, seen, eos = fresh(), {}, -1
    try:
        for K, ends, near in ((4, False, True), (4, False, False), (4, True, True), (2, True, True), (2, False, False), (4, False, True),
                              (4, True, True)):
            dec.window(window if near else 0, sinks if near else 0)
            dec.set_pos(at)
            got = dec.beam(K, 5, n, eos if ends else -1)
            own = fresh()
            try:
                if near:
                    own.window(window, sinks)
                want = own.beam(K, 5, n, eos if ends else -1)
                np.testing.assert_array_equal(got[0], want[0])
                np.testing.assert_array_equal(got[1], want[1])
                if K == S:
                    texts, score = chosen(gpu, own, cfg.n_layers, K, 5, n, eos if ends else -1, at)
                    np.testing.assert_array_equal(got[0], texts)
                    # (as in test_gpu_decode_search.py)
                    np.testing.assert_allclose(got[1], score, atol=n * 2.0 ** -22, rtol=n * 2.0 ** -24)
            finally:
                own.close()
            if (K, ends, near) in seen:
                np.testing.assert_array_equal(got[0], seen[K, ends, near][0])
                np.testing.assert_array_equal(got[1], seen[K, ends, near][1])
            seen[K, ends, near] = got
            if near and not ends:
                eos = int(got[0][0, n // 2])              # a token that a beam takes half way
        assert not np.array_equal(seen[4, False, True][0], seen[4, True, True][0])
        assert not np.array_equal(seen[4, False, True][0], seen[4, False, False][0])
    finally:
        dec.close()
