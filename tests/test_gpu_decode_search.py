"""The decoder under a window, in a beam search and over drafted trees (include/hako_decode.h).

A step under a window is held against the numpy forward of test_gpu_decode_kv.py, whose bars and their derivation are the
same, with attention over what the window shows. A beam search is the decoder's own steps with the continuations chosen
in float64, so its tokens are equal. A drafted tree's picks come from a pass of many tokens: each is the maximum of the
logits of the same steps one at a time, up to what separates the two ways (the bars of test_gpu_decode_kv.py)."""
import numpy as np
import pytest

import attn_ref as ref
import test_gpu_window as window_ref
from hako_amd import mlf2
from hako_amd.decoder import Decoder
from hako_amd.gpu import KV_F16, KV_Q8, HakoGpuError
from helpers import maxabs_rel, near_max_steps, within
from test_gpu_beam import choose
from test_gpu_decode_batched import DENSE, KQM, SMALL_128, TINY, UNTIED_Q4_OUT
from test_gpu_decode_kv import STEP_BAR, Forward, rows_of

pytestmark = pytest.mark.gpu

KINDS = [KV_Q8, KV_F16]


@pytest.fixture
def model(tmp_path):
    def make(cfg, seed):
        path = str(tmp_path / f"m{seed}.mlf2")
        mlf2.write_qwen2(path, cfg, seed)
        return path
    return make


def louder(gpu, dec, n_layers, by=300.0):
    """Cached values times `by`: attention over them then decides the logits (in these models it is a thousandth of the
    residual stream, less than the bars)."""
    for l in range(n_layers):
        kv = dec.cache(l)
        shape = (kv.n_slots, kv.n_kv_heads, kv.max_seq)
        gpu.h2d(kv.v_scale, gpu.download(kv.v_scale, np.float32, shape) * np.float32(by))


# ── windows ──

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cfg,n_seq,window,sinks", [(TINY, 1, 20, 3), (SMALL_128, 1, 64, 0), (SMALL_128, 3, 33, 40), (KQM, 16, 1, 4),
                                                    (DENSE, 4, 1000, 0)])
def test_step_under_a_window(gpu, oracle, model, monkeypatch, kind, cfg, n_seq, window, sinks):
    path = model(cfg, 21)
    rng = np.random.default_rng(n_seq)
    n = [int(x) for x in rng.integers(32, 120, n_seq)]
    dec = Decoder(gpu, path, n_seq, 160, kind)
    try:
        dec.window(window, sinks)
        for s, m in enumerate(n):
            dec.prefill(rng.integers(0, cfg.vocab, m), s)
        louder(gpu, dec, cfg.n_layers)
        tok = rng.integers(0, cfg.vocab, n_seq).astype(np.int32)
        before = [[rows_of(gpu, dec, dec.cache(l), s, n[s]) for l in range(cfg.n_layers)] for s in range(n_seq)]
        _, lg = dec.step(tok, logits=True)
        # the same token as a prompt of one: the other kernel over the same rows
        dec.set_pos(n)
        _, one = dec.prefill(tok[:1], 0, logits=True)
    finally:
        dec.close()
    monkeypatch.setattr(ref, "attend", lambda q, K, V, slot, end, scale: window_ref.attend(q, K, V, slot, end - 1, scale, window, sinks))
    fwd = Forward(oracle, path)
    for s in range(n_seq):
        within(f"sequence {s}", lg[s], fwd.step(int(tok[s]), before[s], n[s], kind)[0], STEP_BAR[kind])
    within("prompt of one", one, lg[0], STEP_BAR[kind])


@pytest.mark.parametrize("kind", KINDS)
def test_window_comes_and_goes(gpu, model, kind):
    """Captured steps follow it; a window that shows everything is none; a prompt in one pass and in several is the same
    text."""
    path = model(SMALL_128, 8)
    rng = np.random.default_rng(3)
    prompt, tok = rng.integers(0, SMALL_128.vocab, 300), np.array([1, 2], np.int32)
    dec = Decoder(gpu, path, 2, 400, kind)

    def steps(n=8):
        dec.set_pos(300)
        cur, got, lgs = tok, [], []
        for _ in range(n):
            cur, lg = dec.step(cur, logits=True)
            got.append(cur)
            lgs.append(lg)
        return np.stack(got), np.stack(lgs)

    def generate(n=8):
        dec.set_pos(300)
        return dec.generate(tok, n)

    try:
        for s in range(2):
            dec.prefill(prompt, s)
        louder(gpu, dec, SMALL_128.n_layers)
        free, free_lg = steps()
        np.testing.assert_array_equal(generate(), free)
        dec.window(40, 4)
        near, near_lg = steps()
        np.testing.assert_array_equal(generate(), near)
        assert maxabs_rel(near_lg, free_lg) > 0.01        # it matters
        dec.window(10 ** 9, 0)
        _, all_lg = steps()
        # other kernels, the same sums in another order: a value next to an edge of the 8-bit activations may cross it
        within("all in sight", all_lg[0], free_lg[0], STEP_BAR[kind])
        dec.window(0)
        np.testing.assert_array_equal(generate(), free)
        dec.window(70, 2)
        dec.set_pos(0)
        _, whole = dec.prefill(prompt, 0, logits=True)
        for a, b in ((0, 113), (113, 114), (114, 300)):
            dec.prefill(prompt[a:b], 1)
        assert gpu.download(dec.cache(0).k, np.int8, (64,)).any()
        rows = [rows_of(gpu, dec, dec.cache(SMALL_128.n_layers - 1), s, 300) for s in range(2)]
        for a, b in zip(*rows):
            assert maxabs_rel(b, a) < 0.05                # through three layers of rounded rows, as test_gpu_decode_kv.py
    finally:
        dec.close()


# ── beams ──

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cfg,n_req,K,eos,prefix", [(TINY, 1, 4, -1, 0), (SMALL_128, 2, 3, 17, 0), (UNTIED_Q4_OUT, 1, 2, -1, 11),
                                                    (KQM, 1, 16, 5, 0), (DENSE, 2, 4, -1, 0)])
def test_beam(gpu, model, kind, cfg, n_req, K, eos, prefix):
    path, n, S = model(cfg, 9), 14, n_req * K
    rng = np.random.default_rng(K)
    lens = [int(x) for x in rng.integers(12, 60, n_req)]
    prompts = [rng.integers(0, cfg.vocab, m) for m in lens]
    first = rng.integers(0, cfg.vocab, n_req).astype(np.int32)
    dec, own = Decoder(gpu, path, S, 100, kind), Decoder(gpu, path, S, 100, kind)
    bufs = [gpu.alloc(4 * S) for _ in range(3)]
    try:
        for d in (dec, own):
            for r in range(n_req):
                d.prefill(prompts[r], r * K)
            if prefix:      # positions below it are sequence 0's alone
                d.set_pos(np.maximum(np.repeat(lens, K), prefix))
                d.share_prefix(0, prefix)
        got = [dec.beam(K, first, n, eos)]
        after = dec.step(got[0][0][:, -1].clip(0), logits=True)[1]
        # again, now from the beams that are there: the first of each goes back to its prompt's end
        dec.set_pos(np.repeat(lens, K))
        got.append(dec.beam(K, first, n, eos))

        # the same with the decoder's steps and a choice in float64
        kv = gpu.kv_layers([own.cache(l) for l in range(cfg.n_layers)])

        def reorder(parent, since, length):
            for b, v in zip(bufs, (parent, since, length)):
                gpu.h2d(b, np.ascontiguousarray(v, dtype=np.int32))
            gpu.kv_reorder(kv, None, bufs[0], n_req, K, bufs[1], bufs[2])

        reorder(np.zeros(S), np.full(n_req, prefix), lens)
        own.set_pos(np.repeat(lens, K))
        tok, texts = np.repeat(first, K), [[] for _ in range(S)]
        score, done = np.tile(np.array([0] + [-np.inf] * (K - 1), np.float32), n_req), np.zeros(S, int)
        for i in range(n):
            _, lg = own.step(tok, logits=True)
            picks = sum((choose(lg[r * K:r * K + K], score[r * K:r * K + K], done[r * K:r * K + K], eos, K, K, True) for r in range(n_req)), [])
            reorder([p for p, *_ in picks], lens, [m + i + 1 for m in lens])
            texts = [texts[s // K * K + p] + [t] for s, (p, t, _, _) in enumerate(picks)]
            tok, score, done = (np.array([c[j] for c in picks], x) for j, x in ((1, np.int32), (2, np.float32), (3, int)))
        _, lg = own.step(tok, logits=True)
    finally:
        dec.close()
        own.close()
        for b in bufs:
            b.free()
    for out, s in got:
        np.testing.assert_array_equal(out, np.array(texts))
        # each step's score is rounded to fp32 once, from a value within 2^-22
        np.testing.assert_allclose(s, score, atol=n * 2.0 ** -22, rtol=n * 2.0 ** -24)
    np.testing.assert_array_equal(after, lg)      # the caches hold the beams' texts


# ── drafted trees ──

def draft(rng, chain, n, vocab):
    """A tree of n nodes with `chain` in it, the other guesses anywhere."""
    tokens, parent = [chain[0]], [-1]
    at = sorted(rng.choice(np.arange(1, n), len(chain) - 1, replace=False)) if n > 1 else []
    last = 0
    for j in range(1, n):
        if j in at:
            tokens.append(chain[1 + at.index(j)])
            parent.append(last)
            last = j
        else:
            tokens.append(int(rng.integers(0, vocab)))
            parent.append(int(rng.integers(0, j)))
    return tokens, parent


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cfg,n_nodes,prefix", [(TINY, 1, 0), (TINY, 12, 0), (SMALL_128, 30, 0), (UNTIED_Q4_OUT, 64, 0), (KQM, 17, 20),
                                                (DENSE, 5, 0)])
def test_verify(gpu, model, kind, cfg, n_nodes, prefix):
    path = model(cfg, 10)
    rng = np.random.default_rng(n_nodes)
    prompts = [rng.integers(0, cfg.vocab, m) for m in (33, 47)]
    seq, rounds = 1, 8
    dec, own = Decoder(gpu, path, 2, 256, kind), Decoder(gpu, path, 2, 256, kind)
    kept = 0
    try:
        for d in (dec, own):
            for s in range(2):
                d.prefill(prompts[s], s)
            if prefix:
                d.share_prefix(0, prefix)
        pos, tok = [33, 47], 3
        other = [rows_of(gpu, dec, dec.cache(l), 0, 33) for l in range(cfg.n_layers)]
        for _ in range(rounds):
            length = min(n_nodes, 6)
            own.set_pos(pos)
            chain = [tok]
            for _ in range(length - 1):       # what greedy steps would say
                chain.append(int(own.step([0, chain[-1]])[1]))
            right = int(rng.integers(1, length + 1))
            chain = chain[:right] + [int(rng.integers(0, cfg.vocab)) for _ in chain[right:]]
            tokens, parent = draft(rng, chain, n_nodes, cfg.vocab)
            out = dec.verify(tokens, parent, seq)
            assert 1 <= len(out) <= n_nodes
            kept += len(out) >= right
            own.set_pos(pos)
            lgs = [own.step([0, t], logits=True)[1][1] for t in [tok] + list(out[:-1])]
            assert near_max_steps(lgs, out, lgs, STEP_BAR[kind]) == []
            pos[1] += len(out)
            tok = int(out[-1])
        assert kept >= rounds - 1             # (a pick may turn at a near tie)
        for a, b in zip(other, (rows_of(gpu, dec, dec.cache(l), 0, 33) for l in range(cfg.n_layers))):
            for x, y in zip(a, b):
                np.testing.assert_array_equal(x, y)
        # the caches hold the text's rows, turned by their places in it: layer 0's follow from tokens and places alone, so that
        # they differ by a code at most, and seldom
        step = 1 / 127 if kind == KV_Q8 else 2.0 ** -10
        for a, b in zip(*(rows_of(gpu, d, d.cache(0), seq, pos[1]) for d in (dec, own))):
            a, b = (x.reshape(-1, cfg.head_dim) for x in (a, b))
            assert (np.abs(a - b) <= (step + 1e-5) * np.abs(b).max(1, keepdims=True)).all()
            assert (np.abs(a - b) > 1e-5 * np.abs(b).max(1, keepdims=True)).mean() < 0.05
        # ... and its next step is that of the steps one at a time
        for d in (dec, own):
            d.set_pos(pos)
        within("next step", dec.step([0, tok], logits=True)[1][1], own.step([0, tok], logits=True)[1][1], 5 * STEP_BAR[kind])
    finally:
        dec.close()
        own.close()


def test_refusals(gpu, model):
    path = model(TINY, 3)
    plain, dec = Decoder(gpu, path, 4, 64), Decoder(gpu, path, 4, 64, KV_Q8)

    def refused(f, *a):
        with pytest.raises(HakoGpuError, match="rc=-1"):
            f(*a)

    try:
        refused(plain.window, 8, 0)
        refused(plain.beam, 2, 1, 3)
        refused(plain.verify, [1], [-1])
        for window, sinks in ((-1, 0), (8, -1)):
            refused(dec.window, window, sinks)
        t, out, score = np.ones(4, np.int32), np.zeros((4, 66), np.int32), np.zeros(4, np.float32)
        for k in (0, 1, 3, -2, 8):
            assert gpu.lib.hako_gpu_decoder_beam(dec.d, k, t.ctypes.data, 3, -1, out.ctypes.data, score.ctypes.data) == -1
        for tok, n in ((TINY.vocab, 3), (-1, 3), (1, 0), (1, -1), (1, 65), (1, 2 ** 31 - 1)):
            t[:] = tok
            assert gpu.lib.hako_gpu_decoder_beam(dec.d, 2, t.ctypes.data, n, -1, out.ctypes.data, score.ctypes.data) == -1
        for tokens, parent in (([1], [0]), ([1, 2], [-1, -1]), ([1, 2], [-1, 1]), ([TINY.vocab], [-1]), ([-1], [-1]), ([1] * 65, [-1] + [0] * 64),
                               ([1, 2, 3], [-1, 0, 2])):
            refused(dec.verify, tokens, parent)
        for seq in (-1, 4):
            refused(dec.verify, [1], [-1], seq)
        dec.set_pos(62)
        refused(dec.verify, [1] * 3, [-1, 0, 1])
        refused(dec.beam, 2, 1, 3)
        dec.verify([1, 1], [-1, 0])                       # what fits
        dec.set_pos(8)
        dec.window(8, 2)
        refused(dec.share_prefix, 0, 4)
        refused(dec.verify, [1], [-1])
        dec.window(0, 0)
        dec.share_prefix(0, 4)
        refused(dec.window, 8, 2)
        dec.set_pos(3)
        refused(dec.verify, [1], [-1])
        refused(dec.beam, 2, 1, 3)
    finally:
        plain.close()
        dec.close()
