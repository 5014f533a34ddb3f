"""Beam selection and the caches that follow it (include/hako_search.h).

Choices are compared exactly with the definition in float64: the kernels' sums of exponentials carry about 2^-24 / sqrt(n),
so two continuations are told apart from 1e-6 on; inputs whose order hangs on less are made equal on purpose (same beam:
equal logits; different beams: equal rows). Scores are rounded once from a value whose error is below 2^-22 of 1 (the
logarithm of a sum to 2^-23, relative) and half an fp32 step of the score itself."""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8

pytestmark = pytest.mark.gpu


def i32(gpu, v):
    return gpu.upload(np.asarray(v, np.int32))


def choose(logits, score, done, eos, n_beams, n_pick, arrange=False):
    """One request: rows of (parent, token, score, done), by the definition."""
    all_ = []
    for b in range(n_beams):
        if done is not None and done[b]:
            if score[b] > -math.inf:
                all_.append((-float(score[b]), b, -math.inf, eos, 1))
            continue
        x = logits[b].astype(np.float64)
        top = x.max()
        if not np.isfinite(top) or np.isnan(x).any():
            continue
        lse = top + math.log(np.exp(x - top).sum())
        best = np.argsort(-x, kind="stable")[:n_pick]
        all_ += [(-(float(score[b]) + (x[t] - lse)), b, -x[t], int(t), int(t == eos)) for t in best]
    all_ = [c for c in all_ if c[0] < math.inf]
    picks = [(b, t, -v, e) for v, b, _, t, e in sorted(all_)[:n_pick]]
    picks += [(-1, -1, -math.inf, 0)] * (n_pick - len(picks))
    if arrange:
        place, rest = [None] * n_pick, []
        for c in picks:
            if c[0] >= 0 and place[c[0]] is None:
                place[c[0]] = c
            else:
                rest.append(c)
        picks = [rest.pop(0) if c is None else c for c in place]
    return picks


def run_select(gpu, logits, score, done, eos, n_req, K, pick, arrange=False, with_done=True, ld=None):
    V = logits.shape[1]
    ld = ld or V
    wide = np.full((n_req * K, ld), np.nan, np.float32)
    wide[:, :V] = logits
    bufs = [gpu.upload(wide), gpu.upload(score.astype(np.float32))] + ([] if done is None else [i32(gpu, done)])
    outs = [gpu.upload(np.full(n_req * pick + 1, 77, np.int32)) for _ in range(4)]
    gpu.beam_select(bufs[0], ld, V, bufs[1], None if done is None else bufs[2], eos, n_req, K, pick, arrange, *outs[:3],
                    outs[3] if with_done else None)
    got = [gpu.download(o, t, (n_req * pick + 1,)) for o, t in zip(outs, (np.int32, np.int32, np.float32, np.int32))]
    for b in bufs + outs:
        b.free()
    assert all(g.view(np.int32)[-1] == 77 for g in got)
    if not with_done:
        assert (got[3] == 77).all()
    return [g[:-1].reshape(n_req, pick) for g in got]


def check(got, logits, score, done, eos, n_req, K, pick, arrange=False):
    parent, token, out, ended = got
    for r in range(n_req):
        at = slice(r * K, r * K + K)
        want = choose(logits[at], score[at], None if done is None else done[at], eos, K, pick, arrange)
        assert list(zip(parent[r], token[r])) == [c[:2] for c in want], r
        assert list(ended[r]) == [c[3] for c in want]
        for g, c in zip(out[r], want):
            assert g == c[2] or abs(float(g) - c[2]) <= 2.0 ** -22 + abs(c[2]) * 2.0 ** -24, (g, c)


@pytest.mark.parametrize("K,pick", [(1, 1), (1, 2), (4, 4), (4, 8), (5, 7), (8, 16), (16, 16), (16, 32), (2, 32)])
@pytest.mark.parametrize("V", [1, 2, 3, 17, 64, 257, 1023, 1024, 1025, 5000, 32003])
def test_select(gpu, K, pick, V):
    """Vocabularies of one token to many parts, odd sizes and strides, fewer continuations than places."""
    rng = np.random.default_rng(K * V + pick)
    n = 3
    logits = rng.standard_normal((n * K, V)).astype(np.float32) * 3
    score = (-20 * rng.random(n * K)).astype(np.float32)
    done = (rng.random(n * K) < 0.2).astype(int)
    for eos, dn in ((V // 2, done), (-1, None)):
        got = run_select(gpu, logits, score, dn, eos, n, K, pick, ld=V + 3)
        check(got, logits, score, dn, eos, n, K, pick)


@pytest.mark.parametrize("rows", [(1, 4), (300, 2), (40, 16)])
def test_select_many_and_large(gpu, rows):
    """The largest vocabulary of the benchmark by few rows (every part a tile), and rows enough that a part is a row's
    length; a spread of scores that leaves beams out."""
    n, K = rows
    V = 152064 if n == 1 else 20011
    rng = np.random.default_rng(n)
    logits = (rng.standard_normal((n * K, V)) * 2.5).astype(np.float32)
    logits[np.arange(n * K), rng.integers(0, V, n * K)] += 9
    score = (-6 * rng.random(n * K)).astype(np.float32)
    got = run_select(gpu, logits, score, None, 7, n, K, 2 * K)
    check(got, logits, score, None, 7, n, K, 2 * K)


@pytest.mark.parametrize("V", [40, 4096, 9001])
@pytest.mark.parametrize("what", ["flat", "two values", "rising", "falling", "few", "zeros of both signs", "every 4th", "lane"])
def test_ties_and_orders(gpu, V, what):
    """Equal continuations go by beam and token, however many there are; orders that make every value a candidate."""
    K, pick = 4, 16
    x = {"flat": np.zeros(V), "two values": np.arange(V) % 2, "rising": np.arange(V) / 1000, "falling": -np.arange(V) / 1000,
         "few": np.where(np.arange(V) < 5, 1.0, -np.inf), "zeros of both signs": np.where(np.arange(V) % 3, -0.0, 0.0),
         "every 4th": (np.arange(V) % 4 == 3) * 2.0, "lane": (np.arange(V) % 256 < 12) * (1 + np.arange(V) / V)}[what]
    logits = np.tile(x, (2 * K, 1)).astype(np.float32)
    score = np.array([-1, -1, -1, -1, -3, -2, -2, -1], np.float32)
    got = run_select(gpu, logits, score, None, 0, 2, K, pick)
    check(got, logits, score, None, 0, 2, K, pick)


def test_rows_that_are_not_finite(gpu):
    """-inf leaves a token or a beam out; NaN and +inf the whole row; then places stay empty. A beam with nothing but
    -inf, scores that are -inf or NaN, and a request with nothing at all."""
    K, V, pick = 4, 3000, 8
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((5 * K, V)).astype(np.float32)
    score = np.full(5 * K, -1.0, np.float32)
    logits[0, :] = -np.inf
    logits[1, 2999] = np.nan
    logits[2, 0] = np.inf
    logits[3, 3:] = -np.inf                      # three continuations in all
    logits[4:8, :2000] = -np.inf                 # whole parts of -inf
    score[8:12] = [-np.inf, -1, np.nan, -2]
    logits[12:16] = np.nan                       # nothing at all
    logits[16] = -np.inf
    logits[16, 17] = np.nan                      # a part with NaN and nothing finite
    score[17], score[18] = -np.inf, -np.inf
    got = run_select(gpu, logits, score, None, 1, 5, K, pick)
    score2 = np.where(np.isnan(score), -np.inf, score)
    check(got, logits, score2, None, 1, 5, K, pick)
    assert (got[0][3] == -1).all() and (got[2][3] == -np.inf).all()
    assert (got[0][0, 3:] == -1).all() and (got[0][0, :3] == 3).all()


@pytest.mark.parametrize("size", [1e-30, 1.0, 300.0, 1e6, 3e37])
def test_logits_of_any_size(gpu, size):
    K, V = 3, 2500
    rng = np.random.default_rng(4)
    logits = (rng.standard_normal((K, V)) * size).astype(np.float32)
    score = np.array([0, -0.5, -1e4], np.float32)
    parent, token, out, _ = run_select(gpu, logits, score, None, 0, 1, K, 6)
    want = choose(logits, score, None, 0, K, 6)
    assert list(zip(parent[0], token[0])) == [c[:2] for c in want]
    np.testing.assert_allclose(out[0], [c[2] for c in want], rtol=2.0 ** -22, atol=2.0 ** -22)


def test_ended_beams(gpu):
    """Their one continuation is eos at their own score, and beats or loses as any; all ended; done_out left out."""
    K, V, pick, eos = 4, 500, 8, 499
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((3 * K, V)).astype(np.float32)
    logits[:, eos] += 8
    score = np.array([-1, -2, -50, -3, -1, -1, -1, -1, -9, -8, -7, -6], np.float32)
    done = np.array([1, 0, 1, 0, 1, 1, 1, 1, 0, 0, 0, 0])
    logits[0] = np.nan                           # what an ended beam's row holds is not looked at
    got = run_select(gpu, logits, score, done, eos, 3, K, pick)
    check(got, logits, score, done, eos, 3, K, pick)
    assert (got[0][1, 4:] == -1).all()
    run_select(gpu, logits, score, done, eos, 3, K, pick, with_done=False)


@pytest.mark.parametrize("K", [1, 2, 3, 8, 16])
def test_arranged(gpu, K):
    """Survivors keep their places; one beam that takes all; every beam its own; too few continuations."""
    rng = np.random.default_rng(K)
    V, n = 700, 40
    logits = (rng.standard_normal((n * K, V)) * 2).astype(np.float32)
    score = (-rng.random(n * K) * rng.choice([0.1, 2.0, 20.0], n * K)).astype(np.float32)
    score[:K] = -1000
    score[K - 1] = 0                             # the last beam takes all
    logits[K:2 * K, 3:] = -np.inf
    score[K:2 * K] = -np.inf
    score[K] = -1                                # three continuations of one beam
    done = (rng.random(n * K) < 0.1).astype(int)
    done[:2 * K] = 0
    got = run_select(gpu, logits, score, done, 5, n, K, K, arrange=True)
    check(got, logits, score, done, 5, n, K, K, arrange=True)
    assert (got[0][0] == K - 1).all()


def test_runs_repeat(gpu):
    rng = np.random.default_rng(6)
    logits = rng.standard_normal((32, 30000)).astype(np.float32)
    score = -rng.random(32).astype(np.float32)
    a, b = (run_select(gpu, logits, score, None, 0, 4, 8, 16) for _ in range(2))
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


# ── the caches ──

def layers(gpu, kind, n_kv, slots, max_seq, kvh, hd, rng):
    cs = [ref.Cache(gpu, kind, slots, max_seq, kvh, hd, rng) for _ in range(n_kv)]
    return cs, gpu.kv_layers([c.kv for c in cs])


@pytest.mark.parametrize("kind", [KV_Q8, KV_F16])
@pytest.mark.parametrize("K,KVH,hd,n_kv", [(2, 2, 128, 2), (4, 1, 64, 35), (5, 3, 128, 1), (8, 2, 64, 2), (16, 1, 128, 2), (1, 1, 64, 1)])
def test_reorder(gpu, kind, K, KVH, hd, n_kv):
    """Swaps, cycles, one for all, parents that are none, ranges of every kind; slots anywhere, some outside the cache;
    every other row as it was."""
    rng = np.random.default_rng(K)
    n, max_seq = 6, 150
    slots = n * K + 3
    cs, kv = layers(gpu, kind, n_kv, slots, max_seq, KVH, hd, rng)
    parent = rng.integers(0, K, (n, K))
    parent[0] = np.roll(np.arange(K), 1)                       # a cycle
    parent[1] = np.arange(K)[::-1]                             # swaps
    parent[2] = K - 1
    parent[3] = rng.choice([-1, K, 2 ** 31 - 1, -2 ** 31, 0], K)
    since, length = [0, 7, 149, 30, -5, 60], [150, 133, 1000, 31, 64, 60]
    for slot in (None, rng.permutation(slots)[:n * K]):
        if slot is not None:
            slot[-1], slot[K] = slots, -1
        for s in (since, None):
            want = []
            for c in cs:
                got = c.pull()
                new = [a.copy() for a in got]
                for r in range(n):
                    lo, hi = max(s[r], 0) if s else 0, min(length[r], max_seq)
                    for b in range(K):
                        p = parent[r, b]
                        at = [r * K + x if slot is None else slot[r * K + x] for x in (b, p if 0 <= p < K else b)]
                        if 0 <= p < K and all(0 <= x < slots for x in at):
                            for x, y in zip(new, got):
                                x[at[0], :, lo:hi] = y[at[1], :, lo:hi]
                want.append(new)
            bufs = [i32(gpu, parent), i32(gpu, length)] + ([] if s is None else [i32(gpu, s)])
            ds = None if slot is None else i32(gpu, slot)
            gpu.kv_reorder(kv, ds, bufs[0], n, K, None if s is None else bufs[2], bufs[1])
            for c, w in zip(cs, want):
                for a, b in zip(c.pull(), w):
                    assert np.array_equal(a, b)
            for b in bufs + ([] if ds is None else [ds]):
                b.free()
    for c in cs:
        c.free()


def test_reorder_long(gpu):
    """Rows past 2^31 bytes of a cache, and ranges that many workgroups share."""
    from hako_amd.gpu import Kv
    K, max_seq, KVH, hd = 2, 600000, 16, 128
    kv = Kv(KV_Q8, K, max_seq, KVH, hd, None, None, None, None)
    codes, scales = gpu.kv_bytes(kv)
    assert codes > 2 ** 31
    bufs = [gpu.alloc(codes), gpu.alloc(codes), gpu.alloc(scales), gpu.alloc(scales)]
    kv = Kv(KV_Q8, K, max_seq, KVH, hd, *(b.ptr for b in bufs))
    rng = np.random.default_rng(1)
    n = 5000
    rows = rng.integers(-127, 128, (n, hd)).astype(np.int8)
    at = ((1 * KVH + 15) * max_seq + max_seq - n) * hd           # the last head of the last slot
    gpu.h2d(bufs[1].ptr + at, rows)
    parent, since, length = i32(gpu, [1, 1]), i32(gpu, [max_seq - n]), i32(gpu, [max_seq])
    gpu.kv_reorder(gpu.kv_layers([kv]), None, parent, 1, K, since, length)
    to = (15 * max_seq + max_seq - n) * hd
    assert np.array_equal(gpu.download(bufs[1].ptr + to, np.int8, (n, hd)), rows)
    for b in bufs + [parent, since, length]:
        b.free()


# ── as they are used ──

@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("arrange", [False, True])
def test_beam_search(gpu, captured, arrange):
    """A search over a small model whose next logits hang on the beam's whole cached text (attention over it, times an
    embedding): every step's beams and scores are those of a search in float64 that keeps texts, not caches."""
    rng = np.random.default_rng(7)
    n, K, H, KVH, hd, V, steps, eos = 2, 4, 4, 2, 64, 301, 24, 9
    D, KV = H * hd, KVH * hd
    ld = D + 2 * KV
    emb = (rng.standard_normal((V, ld))).astype(np.float32)
    head = (rng.standard_normal((V, D)) * 0.25).astype(np.float32)
    c = ref.Cache(gpu, KV_F16, n * K, steps, KVH, hd, fill=0)
    kv = gpu.kv_layers([c.kv])
    # both score buffers and flags in turn: what a call writes overlaps nothing that it reads
    dx, dq, do, dl = gpu.alloc(4 * n * K * ld), gpu.alloc(4 * n * K * D), gpu.alloc(4 * n * K * D), gpu.alloc(4 * n * K * V)
    score = [gpu.upload(np.tile(np.array([0] + [-np.inf] * (K - 1), np.float32), n)), gpu.alloc(4 * n * K)]
    done = [i32(gpu, [0] * (n * K)), gpu.alloc(4 * n * K)]
    parent, token = gpu.alloc(4 * n * K), gpu.alloc(4 * n * K)
    pos, ends, since = gpu.alloc(4 * n * K), gpu.alloc(4 * n * K), i32(gpu, [0] * n)
    ends_req = gpu.alloc(4 * n)

    def select(k):
        gpu.beam_select(dl, V, V, score[k], done[k], eos, n, K, K, arrange, parent, token, score[1 - k], done[1 - k])
        gpu.kv_reorder(kv, None, parent, n, K, since, ends_req)

    def logits(texts):
        """Rows of the cache for the newest tokens, and every beam's logits."""
        t = len(texts[0]) - 1
        gpu.h2d(dx, emb[[x[-1] for x in texts]])
        gpu.h2d(pos, np.full(n * K, t, np.int32))
        gpu.h2d(ends, np.full(n * K, t + 1, np.int32))
        gpu.h2d(ends_req, np.full(n, t + 1, np.int32))
        gpu.kv_append(c.kv, None, pos, n * K, dx.ptr + 4 * D, dx.ptr + 4 * (D + KV), ld)
        gpu.h2d(dq, emb[[x[-1] for x in texts]][:, :D].copy())
        gpu.attn_decode(do, D, dq, D, c.kv, None, ends, n * K, H, 0.125)
        x = gpu.download(do, np.float32, (n * K, D)).astype(np.float64) @ head.T
        gpu.h2d(dl, x.astype(np.float32))
        return x.astype(np.float32)

    def exact_logits(text):
        """The same of a text by itself, in float64 from its cached values."""
        x = emb[text]
        k, v = (x[:, D + i * KV:D + (i + 1) * KV].reshape(len(text), KVH, hd) for i in range(2))
        K_, V_ = (np.moveaxis((lambda r: r[0].astype(np.float64) * r[1].astype(np.float64)[..., None])(ref.rows(a, KV_F16)), 0, 1)[None] for a in (k, v))
        return ref.attend(x[-1, :D].reshape(H, hd), K_, V_, 0, len(text), 0.125).reshape(-1) @ head.T

    texts, graphs, values = [[1]] * (n * K), {}, np.tile(np.array([0.0] + [-np.inf] * (K - 1)), n)
    for t in range(steps - 1):
        k, got = t % 2, logits(texts)
        for r in range(n * K):
            if values[r] > -np.inf and eos not in texts[r][1:]:
                # attention to 1e-5 of its largest output, through D products
                np.testing.assert_allclose(got[r], exact_logits(texts[r]), atol=1e-5 * np.abs(head).sum(1).max() * 4)
        old = gpu.download(score[k], np.float32, (n * K,))
        ended = gpu.download(done[k], np.int32, (n * K,))
        if captured and t >= 2 and k not in graphs:
            gpu.capture_begin()
            select(k)
            graphs[k] = gpu.capture_end()
        if k in graphs:
            gpu.graph_launch(graphs[k])
        else:
            select(k)
        p, tok = (gpu.download(b, np.int32, (n, K)) for b in (parent, token))
        new, nd = gpu.download(score[1 - k], np.float32, (n * K,)), gpu.download(done[1 - k], np.int32, (n * K,))
        check([p, tok, new.reshape(n, K), nd.reshape(n, K)], got, old, ended, eos, n, K, K, arrange)
        assert (p >= 0).all()
        texts = [texts[r * K + p[r, b]] + [int(tok[r, b])] for r in range(n) for b in range(K)]
        values = new.astype(np.float64)
    for r in range(n):                                           # (both requests start alike)
        assert len({tuple(x) for x in texts[r * K:r * K + K]}) == K
    for g in graphs.values():
        gpu.graph_destroy(g)
    for b in [dx, dq, do, dl, parent, token, pos, ends, since, ends_req] + score + done:
        b.free()
    c.free()
