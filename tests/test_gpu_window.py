"""Attention over a window and sinks (include/hako_attn.h) against float64 on the same cached values.

The bound is that of test_gpu_attn.py, 1e-5 of the largest output, with its derivation: the products and sums are the
same, over fewer keys."""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8

pytestmark = pytest.mark.gpu

TUNE_ATTN_PROMPT = 21
TOL = 1e-5
KINDS = [KV_Q8, KV_F16]


def attend(q, K, V, slot, t, scale, window, sinks):
    """The token at position t in float64 (t < 0: none): q [heads][head_dim]."""
    H, hd = q.shape
    G, out = H // K.shape[1], np.zeros(q.shape)
    p = np.arange(t + 1)
    p = p[(p > t - window) | (p < sinks)]
    if not len(p):
        return out
    for g in range(K.shape[1]):
        s = q[g * G:(g + 1) * G].astype(np.float64) @ K[slot, g, p].T * scale
        w = np.exp(s - s.max(1, keepdims=True))
        out[g * G:(g + 1) * G] = w @ V[slot, g, p] / w.sum(1, keepdims=True)
    return out


def close(got, want):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    top = np.nanmax(np.abs(want), initial=0.0)
    err = np.nanmax(np.abs(got - want), initial=0.0)
    assert err <= TOL * top, f"error {err:.3g} of {top:.3g}"


def run_decode(gpu, c, q, slot, lens, scale, window, sinks, ldo=None):
    n, H, hd = q.shape
    D = H * hd
    ldo = ldo or D
    dq, out = gpu.upload(q), gpu.upload(np.full((n, ldo), 7.0, np.float32))
    ds, dl = None if slot is None else gpu.upload(np.asarray(slot, np.int32)), gpu.upload(np.asarray(lens, np.int32))
    gpu.attn_decode_window(out, ldo, dq, D, c.kv, ds, dl, n, H, scale, window, sinks)
    got = gpu.download(out, np.float32, (n, ldo))
    for b in (dq, out, dl) + (() if ds is None else (ds,)):
        b.free()
    assert (got[:, D:] == 7.0).all()
    return got[:, :D].reshape(n, H, hd)


# window, sinks: shorter and longer than the text, sinks inside the window, at its border, past a step, past everything
REACH = [(1, 0), (1, 1), (2, 4), (31, 0), (32, 32), (33, 33), (64, 5), (100, 64), (128, 200), (1000, 4), (200, 1000), (2 ** 31 - 1, 2 ** 31 - 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,KVH,hd", [(28, 4, 128), (16, 1, 64), (8, 8, 128), (14, 2, 64)])
def test_decode(gpu, kind, H, KVH, hd):
    rng = np.random.default_rng(H * 7 + kind)
    lens = [0, 1, 2, 3, 31, 32, 33, 36, 37, 63, 64, 65, 95, 96, 97, 127, 128, 129, 133, 160, 161, 205, 263, 399, 400, -3]
    c = ref.Cache(gpu, kind, len(lens), 400, KVH, hd, rng)
    K, V = c.values()
    q = rng.standard_normal((len(lens), H, hd)).astype(np.float32)
    slot = rng.permutation(len(lens))
    for window, sinks in REACH:
        got = run_decode(gpu, c, q, slot, lens, 1 / math.sqrt(hd), window, sinks, H * hd + 4)
        for i, n in enumerate(lens):
            close(got[i], attend(q[i], K, V, slot[i], n - 1, 1 / math.sqrt(hd), window, sinks))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,max_seq,window,sinks", [(1, 9000, 1024, 4), (3, 9000, 5000, 70), (2, 9000, 8000, 0), (70, 700, 500, 3)])
def test_decode_in_parts(gpu, kind, n, max_seq, window, sinks):
    """Windows that several workgroups share, and sequences enough to fill the chip."""
    H, KVH, hd = 28, 4, 128
    rng = np.random.default_rng(n)
    c = ref.Cache(gpu, kind, n, max_seq, KVH, hd, rng)
    K, V = c.values()
    lens = [max_seq - (i * 677) % (max_seq - 1) for i in range(n)]
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    got = run_decode(gpu, c, q, None, lens, 0.09, window, sinks)
    for i in range(n):
        close(got[i], attend(q[i], K, V, i, lens[i] - 1, 0.09, window, sinks))
    c.free()


def test_decode_of_many_in_parts(gpu):
    """Sequences enough to fill the chip (they read two slots by turns) under a window of several long parts."""
    H, KVH, hd, n, max_seq, W, S = 16, 16, 64, 17, 17000, 16500, 40
    rng = np.random.default_rng(17)
    c = ref.Cache(gpu, KV_Q8, 2, max_seq, KVH, hd, rng)
    K, V = c.values()
    lens = [17000, 3, 16541, 16540, 9000, 16999, 1, 0, 12345, 8192, 8193, 16384, 16500, 16501, 17000, 100, 16700]
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    slot = [i % 2 for i in range(n)]
    got = run_decode(gpu, c, q, slot, lens, 0.125, W, S)
    for i in range(n):
        close(got[i], attend(q[i], K, V, slot[i], lens[i] - 1, 0.125, W, S))
    c.free()


def test_everything_in_sight_is_the_other_call(gpu):
    """A window that covers the text: the same numbers as without one, to the bound."""
    rng = np.random.default_rng(5)
    c = ref.Cache(gpu, KV_Q8, 2, 300, 2, 128, rng)
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    got = run_decode(gpu, c, q, None, [300, 77], 0.1, 300, 0)
    dq, out, dl = gpu.upload(q), gpu.alloc(q.nbytes), gpu.upload(np.array([300, 77], np.int32))
    gpu.attn_decode(out, 1024, dq, 1024, c.kv, None, dl, 2, 8, 0.1)
    close(got, gpu.download(out, np.float32, q.shape).astype(np.float64))
    for b in (dq, out, dl):
        b.free()
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_leaves_out_what_is_not_in_sight(gpu, kind):
    """Rows behind the window, between the sinks and it and past the token hold NaN, infinite and huge rows: no trace.
    A NaN row inside is seen by its own heads alone; a slot outside the cache and a length below 1 give zeros."""
    H, KVH, hd, n, W, S = 8, 2, 128, 150, 40, 5
    rng = np.random.default_rng(11)
    c = ref.Cache(gpu, kind, 3, 200, KVH, hd, rng)
    seen = np.zeros(200, bool)
    seen[:S] = seen[n - W:n] = True
    for a in (c.ks, c.vs):
        a[:, :, ~seen] = np.nan
        a[:, :, S] = np.inf
        a[:, :, n - W - 1] = 1e30
        a[:, :, n] = 1e30
    K, V = c.values()
    q = rng.standard_normal((5, H, hd)).astype(np.float32)
    c.ks[2, 1, n - 3] = np.nan
    c.push()
    got = run_decode(gpu, c, q, [0, 1, 2, 3, -1], [n, n, n, n, n], 0.1, W, S)
    want = [attend(q[i], K, V, i, n - 1, 0.1, W, S) for i in range(3)]
    close(got[:2], np.array(want[:2]))
    close(got[2, :4], want[2][:4])
    assert np.isnan(got[2, 4:]).all()
    assert (got[3:] == 0).all()
    c.free()


def run_prompt(gpu, c, q, slot, start, lens, scale, window, sinks):
    n, H, hd = q.shape
    dq, out = gpu.upload(q), gpu.upload(np.full((n + 2, H * hd), 7.0, np.float32))
    a = [None if v is None else np.asarray(v, np.int32) for v in (slot, start, lens)]
    gpu.attn_prompt_window(out, H * hd, dq, H * hd, c.kv, *a, len(lens), H, scale, window, sinks)
    got = gpu.download(out, np.float32, (n + 2, H, hd))
    dq.free()
    out.free()
    assert (got[n:] == 7.0).all()   # rows behind the last sequence
    return got[:n]


@pytest.mark.parametrize("knob", [1, 2, 3])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,KVH,hd", [(28, 4, 128), (16, 1, 64), (6, 6, 128), (8, 2, 64)])
def test_prompt(gpu, kind, knob, H, KVH, hd):
    """Each kernel: tiles and parts that end anywhere, starts of 0 and later, a prompt of one token and of none."""
    rng = np.random.default_rng(H + knob)
    lens, start, slot = [1, 77, 0, 300, 33, 64, 130], [0, 20, 5, 0, 400, 100, 230], [3, 0, 6, 2, 1, 5, 4]
    c = ref.Cache(gpu, kind, 7, 450, KVH, hd, rng)
    K, V = c.values()
    q = rng.standard_normal((sum(lens), H, hd)).astype(np.float32)
    gpu.tune(TUNE_ATTN_PROMPT, knob)
    try:
        for window, sinks in [(1, 0), (1, 3), (7, 4), (32, 32), (64, 0), (65, 70), (100, 5), (310, 33), (2 ** 31 - 1, 0), (5, 2 ** 31 - 1)]:
            got, row = run_prompt(gpu, c, q, slot, start, lens, 0.1, window, sinks), 0
            want = np.concatenate([[attend(q[r + i], K, V, slot[s], start[s] + i, 0.1, window, sinks) for i in range(lens[s])]
                                   for s, r in enumerate(np.cumsum([0] + lens[:-1])) if lens[s]])
            close(got, want)
    finally:
        gpu.tune(TUNE_ATTN_PROMPT, 0)
    c.free()


@pytest.mark.parametrize("knob", [0, 1, 2, 3])
@pytest.mark.parametrize("lens,start,window,sinks", [([40], [5000], 4000, 4), ([700, 5], [0, 4200], 300, 0), ([257, 1], [3900, 5038], 4000, 100)])
def test_prompt_in_parts(gpu, knob, lens, start, window, sinks):
    """Few tokens under a long window: the keys in parts, the last tile not full."""
    H, KVH, hd = 14, 2, 128
    rng = np.random.default_rng(3)
    c = ref.Cache(gpu, KV_Q8, len(lens), 5040, KVH, hd, rng)
    K, V = c.values()
    q = rng.standard_normal((sum(lens), H, hd)).astype(np.float32)
    gpu.tune(TUNE_ATTN_PROMPT, knob)
    try:
        got, row = run_prompt(gpu, c, q, None, start, lens, 0.09, window, sinks), 0
    finally:
        gpu.tune(TUNE_ATTN_PROMPT, 0)
    for s, n in enumerate(lens):
        for i in sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n))):
            close(got[row + i], attend(q[row + i], K, V, s, start[s] + i, 0.09, window, sinks))
        row += n
    c.free()


@pytest.mark.parametrize("knob", [1, 2, 3])
def test_prompt_leaves_out_what_is_not_in_sight(gpu, knob):
    """A row that is NaN or huge reaches the tokens whose window holds it and no other, whatever else their tile sees."""
    H, KVH, hd, n, W, S, bad = 8, 2, 128, 200, 50, 4, 90
    rng = np.random.default_rng(2)
    c = ref.Cache(gpu, KV_F16, 1, 200, KVH, hd, rng)
    c.vs[0, :, bad] = 1e20
    c.push()
    K, V = c.values()
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    gpu.tune(TUNE_ATTN_PROMPT, knob)
    try:
        got = run_prompt(gpu, c, q, None, [0], [n], 0.1, W, S)
        c.ks[0, :, bad] = np.nan
        c.push()
        nan = run_prompt(gpu, c, q, None, [0], [n], 0.1, W, S)
    finally:
        gpu.tune(TUNE_ATTN_PROMPT, 0)
    sees = np.zeros(n, bool)
    sees[bad:bad + W] = True
    want = np.array([attend(q[i], K, V, 0, i, 0.1, W, S) for i in range(n)])
    close(got[~sees], want[~sees])
    close(got[sees], want[sees])
    assert np.isnan(nan[sees]).all() and (nan[~sees] == got[~sees]).all()
    c.free()


def test_a_ring_is_a_window(gpu):
    """Rows of a slot of sinks + window rows used as a ring, appended with their turns apart: single tokens see in it what
    the window shows in a slot that holds the whole text."""
    H, KVH, hd, W, S, n = 8, 2, 64, 48, 4, 173
    rng = np.random.default_rng(8)
    x = rng.standard_normal((n, (H + 2 * KVH) * hd)).astype(np.float32)
    t = ref.table(n, hd)
    whole, ring = ref.Cache(gpu, KV_Q8, 1, n, KVH, hd, fill=0), ref.Cache(gpu, KV_Q8, 1, S + W, KVH, hd, fill=0)
    from hako_amd.gpu import Rope
    dx, dt, qa, qb, oa, ob = gpu.upload(x), gpu.upload(t), *(gpu.alloc(4 * n * H * hd) for _ in range(4))
    rope, ld, D, KV = Rope(dt.ptr, n, hd, 0), (H + 2 * KVH) * hd, H * hd, KVH * hd
    slot = gpu.upload(np.zeros(n, np.int32))
    pos = np.arange(n, dtype=np.int32)
    dp, dr = gpu.upload(pos), gpu.upload(np.where(pos < S, pos, S + (pos - S) % W).astype(np.int32))
    ends, full = gpu.upload(pos + 1), gpu.upload(np.minimum(pos + 1, S + W).astype(np.int32))
    for i in range(n):
        at = lambda b: b.ptr + 4 * i   # noqa: E731
        row = dx.ptr + 4 * i * ld
        gpu.kv_append(whole.kv, slot, at(dp), 1, row + 4 * D, row + 4 * (D + KV), ld, rope, row, qa.ptr + 4 * i * D, H, ld, D)
        gpu.kv_append_turned(ring.kv, slot, at(dr), at(dp), 1, row + 4 * D, row + 4 * (D + KV), ld, rope, row, qb.ptr + 4 * i * D, H, ld, D)
        gpu.attn_decode_window(oa.ptr + 4 * i * D, D, qa.ptr + 4 * i * D, D, whole.kv, slot, at(ends), 1, H, 0.125, W, S)
        gpu.attn_decode(ob.ptr + 4 * i * D, D, qb.ptr + 4 * i * D, D, ring.kv, slot, at(full), 1, H, 0.125)
    a, b = (gpu.download(o, np.float32, (n, H * hd)) for o in (oa, ob))
    assert np.array_equal(gpu.download(qa, np.float32, (n, D)), gpu.download(qb, np.float32, (n, D)))
    close(b, a.astype(np.float64))
    for buf in (dx, dt, qa, qb, oa, ob, slot, dp, dr, ends, full):
        buf.free()
    whole.free()
    ring.free()


@pytest.mark.parametrize("kind", KINDS)
def test_captured(gpu, kind):
    """A captured call follows slots and lengths; each replay writes the bits of the eager call, and calls repeat."""
    H, KVH, hd, n = 14, 2, 128, 5
    rng = np.random.default_rng(9)
    c = ref.Cache(gpu, kind, n, 2000, KVH, hd, rng)
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    dq, out, ds, dl = gpu.upload(q), gpu.alloc(q.nbytes), gpu.upload(np.arange(n, dtype=np.int32)), gpu.upload(np.ones(n, np.int32))

    def call():
        gpu.attn_decode_window(out, H * hd, dq, H * hd, c.kv, ds, dl, n, H, 0.09, 700, 6)

    call()
    gpu.capture_begin()
    call()
    graph = gpu.capture_end()
    for step in range(4):
        gpu.h2d(ds, rng.permutation(n).astype(np.int32))
        gpu.h2d(dl, rng.integers(0, 2001, n).astype(np.int32))
        call()
        want = gpu.download(out, np.float32, q.shape)
        gpu.h2d(out, np.full(q.shape, 3, np.float32))
        gpu.graph_launch(graph)
        assert np.array_equal(gpu.download(out, np.float32, q.shape), want), step
    gpu.graph_destroy(graph)
    for b in (dq, out, ds, dl):
        b.free()
    c.free()
